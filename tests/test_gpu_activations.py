"""The activations of gemm_epilogue and quantize_gated on NaN."""

import pytest
import torch

import pearl_b200 as pg
from tests.test_gpu_layer_ops import BF16, gen, int8, randn

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield
    torch.cuda.synchronize()


@pytest.mark.parametrize("m,n,k", [(3, 40, 64), (3, 520, 4096), (200, 600, 640), (700, 512, 256)])
@pytest.mark.parametrize("act", list(pg.linear.ACTIVATIONS))
def test_linear_keeps_nan(m, n, k, act):
    """A NaN scale, bias or residual is a NaN in C, whatever the activation."""
    g = gen(m)
    A, B = int8(g, m, k), int8(g, n, k)
    sa, sb = torch.ones(m, device="cuda"), torch.full((n,), 1e-4, device="cuda")
    sa[m // 2], sb[n // 3] = float("nan"), float("nan")
    bias, r = randn(g, n).to(BF16), randn(g, m, n).to(BF16)
    bias[n - 1], r[m - 1, 5] = float("nan"), float("nan")
    C = torch.empty(m, n, dtype=BF16, device="cuda")
    pg.gemm_epilogue(A, B, sa, sb, C, bias=bias, activation=act, residual=r)
    want = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    want[m // 2], want[:, n // 3], want[:, n - 1], want[m - 1, 5] = True, True, True, True
    assert torch.equal(C.isnan(), want)


@pytest.mark.parametrize("n", [64, 1360, 4096, 20000])
@pytest.mark.parametrize("act", list(pg.linear.ACTIVATIONS))
@pytest.mark.parametrize("at", ["gate", "up"])
def test_quantize_gated_keeps_nan(n, act, at):
    g = gen(n)
    x = randn(g, 5, 2 * n).to(BF16)
    x[:, 0] = 1.0  # no row of zeros
    x[2, n - 3 if at == "gate" else 2 * n - 3] = float("nan")
    q, sc = torch.empty(5, n, dtype=torch.int8, device="cuda"), torch.empty(5, device="cuda")
    pg.quantization.quantize_gated(x, q, sc, activation=act)
    assert sc.isnan().tolist() == [False, False, True, False, False]
