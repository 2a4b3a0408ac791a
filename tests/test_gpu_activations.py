"""The activations of gemm_epilogue and quantize_gated at single values: NaN,
and the tails, where a result is small but a 16-bit type still resolves it."""

import pytest
import torch

import pearl_b200 as pg
from tests.test_gpu_layer_ops import BF16, F16, F32, act64, gen, int8, randn

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


def half_spacing(want, dtype):
    """Half the distance between neighbours of ``dtype`` around ``want``."""
    bits, least = (10, -14) if dtype is F16 else (7, -126)
    return torch.exp2(torch.frexp(want.abs())[1].sub(1).clamp(min=least).double() - bits - 1)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("act", list(pg.linear.ACTIVATIONS))
def test_activations_are_rounded_once_in_their_tails(dtype, act):
    """act(x) for x in -9..9 is the 16-bit neighbour of the exact value but
    for 2^-15 of it.  The f32 steps lose less: the exponential's argument (up
    to 96 in powers of two) a few 2^-24 of itself, gelu's polynomial 2^-17."""
    x = torch.linspace(-9, 9, 40000, device="cuda")
    A, B = (torch.ones(s, 16, dtype=torch.int8, device="cuda") for s in (40000, 8))
    C = torch.empty(40000, 8, dtype=dtype, device="cuda")
    pg.gemm_epilogue(A, B, x / 16, torch.ones(8, device="cuda"), C, activation=act)  # 16 * (x / 16), both exact
    want = act64(act, x.double())
    if act == "gelu_tanh":  # without 1 + tanh's cancellation
        u = 0.7978845608028654 * (x.double() + 0.044715 * x.double() ** 3)
        want = x.double() * torch.sigmoid(2 * u)
    off = (C.double() - want[:, None]).abs() - (half_spacing(want, dtype) + want.abs() * 2.0 ** -15)[:, None]
    assert bool((off <= 0).all()), f"worst {float(off.max()):.3g} at {float(x[int(off.amax(1).argmax())])}"
