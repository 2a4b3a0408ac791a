"""quantize_gated on rows at the ends of the float range."""

import pytest
import torch

import pearl_b200 as pg
from tests.test_gpu_layer_ops import BF16, gen, randn

pytestmark = pytest.mark.gpu
WIDTHS = [64, 1360, 4096, 20000]  # a warp, a block, a block's registers full, two passes


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield
    torch.cuda.synchronize()


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("max_val", [127, 63])
def test_rows_of_tiny_products(n, max_val):
    """Products c * 2^-e of integers c, exact in f32 down to its subnormals:
    the bytes are rint(c * max_val / max|c|) for every e, zeros among them."""
    g = gen(n)
    powers = [60, 100, 122, 124, 126, 128, 130, 134, 138, 142, 148]
    c = torch.randint(-100, 101, (len(powers), n), generator=g, device="cuda").double()
    c[:, :3] = torch.tensor([0.0, 100.0, -100.0], device="cuda")
    e = torch.tensor(powers, dtype=torch.float64, device="cuda")[:, None]
    x = torch.cat([c * 2.0 ** -60, torch.exp2(60 - e).expand_as(c)], 1).to(BF16)
    q, sc = torch.full(c.shape, 99, dtype=torch.int8, device="cuda"), torch.empty(len(powers), device="cuda")
    pg.quantization.quantize_gated(x, q, sc, activation="none", max_val=max_val)
    off = (q.double() - c * max_val / 100).abs()
    assert float(off.max()) <= 0.5 + max_val * 2.0 ** -22, off.amax(1).tolist()  # of the scale factor and the product
    most = 100 * torch.exp2(-e[:, 0])
    assert bool(((sc.double() - most / max_val).abs() <= most / max_val * 2.0 ** -22 + 2.0 ** -149).all())


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("act", ["none", "silu", "relu", "gelu", "gelu_tanh"])
def test_rows_with_infinities(n, act):
    """The infinite products are +-max_val, the finite ones 0, the scale
    infinite: the limit of the formula, and no sign is lost."""
    g = gen(n + 1)
    x = randn(g, 3, 2 * n).to(BF16)
    x[1, [3, 5, n - 1]] = 1.0
    x[1, [n + 3, n + 5, 2 * n - 1]] = torch.tensor([float("inf"), float("-inf"), float("inf")], dtype=BF16, device="cuda")
    x[1, 7], x[1, n + 7] = float("inf"), -2.0
    q, sc = torch.full((3, n), 99, dtype=torch.int8, device="cuda"), torch.empty(3, device="cuda")
    pg.quantization.quantize_gated(x, q, sc, activation=act)
    assert sc.isinf().tolist() == [False, True, False] and float(sc[1]) > 0
    want = torch.zeros(n, dtype=torch.int8, device="cuda")
    want[[3, 5, 7, n - 1]] = torch.tensor([127, -127, -127, 127], dtype=torch.int8, device="cuda")
    assert torch.equal(q[1], want)
    assert q[[0, 2]].abs().amax(1).tolist() == [127, 127]


@pytest.mark.parametrize("n", WIDTHS)
def test_rows_with_nan_are_zeros(n):
    x = randn(gen(n + 2), 2, 2 * n).to(BF16)
    x[1, 3], x[1, 9], x[1, n + 9] = float("nan"), 1.0, float("inf")
    q, sc = torch.full((2, n), 99, dtype=torch.int8, device="cuda"), torch.empty(2, device="cuda")
    pg.quantization.quantize_gated(x, q, sc)
    assert sc.isnan().tolist() == [False, True] and not bool(q[1].any()) and bool(q[0].any())


def test_every_index_outside_an_empty_x():
    index = torch.tensor([0, -1, 7], dtype=torch.int32, device="cuda")
    q, sc = torch.full((3, 64), 99, dtype=torch.int8, device="cuda"), torch.full((3,), 9.0, device="cuda")
    pg.quantization.quantize_gated(torch.empty(0, 128, dtype=BF16, device="cuda"), q, sc, row_index=index)
    assert not bool(q.any()) and sc.tolist() == [0.0] * 3
