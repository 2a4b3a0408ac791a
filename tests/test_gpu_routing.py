"""The router's scores far below the top logit, and routing orders of ids
outside the experts."""

import pytest
import torch

import pearl_b200 as pg
from tests.test_gpu_layer_ops import BF16, F32, gen, int8, randn, route, route64, weights64

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield
    torch.cuda.synchronize()


@pytest.mark.parametrize("m,E,k", [(300, 8, 8), (300, 60, 32), (300, 256, 32), (9001, 31, 8), (12001, 128, 8)])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("bias", [False, True])
def test_softmax_weights_far_below_the_top(m, E, k, renormalize, bias):
    """Logits down to 80 below the top, on a grid where differences are exact:
    a weight is within 2 ulps of f32 for the exponential, 16 half ulps for
    the sum of up to 256 terms, two divisions and the renormalized sum."""
    g = gen(m + E)
    x = (torch.rand(m, E, generator=g, device="cuda") * -80 * 8).round() / 8
    b = torch.linspace(0, 0.5, E, device="cuda") if bias else None
    w, ids = route(x, k, bias=b, renormalize=renormalize)
    _, scores = route64(x, k)
    want = weights64(scores, ids, renormalize)
    torch.testing.assert_close(w.double(), want, rtol=2.0 ** -19, atol=2.0 ** -126)


@pytest.mark.parametrize("E", [1, 8, 64, 255, 256])
@pytest.mark.parametrize("m,k", [(1, 1), (777, 4), (9000, 2)])
def test_ids_outside_the_experts_sort_past_them(m, k, E):
    """Whatever an id is, it counts for no expert but its own."""
    g = gen(m + E)
    strange = torch.tensor([-1, 256, 300, -256, 511, 1 << 20, -(1 << 31), (1 << 31) - 1, E, E + 256], device="cuda")
    ids = torch.randint(0, E, (m, k), generator=g, device="cuda")
    pick = torch.randint(0, len(strange), (m, k), generator=g, device="cuda")
    ids = torch.where(torch.rand(m, k, generator=g, device="cuda") < 0.4, strange[pick], ids).int()
    slots = m * k
    data, slot, ends = (torch.full((s,), -7, dtype=torch.int32, device="cuda") for s in (slots, slots, E))
    scratch = torch.empty(pg.moe.get_build_routing_data_scratchpad_bytes(slots), dtype=torch.uint8, device="cuda")
    pg.moe.build_routing_data(ids, data, slot, ends, scratch, E)
    flat = ids.view(-1).long()
    inside = (flat >= 0) & (flat < E)
    want = torch.where(inside, flat, 1 << 40).sort(stable=True).indices
    n = int(inside.sum())
    assert torch.equal(ends.long(), torch.bincount(flat[inside], minlength=E).cumsum(0))
    assert torch.equal(slot[:n].long(), want[:n]) and torch.equal(slot[n:].long().sort().values, want[n:].sort().values)
    assert torch.equal(data.long(), slot.long() // k)


@pytest.mark.parametrize("E", [64, 256])
def test_gated_experts_adds_nothing_for_strange_ids(E):
    m, k, hidden, inner = 33, 4, 136, 64
    g = gen(E)
    w, ids = route(randn(g, m, E), k)
    away = torch.rand(m, k, generator=g, device="cuda") < 0.5
    strange = torch.where(away, torch.where(torch.rand(m, k, generator=g, device="cuda") < 0.5, -1, ids + 256), ids).int()
    x = randn(g, m * k, 2 * inner).to(BF16)
    W, ws = int8(g, E, hidden, inner), (torch.rand(E, hidden, generator=g, device="cuda") + 0.5) * 1e-3
    outs = []
    for use, weights in ((strange, w), (ids, torch.where(away, 0.0, w))):
        slots = m * k
        data, slot, ends = (torch.empty(s, dtype=torch.int32, device="cuda") for s in (slots, slots, E))
        scratch = torch.empty(pg.moe.get_build_routing_data_scratchpad_bytes(slots), dtype=torch.uint8, device="cuda")
        pg.moe.build_routing_data(use, data, slot, ends, scratch, E)
        outs.append(torch.empty(m, hidden, dtype=BF16, device="cuda"))
        pg.moe.gated_experts(x, W, ws, outs[-1], slot, ends, weights)
    assert torch.equal(*outs)
