"""gated_experts and gemm_grouped where the sizes change how they work: slot
products beyond 32 MB, values beyond a 16-bit type's range, K in four ranges,
and calls that follow one another on new weights and a new routing."""

import itertools
import math

import pytest
import torch

import pearl_b200 as pg
from tests.test_gpu_layer_ops import ACC, BF16, F16, F32, gen, int8, randn, route, within

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield
    torch.cuda.synchronize()


def order(ids, E):
    """(slot_indices, routing_offsets) of these ids."""
    slots = ids.numel()
    data, slot, ends = (torch.empty(s, dtype=torch.int32, device="cuda") for s in (slots, slots, E))
    scratch = torch.empty(pg.moe.get_build_routing_data_scratchpad_bytes(slots), dtype=torch.uint8, device="cuda")
    pg.moe.build_routing_data(ids, data, slot, ends, scratch, E)
    return slot, ends


def products64(x, W, ws, slot, ends):
    """Every slot's product in float64 from its quantized row, zeros where no
    expert has the slot."""
    slots, inner = x.shape[0], W.shape[2]
    q, sc = torch.empty(slots, inner, dtype=torch.int8, device="cuda"), torch.empty(slots, device="cuda")
    pg.quantization.quantize_gated(x, q, sc, row_index=slot)
    y = torch.zeros(slots, W.shape[1], dtype=torch.float64, device="cuda")
    for e, (lo, hi) in enumerate(itertools.pairwise([0] + ends.tolist())):
        y[slot[lo:hi].long()] = (q[lo:hi].double() @ W[e].double().T) * sc[lo:hi, None].double() * ws[e].double()
    return y


def run(x, W, ws, slot, ends, w, residual=None):
    """The call with a workspace of exactly its bytes, full of NaN; with its
    own workspace the result is the same."""
    slots, inner, hidden = x.shape[0], W.shape[2], W.shape[1]
    space = torch.full((pg.moe.get_gated_experts_workspace_bytes(slots, inner, hidden),), 255, dtype=torch.uint8, device="cuda")
    out = torch.empty(w.shape[0], hidden, dtype=x.dtype, device="cuda")
    pg.moe.gated_experts(x, W, ws, out, slot, ends, w, residual=residual, workspace=space)
    again = torch.empty_like(out)
    pg.moe.gated_experts(x, W, ws, again, slot, ends, w, residual=residual)
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))
    return out


# Even and odd numbers of columns, whole and ragged tiles, many slots of few columns.
LARGE = [(1025, 8, 2, 4096, 64), (2100, 8, 2, 2056, 64), (1100, 64, 8, 1001, 48), (70000, 4, 2, 72, 32), (1100000, 4, 1, 8, 16),
         (4200000, 2, 2, 1, 16)]


@pytest.mark.parametrize("m,E,k,hidden,inner", LARGE)
@pytest.mark.parametrize("residual", [False, True])
def test_slot_products_beyond_32_mb_are_rounded_once(m, E, k, hidden, inner, residual):
    """bf16: the result is the formula's but for one rounding, and a token's
    does not depend on how many others are in the call."""
    assert m * k * hidden * 4 > 32 << 20
    g = gen(m + hidden)
    w, ids = route(randn(g, m, E), k)
    slot, ends = order(ids, E)
    x = randn(g, m * k, 2 * inner).to(BF16)
    W, ws = int8(g, E, hidden, inner), (torch.rand(E, hidden, generator=g, device="cuda") + 0.5) * 1e-3
    r = randn(g, m, hidden).to(BF16) if residual else None
    out = run(x, W, ws, slot, ends, w, r)
    terms = products64(x, W, ws, slot, ends).view(m, k, hidden) * w.double()[:, :, None]
    total, mag = terms.sum(1), terms.abs().sum(1)
    if residual:
        total, mag = total + r.double(), mag + r.double().abs()
    # two roundings of a product, one a term and one for the residual, in f32
    within(out, total, (k + 4) * 2.0 ** -24 * mag, BF16)
    few = 50
    slot, ends = order(ids[:few].contiguous(), E)
    small = run(x[:few * k].contiguous(), W, ws, slot, ends, w[:few].contiguous(), r[:few].contiguous() if residual else None)
    assert torch.equal(out[:few], small)


@pytest.mark.parametrize("m,E,k,hidden,inner", [(40, 8, 2, 2056, 64), (2100, 8, 2, 2056, 64), (1100, 64, 8, 1001, 48)])
def test_f16_slot_products_beyond_its_range(m, E, k, hidden, inner):
    """Products of 10^5 and more whose weighted sum f16 does hold."""
    g = gen(m + inner)
    w, ids = route(randn(g, m, E), k, scaling=0.05)
    slot, ends = order(ids, E)
    x = randn(g, m * k, 2 * inner).to(F16)
    W, ws = int8(g, E, hidden, inner), (torch.rand(E, hidden, generator=g, device="cuda") + 0.5) * 150
    out = run(x, W, ws, slot, ends, w)
    y = products64(x, W, ws, slot, ends)
    terms = y.view(m, k, hidden) * w.double()[:, :, None]
    total, mag = terms.sum(1), terms.abs().sum(1)
    assert float(y.abs().max()) > 2 * 65504 and float(total.abs().max()) < 60000
    # at most one rounding of each product to f16's eleven bits before the sum
    within(out, total, mag * (2.0 ** -11 * 1.01 + (k + 4) * 2.0 ** -24) + k * 2.0 ** -25, F16)


@pytest.mark.parametrize("counts", [[1], [1, 1], [0, 3, 40], [9, 0, 0, 2]], ids=str)
@pytest.mark.parametrize("n,k,dtype", [(200, 4096, BF16), (129, 2064, F32), (8, 14336, F16)])
def test_gemm_grouped_with_k_in_four_ranges(counts, n, k, dtype):
    g = gen(sum(counts) + n)
    E, m = len(counts), sum(counts)
    ends = torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)
    A, B = int8(g, m, k), int8(g, E, n, k)
    sa = torch.rand(m, generator=g, device="cuda") + 0.5
    sb = (torch.rand(E, n, generator=g, device="cuda") + 0.5) / (73 * 73 * math.sqrt(k))
    want = torch.empty(m, n, dtype=torch.float64, device="cuda")
    for e, (lo, hi) in enumerate(itertools.pairwise([0] + ends.tolist())):
        want[lo:hi] = (A[lo:hi].double() @ B[e].double().T) * sa[lo:hi, None].double() * sb[e].double()
    C = torch.full((m, n), float("nan"), dtype=dtype, device="cuda")
    pg.moe.gemm_grouped(A, B, sa, sb, C, ends)
    within(C, want, ACC * want.abs(), dtype)


@pytest.mark.parametrize("m,E,k,hidden,inner", [(8, 8, 2, 4096, 2048), (2, 8, 2, 512, 4096), (900, 64, 4, 512, 768),
                                                (2100, 8, 2, 2056, 64)])
def test_calls_that_follow_one_another_on_new_weights_and_routings(m, E, k, hidden, inner):
    """Everything a call reads is written just before it on the same stream,
    into the same tensors as before: ids and their order, weights, scales,
    rows.  Some slots have no expert."""
    g = gen(m + inner)
    calls = []
    for _ in range(8):
        w, ids = route(randn(g, m, E) * 3, k)
        ids = torch.where(torch.rand(m, k, generator=g, device="cuda") < 0.2, -1, ids).int()
        calls.append((ids, w, randn(g, m * k, 2 * inner).to(BF16), int8(g, E, hidden, inner),
                      (torch.rand(E, hidden, generator=g, device="cuda") + 0.5) * 1e-3))
    slots = m * k
    now = [torch.empty_like(t) for t in calls[0]]
    data, slot, ends = (torch.empty(s, dtype=torch.int32, device="cuda") for s in (slots, slots, E))
    scratch = torch.empty(pg.moe.get_build_routing_data_scratchpad_bytes(slots), dtype=torch.uint8, device="cuda")
    space = torch.empty(pg.moe.get_gated_experts_workspace_bytes(slots, inner, hidden), dtype=torch.uint8, device="cuda")
    outs = [torch.empty(m, hidden, dtype=BF16, device="cuda") for _ in calls]
    torch.cuda.synchronize()
    for new, out in zip(calls, outs):
        for to, src in zip(reversed(now), reversed(new)):
            to.copy_(src)
        ids, w, x, W, ws = now
        pg.moe.build_routing_data(ids, data, slot, ends, scratch, E)
        pg.moe.gated_experts(x, W, ws, out, slot, ends, w, workspace=space)
    torch.cuda.synchronize()
    for (ids, w, x, W, ws), out in zip(calls, outs):
        at, until = order(ids, E)
        terms = products64(x, W, ws, at, until).view(m, k, hidden) * w.double()[:, :, None]
        within(out, terms.sum(1), (k + 4) * 2.0 ** -24 * terms.abs().sum(1), BF16)
