"""The un-mined layer operators against plain 64-bit implementations.

Tolerances: a result rounded once to a 16-bit type is within half a unit in
the last place of the exact value, plus what the f32 steps before the
rounding can lose: ACC = 2^-20 of the magnitudes that are added up (16 units
of f32; the fast exponential's error grows to about 10 units at the largest
arguments here)."""

import itertools
import math

import pytest
import torch

import pearl_b200 as pg

pytestmark = pytest.mark.gpu

ACC = 2.0 ** -20
# 8, 11 and 24 significant bits
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield
    torch.cuda.synchronize()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def int8(g, *shape):
    return torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)


def within(got, want, slack, dtype):
    """got (16-bit) within half an ulp of want (float64) plus slack."""
    tol = want.abs() * HALF_ULP[dtype] * (1 + 2.0 ** -6) + 2.0 ** -25 + slack
    off = (got.double() - want).abs() - tol
    assert bool((off <= 0).all()), f"worst excess {float(off.max()):.3g} at {int(off.argmax())}"


def act64(name, y):
    return {"none": lambda: y, "relu": lambda: y.clamp(min=0), "silu": lambda: y * torch.sigmoid(y),
            "gelu": lambda: 0.5 * y * torch.special.erfc(-y * math.sqrt(0.5)),
            "gelu_tanh": lambda: 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))}[name]()


# ------------------------------------------------------------------ linear --
def linear64(A, B, sa, sb, bias, act, residual):
    z = (A.double() @ B.double().T) * sa.double()[:, None] * sb.double()
    mag = 1 + z.abs()
    if bias is not None:
        z, mag = z + bias.double(), mag + bias.double().abs()
    y = act64(act, z)
    if residual is not None:
        y, mag = y + residual.double(), mag + residual.double().abs()
    return y, mag * ACC


def linear_case(m, n, k, dtype, act="none", bias=None, residual=False, seed=0):
    g = gen(1000003 * m + 1009 * n + k + seed)
    A, B = int8(g, m, k), int8(g, n, k)
    sa = torch.rand(m, generator=g, device="cuda") + 0.5
    sb = (torch.rand(n, generator=g, device="cuda") + 0.5) / (73 * 73 * math.sqrt(k))
    b = None if bias is None else randn(g, n).to(bias)
    r = randn(g, m, n).to(dtype) if residual else None
    C = torch.full((m, n), float("nan"), dtype=dtype, device="cuda")
    pg.gemm_epilogue(A, B, sa, sb, C, bias=b, activation=act, residual=r)
    want, slack = linear64(A, B, sa, sb, b, act, r)
    within(C, want, slack, dtype)


@pytest.mark.parametrize("m,n,k", [
    (1, 1, 16), (1, 8, 16), (1, 4096, 4096), (2, 7, 48), (7, 129, 112), (8, 64, 128), (16, 4096, 1024), (31, 65, 144),
    (33, 1000, 272), (64, 2048, 14336), (127, 127, 127 * 16), (128, 128, 128), (129, 257, 256), (200, 1001, 1040),
    (256, 4096, 2048), (257, 511, 4096), (300, 4104, 528), (512, 1024, 1024), (1000, 3000, 400), (2500, 2504, 2512)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_sizes(m, n, k, dtype):
    linear_case(m, n, k, dtype, "silu", dtype, True)


# Row tiles of 32, 64 and 128 rows, whole and ragged, K in one, two and four
# ranges of even and uneven length, also in pairs.
@pytest.mark.parametrize("m,n,k", [
    (32, 4096, 1040), (40, 1024, 1040), (64, 1023, 14336), (65, 512, 1280), (97, 1000, 1008), (100, 768, 4112),
    (128, 300, 16384), (129, 1024, 8208), (160, 4096, 8192), (200, 2048, 2048), (300, 304, 304), (333, 2048, 1040),
    (500, 512, 512), (256, 4096, 4224)])
@pytest.mark.parametrize("act,residual", [("none", False), ("gelu", True)])
def test_linear_row_tiles(m, n, k, act, residual):
    linear_case(m, n, k, BF16, act, torch.float32, residual)


@pytest.mark.parametrize("act", list(pg.linear.ACTIVATIONS))
@pytest.mark.parametrize("bias", [None, F32, BF16])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("m,n,k", [(5, 200, 160), (300, 600, 640)])
def test_linear_epilogues(act, bias, residual, m, n, k):
    linear_case(m, n, k, BF16, act, bias, residual)


def test_linear_extreme_integers():
    """-128 everywhere: the largest sums, beyond 2^24, exact before the scales."""
    m, n, k = 40, 72, 14336
    A, B = torch.full((m, k), -128, dtype=torch.int8, device="cuda"), torch.full((n, k), -128, dtype=torch.int8, device="cuda")
    B[:, 1] = 127
    C = torch.empty(m, n, dtype=BF16, device="cuda")
    one = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
    pg.gemm_epilogue(A, B, *one, C)
    assert bool((C.double() == float(torch.tensor((k - 1) * 16384 - 128 * 127, dtype=BF16))).all())


def test_linear_activations_at_large_arguments():
    """Saturated activations stay finite: x for large x, 0 for large -x."""
    A = torch.ones(4, 16, dtype=torch.int8, device="cuda")
    B = torch.ones(8, 16, dtype=torch.int8, device="cuda")
    B[4:] = -1
    sa, sb = torch.full((4,), 1e4, device="cuda"), torch.ones(8, device="cuda")
    for act in ("silu", "gelu", "gelu_tanh", "relu"):
        C = torch.empty(4, 8, dtype=BF16, device="cuda")
        pg.gemm_epilogue(A, B, sa, sb, C, activation=act)
        assert bool((C[:, :4] == torch.tensor(1.6e5, dtype=BF16)).all()) and bool((C[:, 4:] == 0).all()), act


def test_linear_residual_in_place_and_unaligned_output():
    g = gen(3)
    A, B = int8(g, 77, 96), int8(g, 40, 96)
    sa, sb = torch.ones(77, device="cuda"), torch.full((40,), 1e-3, device="cuda")
    base = randn(g, 77, 40).to(BF16)
    want, slack = linear64(A, B, sa, sb, None, "none", base)
    C = base.clone()
    pg.gemm_epilogue(A, B, sa, sb, C, residual=C)
    within(C, want, slack, BF16)
    buf = torch.zeros(77 * 40 + 9, dtype=BF16, device="cuda")
    D = buf[1:1 + 77 * 40].view(77, 40)  # 2-byte aligned rows
    pg.gemm_epilogue(A, B, sa, sb, D, residual=base)
    assert torch.equal(C, D) and bool((buf[:1] == 0).all()) and bool((buf[-8:] == 0).all())


def test_linear_no_rows():
    C = torch.empty(0, 64, dtype=BF16, device="cuda")
    pg.gemm_epilogue(torch.empty(0, 32, dtype=torch.int8, device="cuda"), torch.ones(64, 32, dtype=torch.int8, device="cuda"),
                     torch.empty(0, device="cuda"), torch.ones(64, device="cuda"), C)


def test_linear_offsets_past_32_bits():
    """C with more than 2^31 elements: the last rows and columns are right."""
    m, n, k = 66001, 32776, 16
    g = gen(9)
    A, B = int8(g, m, k), int8(g, n, k)
    sa, sb = torch.rand(m, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda") * 1e-3
    C = torch.empty(m, n, dtype=BF16, device="cuda")
    pg.gemm_epilogue(A, B, sa, sb, C)
    for rows in (slice(0, 64), slice(m - 300, m)):
        want, slack = linear64(A[rows], B, sa[rows], sb, None, "none", None)
        within(C[rows], want, slack, BF16)


def test_linear_on_another_stream_and_in_a_graph():
    g = gen(4)
    A, B = int8(g, 33, 512), int8(g, 520, 512)
    sa, sb = torch.ones(33, device="cuda"), torch.full((520,), 1e-4, device="cuda")
    C, D = (torch.empty(33, 520, dtype=F16, device="cuda") for _ in range(2))
    pg.gemm_epilogue(A, B, sa, sb, C)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pg.gemm_epilogue(A, B, sa, sb, D)
    side.synchronize()
    assert torch.equal(C, D)
    D.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pg.gemm_epilogue(A, B, sa, sb, D)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(C, D)


@pytest.mark.parametrize("m,n,k", [(128, 128, 262144), (600, 512, 131072)])
def test_linear_wait_budget(m, n, k):
    """A budget that the epilogue's wait for its sums outlasts ends the kernel
    with a status, and the next call finds everything as it was."""
    g = gen(m)
    A, B = int8(g, m, k), int8(g, n, k)
    sa, sb = torch.ones(m, device="cuda"), torch.full((n,), 1e-6, device="cuda")
    C = torch.empty(m, n, dtype=BF16, device="cuda")
    sync = torch.zeros(pg.get_host_signal_sync_size(), dtype=torch.int8, device="cuda")
    before = pg.device_waits.set_wait_budget_cycles(64)
    try:
        pg.gemm_epilogue(A, B, sa, sb, C, host_signal_sync=sync)
        torch.cuda.synchronize()
    finally:
        pg.device_waits.set_wait_budget_cycles(before)
    assert pg.get_host_signal_sync_fields(sync)["error"] == pg._lib.PB2_ERR_DEVICE_TIMEOUT
    sync.zero_()
    pg.gemm_epilogue(A, B, sa, sb, C, host_signal_sync=sync)
    torch.cuda.synchronize()
    assert pg.get_host_signal_sync_fields(sync)["error"] == 0
    want, slack = linear64(A, B, sa, sb, None, "none", None)
    within(C, want, slack, BF16)


# ------------------------------------------------------------------ router --
def route(logits, top_k, **kw):
    m = logits.shape[0]
    ids = torch.full((m, top_k), -1, dtype=torch.int32, device="cuda")
    w = torch.full((m, top_k), float("nan"), device="cuda")
    pg.moe.route_tokens(logits, w, ids, **kw)
    return w, ids


def route64(x, top_k, scoring="softmax", bias=None, num_groups=1, topk_groups=1, renormalize=True, scaling=1.0):
    """(choice keys with -inf for experts that take no part, scores) in float64."""
    x = x.double()
    scores = torch.softmax(x, 1) if scoring == "softmax" else torch.sigmoid(x)
    key = x if bias is None else scores + bias.double()
    m, E = x.shape
    if num_groups > 1:
        parts = key.view(m, num_groups, -1).sort(2, descending=True).values
        value = parts[:, :, 0] if bias is None or E == num_groups else parts[:, :, :2].sum(2)
        kept = value.sort(dim=1, descending=True, stable=True).indices[:, :topk_groups]
        part = torch.zeros_like(value, dtype=torch.bool).scatter_(1, kept, True).repeat_interleave(E // num_groups, 1)
        key = torch.where(part, key, -math.inf)
    return key, scores


def weights64(scores, ids, renormalize=True, scaling=1.0):
    w = scores.gather(1, ids.long())
    return (w / w.sum(1, keepdim=True) if renormalize else w) * scaling


SHAPES = [(1, 1, 1, 1, 1), (1, 8, 2, 1, 1), (3, 2, 2, 1, 1), (5, 8, 8, 4, 2 + 2), (9, 16, 3, 4, 2), (33, 31, 5, 1, 1),
          (64, 60, 4, 1, 1), (77, 64, 6, 8, 3), (130, 72, 4, 6, 5), (257, 100, 7, 1, 1), (500, 128, 8, 1, 1),
          (321, 160, 6, 8, 3), (1000, 256, 8, 8, 4), (100, 256, 32, 1, 1), (40, 256, 8, 256, 16), (50, 255, 9, 51, 7)]


@pytest.mark.parametrize("m,E,k,G,kept", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_without_bias(m, E, k, G, kept, dtype, scoring):
    """Logits on a coarse grid, so many tie: the choice is exact, ties included."""
    g = gen(m * 7 + E)
    x = (randn(g, m, E) * 4).round().div(2).to(dtype)
    kw = dict(scoring=scoring, num_groups=G, topk_groups=kept, scaling=1.5)
    w, ids = route(x, k, **kw)
    key, scores = route64(x, k, **kw)
    want = key.sort(dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(ids.long(), want)
    # f32 softmax of <= 256 terms: 2^-24 for every step of the sums and 2^-22 for the exponentials
    torch.testing.assert_close(w.double(), weights64(scores, ids, True, 1.5), rtol=2.0 ** -18, atol=0)


@pytest.mark.parametrize("m,E,k,G,kept", SHAPES)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_with_bias(m, E, k, G, kept, scoring):
    """The choice goes by score + bias in float32: right up to that rounding."""
    g = gen(m * 11 + E)
    x, bias = randn(g, m, E) * 2, randn(g, E) * 0.2
    kw = dict(scoring=scoring, bias=bias, num_groups=G, topk_groups=kept)
    w, ids = route(x, k, renormalize=False, **kw)
    eps = 4e-6  # a few 2^-22 of |score| + |bias|, twice for a group's two best
    if G > 1:  # groups within eps of one another may swap: leave those rows out
        parts = (route64(x, k, scoring, bias)[0]).view(m, G, -1).sort(2, descending=True).values
        value = (parts[:, :, 0] if E == G else parts[:, :, :2].sum(2)).sort(1, descending=True).values
        clear = torch.ones(m, dtype=torch.bool, device="cuda") if kept == G else value[:, kept - 1] - value[:, kept] > eps
        assert float(clear.double().mean()) > 0.9
        x, ids, w, m = x[clear], ids[clear], w[clear], int(clear.sum())
    key, scores = route64(x, k, **kw)
    got = key.gather(1, ids.long())
    assert bool((got > -math.inf).all())
    assert all(len(set(row)) == k for row in ids.tolist())
    assert bool((got[:, :-1] >= got[:, 1:] - eps).all())
    rest = key.scatter(1, ids.long(), -math.inf).amax(1)
    assert bool((rest <= got[:, -1] + eps).all())
    torch.testing.assert_close(w.double(), weights64(scores, ids, False), rtol=2.0 ** -18, atol=0)


def test_route_masked_experts():
    inf, nan = math.inf, math.nan
    low = torch.finfo(F32).min
    x = torch.tensor([[-inf, 1.0, -inf, 2.0], [-inf, -inf, -inf, -inf], [nan, 0.0, nan, -inf], [low, -inf, low, 3.0],
                      [inf, 0.0, inf, 1.0], [low, low, low, low], [-0.0, 0.0, -1.0, 0.0]], device="cuda")
    w, ids = route(x, 3)
    e = math.exp
    assert ids.tolist() == [[3, 1, 0], [0, 1, 2], [1, 0, 2], [3, 0, 2], [0, 2, 3], [0, 1, 2], [0, 1, 3]]
    want = torch.tensor([[1 / (1 + e(-1)), e(-1) / (1 + e(-1)), 0], [0, 0, 0], [1, 0, 0], [1, 0, 0], [0.5, 0.5, 0],
                         [1 / 3] * 3, [1 / 3] * 3], device="cuda")
    torch.testing.assert_close(w, want, rtol=1e-6, atol=0)
    w, ids = route(x, 2, scoring="sigmoid", bias=torch.tensor([0.0, 0.0, 5.0, 0.0], device="cuda"))
    assert ids.tolist() == [[3, 1], [0, 1], [1, 0], [2, 3], [2, 0], [2, 0], [2, 0]]
    assert w[1].tolist() == [0.0, 0.0] and w[2].tolist() == [1.0, 0.0]
    # A masked expert of a kept group still comes before any expert of a dropped one.
    x = torch.tensor([[5.0, -inf, 4.0, 4.0]], device="cuda")
    w, ids = route(x, 2, num_groups=2, topk_groups=1)
    assert ids.tolist() == [[0, 1]] and w.tolist() == [[1.0, 0.0]]
    w, ids = route(x.to(F16), 2, num_groups=2, topk_groups=1, scoring="sigmoid",
                   bias=torch.full((4,), -inf, device="cuda"))
    assert ids.tolist() == [[0, 1]]


# So many tokens that several share a warp.
MANY = [(5001, 1, 1, 1, 1), (6001, 8, 2, 1, 1), (5999, 8, 8, 4, 2 + 2), (9001, 31, 5, 1, 1), (9999, 60, 4, 1, 1), (5003, 64, 6, 8, 3),
        (10007, 72, 4, 6, 5), (12001, 128, 8, 1, 1), (11003, 128, 16, 4, 2), (10001, 100, 12, 1, 1), (10003, 127, 9, 1, 1)]


@pytest.mark.parametrize("m,E,k,G,kept", MANY)
@pytest.mark.parametrize("dtype,scoring", [(F32, "softmax"), (BF16, "sigmoid")])
def test_route_many_tokens(m, E, k, G, kept, dtype, scoring):
    test_route_without_bias(m, E, k, G, kept, dtype, scoring)
    test_route_with_bias(m, E, k, G, kept, scoring)


@pytest.mark.parametrize("E,k,G,kept", [(4, 3, 1, 1), (4, 2, 2, 1), (60, 4, 1, 1), (128, 8, 8, 3), (100, 12, 1, 1)])
@pytest.mark.parametrize("bias", [False, True])
def test_route_does_not_depend_on_the_number_of_tokens(E, k, G, kept, bias):
    """A token's experts are the same among many as among few, with masked
    experts, ties, infinities and NaN; its weights up to the order of sums."""
    g = gen(E + k)
    x = (randn(g, 12000, E) * 2).round()
    x[torch.rand(12000, E, generator=g, device="cuda") < 0.3] = -math.inf
    x[5::17, 1] = math.nan
    x[3::19] = -math.inf
    kw = dict(num_groups=G, topk_groups=kept, bias=(randn(g, E) * 0.2).round(decimals=1) if bias else None, scoring="sigmoid")
    w, ids = route(x, k, **kw)
    for at in (0, 4000, 11500):
        w2, ids2 = route(x[at:at + 500].contiguous(), k, **kw)
        assert torch.equal(ids[at:at + 500], ids2)
        torch.testing.assert_close(w[at:at + 500], w2, rtol=2.0 ** -20, atol=0)


def test_route_no_tokens():
    w, ids = route(torch.empty(0, 8, device="cuda"), 2)
    assert w.shape == (0, 2)


# ------------------------------------------------------- gated quantization --
def hadamard64(v, block):
    if not block:
        return v
    m, n = v.shape
    H = torch.ones(1, 1, dtype=torch.float64, device=v.device)
    while H.shape[0] < block:
        H = torch.cat([torch.cat([H, H], 1), torch.cat([H, -H], 1)], 0)
    y = (v.view(m, n // block, block) @ H.T) / math.sqrt(block)
    y[:, :, 0] = -y[:, :, 0]
    return y.reshape(m, n)


@pytest.mark.parametrize("rows,n", [(1, 8), (3, 1360), (5, 2048), (4, 2056), (2, 8192), (3, 14336), (2, 16384), (2, 16392), (65, 256)])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("act,smooth,block,max_val", [("silu", False, 0, 127), ("gelu", True, 8, 63), ("gelu_tanh", True, 0, 127),
                                                      ("none", False, 8, 127), ("relu", False, 0, 1)])
def test_quantize_gated(rows, n, dtype, act, smooth, block, max_val):
    g = gen(rows * n)
    x = (randn(g, rows, 2 * n) * 2).to(dtype)
    x[rows // 2, :n] = 0  # a row whose products are all zero (every act(0) = 0)
    s = torch.rand(n, generator=g, device="cuda") + 0.5 if smooth else None
    index = torch.randint(0, rows, (rows + 3,), generator=g, device="cuda", dtype=torch.int32)
    index[0], index[-1], index[1] = rows, -1, rows // 2
    q = torch.full((rows + 3, n), 99, dtype=torch.int8, device="cuda")
    sc = torch.full((rows + 3, 1), -1.0, device="cuda")
    pg.quantization.quantize_gated(x, q, sc, activation=act, row_index=index, smooth_scale=s, max_val=max_val, block_size=block)
    xd = x.double()
    pre = act64(act, xd[:, :n]) * xd[:, n:]
    v = hadamard64(pre, block) * (1 if s is None else s.double())
    # f32 products to ACC each; the transform adds `block` of them
    slack = 2 * ACC * (pre.abs().amax(1) * math.sqrt(max(block, 1)) * 1.5 + v.abs().amax(1))
    for i, src in enumerate(index.tolist()):
        if not 0 <= src < rows or not bool(v[src].any()):
            assert not bool(q[i].any()) and float(sc[i]) == 0
            continue
        most = float(v[src].abs().max())
        assert abs(float(sc[i]) - most / max_val) <= float(slack[src]) / max_val + most / max_val * 2.0 ** -22
        off = (q[i].double() - v[src] * max_val / most).abs().max()
        assert float(off) <= 0.5 + 2 * max_val * float(slack[src]) / most
        assert int(q[i].abs().max()) == max_val
    # without an index: the same bytes for the same rows
    q2, sc2 = torch.empty(rows, n, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    pg.quantization.quantize_gated(x, q2, sc2, activation=act, smooth_scale=s, max_val=max_val, block_size=block)
    live = (index >= 0) & (index < rows)
    assert torch.equal(q[live], q2[index[live].long()]) and torch.equal(sc[live, 0], sc2[index[live].long()])


@pytest.mark.parametrize("n", [64, 1360, 4096, 20000])  # a warp, a block, a block in registers, in two passes
@pytest.mark.parametrize("at", ["gate", "up"])
def test_quantize_gated_keeps_nan_and_infinity(n, at):
    g = gen(n)
    x = randn(g, 9, 2 * n).to(BF16)
    clean = x.clone()
    column = n - 3 if at == "gate" else 2 * n - 3
    x[2, column] = float("nan")
    x[7, column] = float("inf")
    clean[7, column % n] = clean[7, n + column % n] = 1.0  # a product of the infinity that is not NaN
    x[7, column % n if at == "up" else n + column % n] = 1.0
    q, sc, q2, sc2 = (torch.empty(s, dtype=t, device="cuda") for _ in range(2) for s, t in (((9, n), torch.int8), ((9,), F32)))
    pg.quantization.quantize_gated(x, q, sc)
    pg.quantization.quantize_gated(clean, q2, sc2)
    assert sc.isnan().tolist() == [r == 2 for r in range(9)] and sc.isinf().tolist() == [r == 7 for r in range(9)]
    others = [0, 1, 3, 4, 5, 6, 8]
    assert torch.equal(q[others], q2[others]) and torch.equal(sc[others], sc2[others])


# ------------------------------------------------------- experts' products --
def routing(g, counts, seed_order=True):
    """(expert ids of the slots shuffled, slot_indices, offsets) with these rows per expert."""
    ids = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), torch.tensor(counts, device="cuda"))
    ids = ids[torch.randperm(len(ids), generator=g, device="cuda")]
    return ids, ids.sort(stable=True).indices.to(torch.int32), torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)


COUNTS = [[1], [0, 1, 0], [5, 0, 3], [0, 0, 130, 7, 0], [128, 128], [129, 1, 255, 0, 257, 31], [300, 0, 0, 700], [1] * 60,
          [3, 17, 0, 64, 33] * 12 + [2], [0] * 255 + [9], [2] * 256, [1500, 20, 0, 900]]


@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: f"{len(c)}x{sum(c)}")
@pytest.mark.parametrize("n,k,dtype", [(8, 16, BF16), (264, 144, F16), (129, 272, BF16), (1000, 1360, F16), (200, 400, F32),
                                       (131, 96, F32)])
def test_gemm_grouped(counts, n, k, dtype):
    g = gen(sum(counts) * 31 + n)
    E, m = len(counts), sum(counts)
    _, slot, ends = routing(g, counts)
    A, B = int8(g, m, k), int8(g, E, n, k)
    sa = torch.rand(m, generator=g, device="cuda") + 0.5
    sb = (torch.rand(E, n, generator=g, device="cuda") + 0.5) / (73 * 73 * math.sqrt(k))
    want = torch.empty(m, n, dtype=torch.float64, device="cuda")
    for e, (lo, hi) in enumerate(itertools.pairwise([0] + ends.tolist())):
        want[lo:hi] = (A[lo:hi].double() @ B[e].double().T) * sa[lo:hi, None].double() * sb[e].double()
    C = torch.full((m, n), float("nan"), dtype=dtype, device="cuda")
    pg.moe.gemm_grouped(A, B, sa, sb, C, ends)
    within(C, want, ACC * want.abs(), dtype)
    # scattered into a larger C; an index outside it is skipped, the other rows untouched
    D = torch.full((m + 4, n), 7.0, dtype=dtype, device="cuda")
    index = slot + 2
    if m > 3:
        index[1], index[2] = -5, m + 4
    pg.moe.gemm_grouped(A, B, sa, sb, D, ends, c_row_index=index)
    expect = torch.full((m + 4, n), 7.0, dtype=dtype, device="cuda")
    ok = (index >= 0) & (index < m + 4)
    expect[index[ok].long()] = C[ok]
    assert torch.equal(D, expect)


def test_gemm_grouped_rows_past_the_last_expert_stay():
    g = gen(5)
    A, B = int8(g, 50, 64), int8(g, 3, 24, 64)
    ends = torch.tensor([10, 10, 30], dtype=torch.int32, device="cuda")
    C = torch.full((50, 24), 7.0, dtype=BF16, device="cuda")
    pg.moe.gemm_grouped(A, B, torch.ones(50, device="cuda"), torch.ones(3, 24, device="cuda"), C, ends)
    assert bool((C[30:] == 7).all()) and not bool((C[:30] == 7).all())


@pytest.mark.parametrize("m,k,n", [(1, 1, 8), (1, 2, 4096), (5, 3, 17), (33, 8, 264), (7, 32, 1001)])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("slots_f32", [False, True])
@pytest.mark.parametrize("residual", [False, True])
def test_combine_slots(m, k, n, dtype, slots_f32, residual):
    g = gen(m + k + n)
    y = randn(g, m * k, n).to(F32 if slots_f32 else dtype)
    w = torch.rand(m, k, generator=g, device="cuda")
    if k > 1:
        w[m // 2, 0] = 0
        y[(m // 2) * k] = float("nan")  # weight 0: not read
    r = randn(g, m, n).to(dtype) if residual else None
    out = torch.empty(m, n, dtype=dtype, device="cuda")
    pg.moe.combine_slots(y, w, out, residual=r)
    terms = (torch.where(w[:, :, None] == 0, 0.0, y.view(m, k, n).double())) * w.double()[:, :, None]
    want, mag = terms.sum(1), terms.abs().sum(1)
    if residual:
        want, mag = want + r.double(), mag + r.double().abs()
    within(out, want, (k + 1) * 2.0 ** -23 * mag, dtype)
    if residual:
        pg.moe.combine_slots(y, w, r, residual=r)
        assert torch.equal(r, out)


@pytest.mark.parametrize("m,E,k,hidden,inner,dtype", [
    (1, 4, 1, 64, 32, BF16), (1, 8, 2, 4096, 1024, BF16), (3, 60, 4, 2040, 1360, F16), (40, 16, 8, 136, 272, F16),
    (300, 8, 2, 1000, 528, BF16), (700, 4, 3, 264, 2048, BF16),
    (1500, 8, 6, 1024, 64, F16)])
@pytest.mark.parametrize("residual,smooth", [(False, False), (True, True)])
def test_gated_experts_is_its_three_steps(m, E, k, hidden, inner, dtype, residual, smooth):
    g = gen(m + hidden)
    w, ids = route(randn(g, m, E), k)
    slots = m * k
    data, slot, ends = (torch.empty(s, dtype=torch.int32, device="cuda") for s in (slots, slots, E))
    scratch = torch.empty(pg.moe.get_build_routing_data_scratchpad_bytes(slots), dtype=torch.uint8, device="cuda")
    pg.moe.build_routing_data(ids, data, slot, ends, scratch, E)
    x = randn(g, slots, 2 * inner).to(dtype)
    W, ws = int8(g, E, hidden, inner), (torch.rand(E, hidden, generator=g, device="cuda") + 0.5) * 1e-3
    r = randn(g, m, hidden).to(dtype) if residual else None
    s = torch.rand(inner, generator=g, device="cuda") + 0.5 if smooth else None
    out = torch.empty(m, hidden, dtype=dtype, device="cuda")
    pg.moe.gated_experts(x, W, ws, out, slot, ends, w, residual=r, smooth_scale=s)
    q, sc = torch.empty(slots, inner, dtype=torch.int8, device="cuda"), torch.empty(slots, device="cuda")
    pg.quantization.quantize_gated(x, q, sc, row_index=slot, smooth_scale=s)
    kept = F32 if slots * hidden * 4 <= 32 << 20 else dtype
    y = torch.empty(slots, hidden, dtype=kept, device="cuda")
    pg.moe.gemm_grouped(q, W, sc, ws, y, ends, c_row_index=slot)
    want = torch.empty_like(out)
    pg.moe.combine_slots(y, w, want, residual=r)
    assert torch.equal(out, want)
    # and the whole of it against the formula with these quantized rows
    full = torch.zeros(slots, hidden, dtype=torch.float64, device="cuda")
    for e, (lo, hi) in enumerate(itertools.pairwise([0] + ends.tolist())):
        full[slot[lo:hi].long()] = (q[lo:hi].double() @ W[e].double().T) * sc[lo:hi, None].double() * ws[e].double()
    terms = full.view(m, k, hidden) * w.double()[:, :, None]
    total, mag = terms.sum(1), terms.abs().sum(1)
    if residual:
        total, mag = total + r.double(), mag + r.double().abs()
    # each slot's product is rounded to the kept type before the sum
    within(out, total, mag * (HALF_ULP[kept] * 1.01 + 2.0 ** -19) + k * 2.0 ** -25, dtype)


@pytest.mark.parametrize("m,E,k,hidden,inner,dtype", [
    (1, 4, 1, 64, 32, BF16), (1, 8, 2, 4096, 2048, F16), (3, 60, 4, 2041, 1360, F16), (300, 8, 2, 1000, 528, BF16),
    (700, 200, 8, 136, 272, F16), (1500, 8, 6, 1024, 64, BF16)])
@pytest.mark.parametrize("elsewhere", ["some", "all"])
@pytest.mark.parametrize("residual", [False, True])
def test_gated_experts_slots_of_no_expert_count_nothing(m, E, k, hidden, inner, dtype, elsewhere, residual):
    """Ids outside 0..E-1 (an expert that another GPU holds) sort past the last
    expert's end; whatever the workspace and those rows of x hold is not used."""
    g = gen(m + hidden + 1)
    w, ids = route(randn(g, m, E), k)
    away = torch.rand(m, k, generator=g, device="cuda") < 0.6 if elsewhere == "some" else torch.ones(m, k, device="cuda") > 0
    ids = torch.where(away, torch.where(torch.rand(m, k, generator=g, device="cuda") < 0.5, -1, 255), ids).int()
    slots = m * k
    data, slot, ends = (torch.empty(s, dtype=torch.int32, device="cuda") for s in (slots, slots, E))
    scratch = torch.empty(pg.moe.get_build_routing_data_scratchpad_bytes(slots), dtype=torch.uint8, device="cuda")
    pg.moe.build_routing_data(ids, data, slot, ends, scratch, E)
    x = randn(g, slots, 2 * inner).to(dtype)
    W, ws = int8(g, E, hidden, inner), (torch.rand(E, hidden, generator=g, device="cuda") + 0.5) * 1e-3
    r = randn(g, m, hidden).to(dtype) if residual else None
    space = torch.full((pg.moe.get_gated_experts_workspace_bytes(slots, inner, hidden),), 255, dtype=torch.uint8, device="cuda")
    out, want = (torch.empty(m, hidden, dtype=dtype, device="cuda") for _ in range(2))
    dirty = torch.where(away.view(-1, 1), float("nan"), x)
    pg.moe.gated_experts(dirty, W, ws, out, slot, ends, w, residual=r, workspace=space)
    # the same slots with an expert of their own (any) and no weight
    home = torch.where(away, 0, ids)
    pg.moe.build_routing_data(home, data, slot, ends, scratch, E)
    pg.moe.gated_experts(x, W, ws, want, slot, ends, torch.where(away, 0.0, w), residual=r)
    assert torch.equal(out, want)


def test_gated_experts_refuses_workspaces_without_their_bytes():
    x, w, ws = torch.zeros(8, 64, dtype=BF16, device="cuda"), torch.zeros(2, 8, 32, dtype=torch.int8, device="cuda"), torch.ones(2, 8, device="cuda")
    out, weights = torch.zeros(4, 8, dtype=BF16, device="cuda"), torch.ones(4, 2, device="cuda")
    slot, ends = torch.arange(8, dtype=torch.int32, device="cuda"), torch.tensor([4, 8], dtype=torch.int32, device="cuda")
    need = pg.moe.get_gated_experts_workspace_bytes(8, 32, 8)
    one = torch.zeros(1, dtype=torch.uint8, device="cuda")
    for space in (one.expand(need), torch.zeros(need - 1, dtype=torch.uint8, device="cuda"),
                  torch.zeros(need, dtype=torch.int8, device="cuda"), torch.zeros(need, dtype=torch.uint8)):
        with pytest.raises(RuntimeError, match="workspace must be"):
            pg.moe.gated_experts(x, w, ws, out, slot, ends, weights, workspace=space)
    word = torch.zeros(1, dtype=torch.int8, device="cuda")
    for sync in (word.expand(pg._lib.HOST_SIGNAL_SYNC_SIZE), torch.zeros(pg._lib.HOST_SIGNAL_SYNC_SIZE, dtype=torch.int8), word):
        with pytest.raises(RuntimeError, match="host_signal_sync must be"):
            pg.moe.gated_experts(x, w, ws, out, slot, ends, weights, host_signal_sync=sync)


@pytest.mark.parametrize("m,E,k,hidden,inner", [(8, 8, 2, 4096, 2048), (2, 8, 2, 512, 4096), (900, 64, 4, 512, 768), (1500, 4, 2, 1024, 512)])
def test_gated_experts_back_to_back(m, E, k, hidden, inner):
    """Calls queued one behind the other, each with inputs written just before
    it on the same stream: the product's early loads take none of them."""
    g = gen(m + inner)
    w, ids = route(randn(g, m, E), k)
    slots = m * k
    data, slot, ends = (torch.empty(s, dtype=torch.int32, device="cuda") for s in (slots, slots, E))
    scratch = torch.empty(pg.moe.get_build_routing_data_scratchpad_bytes(slots), dtype=torch.uint8, device="cuda")
    pg.moe.build_routing_data(ids, data, slot, ends, scratch, E)
    W, ws = int8(g, E, hidden, inner), (torch.rand(E, hidden, generator=g, device="cuda") + 0.5) * 1e-3
    xs = [randn(g, slots, 2 * inner).to(BF16) for _ in range(12)]
    x = torch.empty_like(xs[0])
    space = torch.empty(pg.moe.get_gated_experts_workspace_bytes(slots, inner, hidden), dtype=torch.uint8, device="cuda")
    outs = [torch.empty(m, hidden, dtype=BF16, device="cuda") for _ in xs]
    torch.cuda.synchronize()
    for src, out in zip(xs, outs):
        x.copy_(src)
        pg.moe.gated_experts(x, W, ws, out, slot, ends, w, workspace=space)
    torch.cuda.synchronize()
    for src, out in zip(xs, outs):
        q, sc = torch.empty(slots, inner, dtype=torch.int8, device="cuda"), torch.empty(slots, device="cuda")
        y, want = torch.empty(slots, hidden, dtype=F32, device="cuda"), torch.empty_like(out)
        for step in (lambda: pg.quantization.quantize_gated(src, q, sc, row_index=slot),
                     lambda: pg.moe.gemm_grouped(q, W, sc, ws, y, ends, c_row_index=slot),
                     lambda: pg.moe.combine_slots(y, w, want)):
            step()
            torch.cuda.synchronize()
        assert torch.equal(out, want)
