"""The layer operators together as a layer uses them: moe_layer (routing,
first product, gated second half, combination) and PearlLinear.apply_fused.

The bounds on the whole layer are those of its quantization: rounding a row
of n normal values to steps of max / 127 leaves a relative error of about
(max / rms) / (127 sqrt 12): 1% for the input (max / rms up to 4.5), 3% for
products of two normals (up to 13), twice as much in 7 bits."""

import math

import pytest
import torch

import pearl_b200 as pg
from pearl_b200 import miner as MN

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield
    torch.cuda.synchronize()


def layer(seed, m, E, K, inner, dtype=torch.bfloat16, limit=127):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    i8 = lambda *s: (r(*s) * limit / 4).round().clamp(-limit, limit).to(torch.int8)  # noqa: E731
    x, logits = r(m, K).to(dtype), r(m, E)
    w1, w2 = i8(E, 2 * inner, K), i8(E, K, inner)
    s1 = (torch.rand(E, 2 * inner, generator=g, device="cuda") + 0.5) * 4 / (limit * math.sqrt(K))
    s2 = (torch.rand(E, K, generator=g, device="cuda") + 0.5) * 4 / (limit * math.sqrt(inner))
    return x, logits, w1, s1, w2, s2, r(m, K).to(dtype)


def exact(x, logits, w1, s1, w2, s2, top_k, residual):
    x, out = x.double(), residual.double().clone()
    p = torch.softmax(logits.double(), 1)
    val, ids = p.sort(dim=1, descending=True, stable=True)
    val, ids = val[:, :top_k] / val[:, :top_k].sum(1, keepdim=True), ids[:, :top_k]
    for e in range(w1.shape[0]):
        t, j = (ids == e).nonzero(as_tuple=True)
        h = (x[t] @ w1[e].double().T) * s1[e].double()
        n = h.shape[1] // 2
        y = (h[:, :n] * torch.sigmoid(h[:, :n]) * h[:, n:]) @ w2[e].double().T * s2[e].double()
        out.index_add_(0, t, y * val[t, j, None])
    return out


@pytest.mark.parametrize("m,E,K,inner,top_k", [(1, 8, 512, 1024, 2), (7, 16, 272, 144, 4), (300, 8, 1024, 512, 2),
                                               (513, 64, 512, 256, 6)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_moe_layer(m, E, K, inner, top_k, dtype):
    x, logits, w1, s1, w2, s2, res = layer(m + E, m, E, K, inner, dtype)
    out, mined = MN.moe_layer(x, logits, w1, s1, w2, s2, top_k, residual=res)
    assert mined is None and out.dtype is dtype
    want = exact(x, logits, w1, s1, w2, s2, top_k, res)
    moved = (want - res.double()).norm()
    assert float((out.double() - want).norm() / moved) < 0.05 + 2.0 ** -8 * float(want.norm() / moved)


def test_moe_layer_is_its_operators():
    m, E, K, inner, top_k = 65, 16, 512, 256, 4
    x, logits, w1, s1, w2, s2, res = layer(3, m, E, K, inner)
    bias = torch.linspace(-0.1, 0.1, E, device="cuda")
    kw = dict(scoring="sigmoid", bias=bias, num_groups=4, topk_groups=2, scaling=2.5)
    out, _ = MN.moe_layer(x, logits, w1, s1, w2, s2, top_k, residual=res, **kw)
    ids, w = torch.empty(m, top_k, dtype=torch.int32, device="cuda"), torch.empty(m, top_k, device="cuda")
    pg.moe.route_tokens(logits, w, ids, **kw)
    xq, xs, _ = MN.quant_8bit(x)
    order = ids.view(-1).long().sort(stable=True)
    ends = torch.bincount(order.values, minlength=E).cumsum(0).to(torch.int32)
    slot = order.indices.to(torch.int32)
    tok = order.indices // top_k
    h = torch.empty(m * top_k, 2 * inner, dtype=x.dtype, device="cuda")
    pg.moe.gemm_grouped(xq[tok], w1, xs.squeeze(-1)[tok], s1, h, ends, c_row_index=slot)
    want = torch.empty_like(res)
    pg.moe.gated_experts(h, w2, s2, want, slot, ends, w, residual=res)
    assert torch.equal(out, want)


def test_moe_layer_in_a_graph():
    """The whole un-mined layer as one CUDA graph, replayed on new inputs."""
    x, logits, w1, s1, w2, s2, res = layer(4, 8, 8, 512, 512)
    run = lambda: MN.moe_layer(x, logits, w1, s1, w2, s2, 2, residual=res)[0]  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for seed in (5, 6):
        x2, logits2, *_ = layer(seed, 8, 8, 512, 512)
        x.copy_(x2)
        logits.copy_(logits2)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, run())


def test_moe_layer_mined():
    """With a job and a large enough batch the first product is mined: the
    same layer within 7-bit quantization, and every expert's mining product."""
    m, E, K, inner, top_k = 384, 4, 512, 256, 2
    x, logits, w1, s1, w2, s2, res = layer(7, m, E, K, inner, limit=63)
    cfg = MN.MiningConfig(min_m=256, min_n=256, min_k=256)
    job = MN.MiningJob(bytes(range(32)), 0, True)
    out, mined = MN.moe_layer(x, logits, w1, s1, w2, s2, top_k, job=job, config=cfg, residual=res)
    torch.cuda.synchronize()
    assert mined is not None and mined.per_expert
    for e in mined.per_expert.values():
        assert e.sync_fields()["error"] == 0
        MN.release_header(e.host_signal_header_pinned)
    want = exact(x, logits, w1, s1, w2, s2, top_k, res)
    moved = (want - res.double()).norm()
    assert float((out.double() - want).norm() / moved) < 0.08 + 2.0 ** -8 * float(want.norm() / moved)
    small, none = MN.moe_layer(x[:8], logits[:8], w1, s1, w2, s2, top_k, job=job, config=cfg, residual=res[:8])
    assert none is None
    assert float((small.double() - want[:8]).norm() / (want[:8] - res[:8].double()).norm()) < 0.08


class Layer:
    pass


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("mining", [True, False])
@pytest.mark.parametrize("act", ["none", "gelu", "silu"])
def test_apply_fused(dtype, mining, act):
    g = torch.Generator(device="cuda").manual_seed(2)
    m, n, k = 40, 264, 512
    lay = Layer()
    lay.weight = torch.randint(-63, 64, (n, k), generator=g, device="cuda", dtype=torch.int8)
    lay.weight_scale = (torch.rand(n, 1, generator=g, device="cuda") + 0.5) / (36 * math.sqrt(k))
    lay.smooth_quant_scale = torch.rand(k, generator=g, device="cuda") + 0.5
    x = torch.randn(m, k, generator=g, device="cuda").to(dtype)
    bias = torch.randn(n, generator=g, device="cuda").to(dtype)
    res = torch.randn(m, n, generator=g, device="cuda").to(dtype)
    got = MN.PearlLinear(mining).apply_fused(lay, x, bias=bias, activation=act, residual=res)
    xq, xs, _ = (MN.quant_7bit if mining else MN.quant_8bit)(x, lay.smooth_quant_scale)
    z = (xq.double() @ lay.weight.double().T) * xs.double() * lay.weight_scale.reshape(1, -1).double() + bias.double()
    want = MN._ELEMENTWISE[act](z) + res.double()
    tol = want.abs() * (2.0 ** -8 if dtype is torch.bfloat16 else 2.0 ** -11) * 1.02 + 2.0 ** -18 * (1 + z.abs() + res.double().abs())
    assert bool(((got.double() - want).abs() <= tol).all())


def test_apply_fused_mined_takes_the_epilogue_behind_it():
    g = torch.Generator(device="cuda").manual_seed(8)
    m, n, k = 384, 512, 1024
    lay = Layer()
    lay.weight = torch.randint(-63, 64, (n, k), generator=g, device="cuda", dtype=torch.int8)
    lay.weight_scale = (torch.rand(n, 1, generator=g, device="cuda") + 0.5) / (36 * math.sqrt(k))
    x = torch.randn(m, k, generator=g, device="cuda").to(torch.bfloat16)
    bias, res = torch.randn(n, generator=g, device="cuda"), torch.randn(m, n, generator=g, device="cuda").to(torch.bfloat16)
    cfg = MN.MiningConfig(min_m=256, min_n=256, min_k=256)
    lin = MN.PearlLinear(True, cfg, MN.MiningJob(bytes(32), 0, True))
    got = lin.apply_fused(lay, x, bias=bias, activation="silu", residual=res)
    assert len(lin.mined) == 1 and lin.mined[0].sync_fields()["error"] == 0
    MN.release_header(lin.mined[0].host_signal_header_pinned)
    plain = MN.PearlLinear(True).apply_fused(lay, x, bias=bias, activation="silu", residual=res)
    # the mined product is within the denoising tolerance (0.1 + 1%) of the plain one
    torch.testing.assert_close(got.float(), plain.float(), atol=0.12, rtol=0.02)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_no_tokens(dtype):
    x, logits, w1, s1, w2, s2, res = layer(3, 4, 8, 256, 128, dtype)
    out, mined = MN.moe_layer(x[:0], logits[:0], w1, s1, w2, s2, 2, residual=res[:0])
    assert mined is None and out.shape == (0, w2.shape[1]) and out.dtype is dtype and out.is_cuda
    lay = Layer()
    lay.weight, lay.weight_scale = w2[0], s2[0]
    got = MN.PearlLinear(False).apply_fused(lay, x[:0, :w2.shape[2]], activation="gelu")
    assert got.shape == (0, w2.shape[1]) and got.dtype is dtype and got.is_cuda
    with pytest.raises(RuntimeError, match="activation must be"):
        MN.PearlLinear(False).apply_fused(lay, x[:0, :w2.shape[2]], activation="tanh")
