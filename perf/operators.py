"""The operators around a quantized MoE layer and a quantized linear layer, as they are measured.

Three operators, each in its plain form (elementary torch operations in 32 bits, rounded once) and as a user calls it:

* ``route``: router logits (tokens, experts) -> the top_k experts of every token, in descending order, and their weights.
  Scores are a softmax or sigmoids; a bias per expert may take part in the choice but not in the weights; groups of experts may be
  dropped first.  Ties go to the lowest index.
* ``linear``: an int8 product with row and column scales, then bias, activation and residual in its epilogue:
  ``C = act(A_scale * B_scale * (A . B^T) + bias) + residual``.
* ``experts``: the second half of the experts' MLP.  The first product's output (one row per routed slot: gate half, up half) goes
  through silu(gate) * up, is quantized to int8 per row, multiplied by its expert's down projection, and the slots of a token are
  added up with the router's weights.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh")
DEVICE = "cuda"


def listed():
    return [
        # The router of one small decode step: launch latency, nothing else.
        dict(name="route decode 4x8", op="route", tokens=4, experts=8, top_k=2, scoring="softmax", bias=False, groups=1,
             kept_groups=1, dtype="bf16"),
        # An odd number of tokens and of experts, half-precision logits.
        dict(name="route odd 777x60", op="route", tokens=777, experts=60, top_k=4, scoring="softmax", bias=False, groups=1,
             kept_groups=1, dtype="f16"),
        # Many fine-grained experts in groups, sigmoid scores with a balance bias.
        dict(name="route groups 4099x256", op="route", tokens=4099, experts=256, top_k=8, scoring="sigmoid", bias=True, groups=8,
             kept_groups=4, dtype="f32"),
        # A long prefill batch.
        dict(name="route prefill 32768x128", op="route", tokens=32768, experts=128, top_k=8, scoring="softmax", bias=False,
             groups=1, kept_groups=1, dtype="f32"),
        # One token through an attention output projection with bias and the residual stream: the weights are read once.
        dict(name="linear token 1x4096x4096", op="linear", m=1, n=4096, k=4096, bias=True, activation="none", residual=True,
             dtype="bf16"),
        # A decode batch through the down projection of the framework's decode workload.
        dict(name="linear batch 256x4096x14336", op="linear", m=256, n=4096, k=14336, bias=False, activation="none",
             residual=True, dtype="bf16"),
        # Ragged in every direction: K not a multiple of the K tile, N and M not of theirs.
        dict(name="linear ragged 333x5000x1040", op="linear", m=333, n=5000, k=1040, bias=True, activation="gelu_tanh",
             residual=False, dtype="f16"),
        # Prefill through the up projection of an MLP with bias and gelu.
        dict(name="linear prefill 8192x14336x4096", op="linear", m=8192, n=14336, k=4096, bias=True, activation="gelu",
             residual=False, dtype="bf16"),
        # A decode step of eight wide experts: their weights are read once.
        dict(name="experts decode 8x8", op="experts", tokens=8, experts=8, top_k=2, hidden=4096, inner=14336, smooth=False,
             residual=True, dtype="bf16"),
        # An odd batch over many narrow experts, some of them empty, smooth scales, no residual.
        dict(name="experts ragged 331x60", op="experts", tokens=331, experts=60, top_k=4, hidden=2040, inner=1360, smooth=True,
             residual=False, dtype="f16"),
        # A batch of 128 fine-grained experts at about 128 rows each.
        dict(name="experts fine 2048x128", op="experts", tokens=2048, experts=128, top_k=8, hidden=2048, inner=768, smooth=False,
             residual=True, dtype="bf16"),
        # The framework's MoE prefill widths at half of its batch.
        dict(name="experts prefill 8192x8", op="experts", tokens=8192, experts=8, top_k=2, hidden=4096, inner=14336, smooth=False,
             residual=True, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "linear", "experts"])
    if op == "route":
        experts, groups = rng.choice([(8, 1), (16, 4), (60, 1), (64, 8), (72, 6), (100, 1), (128, 1), (160, 8), (256, 1), (256, 8)])
        kept = rng.randint(max(1, groups // 2), groups)
        scoring = rng.choice(["softmax", "sigmoid"])
        return dict(op=op, tokens=min(32768, _log(rng, 1, 32768) | rng.randint(0, 1)), experts=experts,
                    top_k=rng.randint(1, min(8, kept * (experts // groups))), scoring=scoring,
                    bias=scoring == "sigmoid" and rng.random() < 0.7, groups=groups, kept_groups=kept,
                    dtype=rng.choice(["f32", "bf16", "f16"]))
    if op == "linear":
        most = 8192 * 14336 * 4096
        while True:
            m, n, k = _log(rng, 1, 8192), 8 * _log(rng, 8, 1792), 16 * _log(rng, 16, 896)
            if m * n * k <= most:
                break
        return dict(op=op, m=m, n=n, k=k, bias=rng.random() < 0.6, activation=rng.choice(ACTIVATIONS),
                    residual=rng.random() < 0.5, dtype=rng.choice(["bf16", "f16"]))
    while True:
        tokens, experts = _log(rng, 1, 8192), rng.choice([4, 8, 16, 60, 64, 128])
        top_k = rng.randint(1, min(8, experts))
        hidden, inner = 8 * _log(rng, 32, 512), 16 * _log(rng, 16, 896)
        if (tokens * top_k * inner <= 8192 * 2 * 14336 and experts * hidden * inner <= 8 * 4096 * 14336
                and tokens * top_k * hidden <= 8192 * 2 * 4096):
            break
    return dict(op=op, tokens=tokens, experts=experts, top_k=top_k, hidden=hidden, inner=inner, smooth=rng.random() < 0.4,
                residual=rng.random() < 0.5, dtype=rng.choice(["bf16", "f16"]))


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE)


def _int8(g, rows, cols):
    """Quantized values of a normal distribution: what a row of activations or weights holds after its scale is taken out."""
    out = torch.empty(rows, cols, dtype=torch.int8, device=DEVICE)
    step = max(1, (1 << 26) // cols)
    for r in range(0, rows, step):
        n = min(step, rows - r)
        out[r:r + n] = (_randn(g, n, cols) * 32).round_().clamp_(-127, 127).to(torch.int8)
    return out


def _scales(g, n, middle):
    return (torch.rand(n, generator=g, device=DEVICE) + 0.5) * middle


def _logits(g, tokens, experts):
    """A router's logits: some experts are more popular than others."""
    return _randn(g, tokens, experts) * 1.5 + _randn(g, experts) * 0.7


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case=case)
    if case["op"] == "route":
        s["logits"] = _logits(g, case["tokens"], case["experts"]).to(DTYPES[case["dtype"]])
        s["bias"] = _randn(g, case["experts"]) * 0.1 if case["bias"] else None
        s["scaling"] = 2.5 if case["scoring"] == "sigmoid" else 1.0
    elif case["op"] == "linear":
        m, n, k, dt = case["m"], case["n"], case["k"], DTYPES[case["dtype"]]
        s["A"], s["B"] = _int8(g, m, k), _int8(g, n, k)
        s["A_scales"], s["B_scales"] = _scales(g, m, 1 / 32), _scales(g, n, 1 / (32 * math.sqrt(k)))
        s["bias"] = _randn(g, n).to(dt) if case["bias"] else None
        s["residual"] = _randn(g, m, n).to(dt) if case["residual"] else None
    else:
        tokens, experts, top_k, hidden, inner = (case[w] for w in ("tokens", "experts", "top_k", "hidden", "inner"))
        dt, slots = DTYPES[case["dtype"]], tokens * top_k
        top = _logits(g, tokens, experts).sort(dim=1, descending=True, stable=True)
        ids = top.indices[:, :top_k].reshape(-1)
        s["weights"] = torch.softmax(top.values[:, :top_k], dim=1)
        s["slots"] = ids.sort(stable=True).indices.to(torch.int32)
        counts = torch.bincount(ids, minlength=experts)
        s["offsets"] = counts.cumsum(0).to(torch.int32)
        s["most_rows"] = int(counts.max())
        s["x"] = torch.empty(slots, 2 * inner, dtype=dt, device=DEVICE)
        step = max(1, (1 << 26) // (2 * inner))
        for r in range(0, slots, step):
            s["x"][r:r + step] = _randn(g, min(step, slots - r), 2 * inner).to(dt)
        s["w"] = _int8(g, experts * hidden, inner).view(experts, hidden, inner)
        s["w_scales"] = _scales(g, experts * hidden, 1 / (32 * math.sqrt(inner))).view(experts, hidden)
        s["smooth"] = _scales(g, inner, 1.0).view(1, inner) if case["smooth"] else None
        s["residual"] = _randn(g, tokens, hidden).to(dt) if case["residual"] else None
    return s


# ------------------------------------------------------------------ run
def run(s):
    op = s["case"]["op"]
    if own:
        import pearl_b200
        return {"route": _route_own, "linear": _linear_own, "experts": _experts_own}[op](pearl_b200, s)
    return {"route": _route_plain, "linear": _linear_plain, "experts": _experts_plain}[op](s)


def _route_own(pearl, s):
    c, x = s["case"], s["logits"]
    ids = torch.empty(c["tokens"], c["top_k"], dtype=torch.int32, device=x.device)
    weights = torch.empty(c["tokens"], c["top_k"], dtype=torch.float32, device=x.device)
    pearl.moe.route_tokens(x, weights, ids, scoring=c["scoring"], bias=s["bias"], num_groups=c["groups"],
                           topk_groups=c["kept_groups"], scaling=s["scaling"])
    return {"ids": ids, "weights": weights}


def _route_plain(s):
    c, x = s["case"], s["logits"].float()
    m, experts = x.shape
    if c["scoring"] == "softmax":
        e = torch.exp(x - x.amax(dim=1, keepdim=True))
        scores = e / e.sum(dim=1, keepdim=True)
    else:
        scores = 1 / (1 + torch.exp(-x))
    # Both scores grow with the logit, so without a bias the choice goes by the logits.
    key = x if s["bias"] is None else scores + s["bias"]
    if c["groups"] > 1:
        by_group = key.view(m, c["groups"], -1)
        if s["bias"] is None:
            group = by_group.amax(dim=2)
        else:
            group = by_group.sort(dim=2, descending=True).values[:, :, :2].sum(dim=2)
        kept = group.sort(dim=1, descending=True, stable=True).indices[:, :c["kept_groups"]]
        keep = torch.zeros_like(group, dtype=torch.bool).scatter_(1, kept, True)
        key = torch.where(keep[:, :, None], by_group, -math.inf).view(m, experts)
    ids = key.sort(dim=1, descending=True, stable=True).indices[:, :c["top_k"]]
    w = scores.gather(1, ids)
    return {"ids": ids.to(torch.int32), "weights": w / w.sum(dim=1, keepdim=True) * s["scaling"]}


def _linear_own(pearl, s):
    A, B = s["A"], s["B"]
    C = torch.empty(A.shape[0], B.shape[0], dtype=DTYPES[s["case"]["dtype"]], device=A.device)
    pearl.gemm_epilogue(A, B, s["A_scales"], s["B_scales"], C, bias=s["bias"], activation=s["case"]["activation"],
                        residual=s["residual"])
    return C


def _linear_plain(s):
    c = s["case"]
    y = (s["A"].float() @ s["B"].float().T) * s["A_scales"][:, None] * s["B_scales"][None, :]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if c["activation"] == "relu":
        y = torch.where(y > 0, y, 0.0)
    elif c["activation"] == "silu":
        y = y / (1 + torch.exp(-y))
    elif c["activation"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    elif c["activation"] == "gelu_tanh":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(DTYPES[c["dtype"]])


def _experts_own(pearl, s):
    x = s["x"]
    out = torch.empty(s["case"]["tokens"], s["case"]["hidden"], dtype=x.dtype, device=x.device)
    pearl.moe.gated_experts(x, s["w"], s["w_scales"], out, s["slots"], s["offsets"], s["weights"], smooth_scale=s["smooth"],
                            residual=s["residual"])
    return out


def _experts_plain(s):
    c, x, slots = s["case"], s["x"], s["slots"].long()
    inner, hidden = c["inner"], c["hidden"]
    gate, up = x[:, :inner].float(), x[:, inner:].float()
    v = gate / (1 + torch.exp(-gate)) * up
    if s["smooth"] is not None:
        v = v * s["smooth"]
    most = v.abs().amax(dim=1, keepdim=True)
    q = torch.round(v * torch.where(most > 0, 127 / most, 0.0)).clamp(-127, 127)
    row_scale = most * (1 / 127)
    # The experts' rows as one batch, padded to the longest expert.
    ends = s["offsets"].long()
    begins = torch.nn.functional.pad(ends, (1, 0))[:-1]
    at = begins[:, None] + torch.arange(s["most_rows"], device=x.device)
    live = at < ends[:, None]
    slot = slots[at.clamp(max=slots.numel() - 1)]
    y = torch.bmm(q[slot], s["w"].float().transpose(1, 2)) * row_scale[slot] * s["w_scales"][:, None, :]
    flat = torch.empty(slots.numel() + 1, hidden, device=x.device)
    flat[torch.where(live, slot, slots.numel()).view(-1)] = y.view(-1, hidden)
    out = (flat[:-1].view(c["tokens"], c["top_k"], hidden) * s["weights"][:, :, None]).sum(dim=1)
    if s["residual"] is not None:
        out = out + s["residual"].float()
    return out.to(x.dtype)


# ------------------------------------------------------------------ work
def work(case):
    if case["op"] == "route":
        m, e, k = case["tokens"], case["experts"], case["top_k"]
        return {"bytes": m * e * (4 if case["dtype"] == "f32" else 2) + m * k * 8 + (4 * e if case["bias"] else 0),
                "flops": 5 * m * e}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + 4 * (m + n) + 2 * m * n * (2 if case["residual"] else 1) + (2 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    t, e, k, h, i = (case[w] for w in ("tokens", "experts", "top_k", "hidden", "inner"))
    touched = e * (1 - (1 - k / e) ** t)  # experts that some token chose, were all alike popular
    return {"bytes": 4 * t * k * i + touched * h * (i + 4) + 2 * t * h * (2 if case["residual"] else 1) + 8 * t * k,
            "flops": 2 * t * k * h * i}


# ------------------------------------------------------------------ exact
def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _route_exact, "linear": _linear_exact, "experts": _experts_exact}[case["op"]](case, s)


def _route_exact(c, s):
    x = s["logits"].double().cpu().numpy()
    m, experts = x.shape
    if c["scoring"] == "softmax":
        p = np.exp(x - x.max(axis=1)[:, None])
        p /= p.sum(axis=1)[:, None]
    else:
        p = 1.0 / (1.0 + np.exp(-x))
    key = x if s["bias"] is None else p + s["bias"].double().cpu().numpy()[None]
    width = experts // c["groups"]
    if c["groups"] > 1:
        parts = np.sort(key.reshape(m, c["groups"], width), axis=2)
        group = parts[:, :, -1] if s["bias"] is None else parts[:, :, -2:].sum(axis=2)
        order = np.argsort(-group, axis=1, kind="stable")
        rank = np.empty_like(order)
        np.put_along_axis(rank, order, np.broadcast_to(np.arange(c["groups"]), order.shape).copy(), axis=1)
        key = np.where(np.repeat(rank, width, axis=1) < c["kept_groups"], key, -np.inf)
    ids = np.argsort(-key, axis=1, kind="stable")[:, :c["top_k"]]
    w = np.take_along_axis(p, ids, axis=1)
    w = w / w.sum(axis=1, keepdims=True) * s["scaling"]
    # With a bias two experts' 32-bit scores can stand in another order than their 64-bit ones.
    return {"ids": None if c["bias"] else ids.astype(np.int32), "weights": w}


def _linear_exact(c, s):
    A, B = s["A"].double(), s["B"].double()
    out = torch.empty(c["m"], c["n"], dtype=torch.float64, device=A.device)
    for r in range(0, c["m"], 1024):
        y = A[r:r + 1024].matmul(B.t()).mul_(s["A_scales"][r:r + 1024].double().unsqueeze(1)).mul_(s["B_scales"].double())
        if s["bias"] is not None:
            y += s["bias"].double()
        if c["activation"] == "relu":
            y = y.clamp(min=0)
        elif c["activation"] == "silu":
            y = y * torch.sigmoid(y)
        elif c["activation"] == "gelu":
            y = y * torch.special.ndtr(y)
        elif c["activation"] == "gelu_tanh":
            y = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
        if s["residual"] is not None:
            y = y + s["residual"][r:r + 1024].double()
        out[r:r + 1024] = y
    return out


def _experts_exact(c, s):
    slots, ends, inner = s["slots"].long(), [0] + s["offsets"].tolist(), c["inner"]
    per_slot = torch.zeros(slots.numel(), c["hidden"], dtype=torch.float64, device=slots.device)
    for e in range(c["experts"]):
        for r in range(ends[e], ends[e + 1], 1024):
            rows = slots[r:min(r + 1024, ends[e + 1])]
            x = s["x"][rows].double()
            v = x[:, :inner] * torch.sigmoid(x[:, :inner]) * x[:, inner:]
            if s["smooth"] is not None:
                v = v * s["smooth"].double()
            unit = v.abs().max(dim=1, keepdim=True).values / 127
            q = (v / unit.clamp(min=1e-300)).round()
            per_slot[rows] = unit * q.matmul(s["w"][e].double().t()) * s["w_scales"][e].double()
    out = torch.einsum("tkh,tk->th", per_slot.view(c["tokens"], c["top_k"], -1), s["weights"].double())
    return out if s["residual"] is None else out + s["residual"].double()
