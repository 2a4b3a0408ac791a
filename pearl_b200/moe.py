"""Mirror of ``pearl_gemm.moe`` (miner/pearl-gemm/src/pearl_gemm/moe.py):
the canonical MoE routing order a mined expert layer commits to, computed on
the B200 (pearl_b200/csrc/routing.cu) through the C ABI."""

from __future__ import annotations

import torch

from . import _lib
from .linear import _FLOAT, _INT8, _INT32, _TYPES, _activation, _half_type, _operand, _sync_word
from .pearl_gemm_interface import _call_on, _device_index, _fail, _stream
from .quantization import _check_block

_SCORING = {"softmax": 0, "sigmoid": 1}
_LOGIT_TYPES = tuple(_TYPES)
_PACK_ROUTE, _PACK_GROUPED = _lib.packer(_lib.RouteParams), _lib.packer(_lib.GemmGroupedParams)
_PACK_COMBINE, _PACK_EXPERTS = _lib.packer(_lib.CombineParams), _lib.packer(_lib.GatedExpertsParams)
MAX_EXPERTS = 256  # the routing order sorts 8-bit expert ids
MAX_TOP_K = 32


def get_build_routing_data_scratchpad_bytes(numel: int) -> int:
    """Scratch bytes build_routing_data needs for ``numel`` routed slots."""
    return int(_lib.load().pb2_build_routing_data_scratchpad_bytes(int(numel)))


def build_routing_data(
    topk_ids: torch.Tensor,
    routing_data: torch.Tensor,
    slot_indices: torch.Tensor,
    routing_offsets: torch.Tensor,
    scratchpad: torch.Tensor,
    num_experts: int,
) -> None:
    """Stable per-expert ordering of the routed slots
    (build_routing_data.cu:127-166): ``slot_indices`` = flat slot indices
    sorted by expert id, ``routing_data`` = their tokens
    (``slot_indices // top_k``), ``routing_offsets[e]`` = exclusive end of
    expert e's segment.  Slots of ids outside 0..num_experts-1 come after the
    last segment."""
    named = ((topk_ids, "topk_ids"), (routing_data, "routing_data"), (slot_indices, "slot_indices"),
             (routing_offsets, "routing_offsets"), (scratchpad, "scratchpad"))
    for t, name in named:
        if not t.is_cuda:
            _fail(f"{name} must be on CUDA")
    for t, name in named:
        if not t.is_contiguous():
            _fail(f"{name} must be contiguous")
    for t, name in named[:4]:
        if t.dtype != torch.int32:
            _fail(f"{name} must be int32")
    if scratchpad.dtype != torch.uint8:
        _fail("scratchpad must be uint8")
    if topk_ids.dim() != 2:
        _fail("topk_ids must be 2D (m, K)")
    num_tokens, top_k = topk_ids.shape
    numel = num_tokens * top_k
    if routing_data.numel() != numel:
        _fail("routing_data must have m*K elements")
    if slot_indices.numel() != numel:
        _fail("slot_indices must have m*K elements")
    if num_experts > 256:
        _fail(f"build_routing_data sorts on 8-bit expert IDs, got num_experts={num_experts}")
    if routing_offsets.numel() != num_experts:
        _fail("routing_offsets must have num_experts elements")
    required = get_build_routing_data_scratchpad_bytes(numel)
    if scratchpad.numel() < required:
        _fail(f"scratchpad too small: need {required} bytes, got {scratchpad.numel()}")
    p = _lib.RoutingParams()
    p.device = _device_index(topk_ids)
    p.topk_ids, p.num_tokens, p.top_k = topk_ids.data_ptr(), num_tokens, top_k
    p.routing_data, p.slot_indices = routing_data.data_ptr(), slot_indices.data_ptr()
    p.routing_offsets, p.num_experts = routing_offsets.data_ptr(), num_experts
    p.scratchpad, p.scratchpad_bytes = scratchpad.data_ptr(), scratchpad.numel()
    with torch.cuda.device(topk_ids.device):
        _lib.call("pb2_build_routing_data", p, _stream(topk_ids.device), "build_routing_data")


def scatter_rows(src: torch.Tensor, dst: torch.Tensor, indices: torch.Tensor) -> None:
    """``dst[indices] = src`` for whole rows (2-D, contiguous, same dtype and
    row length; ``indices`` int32 on the same device): the per-expert step
    that puts a mined expert GEMM's rows back in routing-slot order
    (pearl_moe_experts.py:347).  A B200 kernel in place of torch's index_put;
    indices outside ``dst`` are skipped."""
    if not (src.is_cuda and dst.is_cuda and indices.is_cuda):
        _fail("scatter_rows: tensors must be on CUDA")
    if src.dim() != 2 or dst.dim() != 2 or src.shape[1] != dst.shape[1] or src.dtype != dst.dtype:
        _fail("scatter_rows: src and dst must be 2-D with the same row length and dtype")
    if not (src.is_contiguous() and dst.is_contiguous() and indices.is_contiguous()):
        _fail("scatter_rows: tensors must be contiguous")
    if indices.dtype != torch.int32 or indices.numel() != src.shape[0]:
        _fail("scatter_rows: indices must be int32 with one entry per src row")
    row_bytes = src.shape[1] * src.element_size()
    if row_bytes % 16 != 0:
        _fail("scatter_rows: rows must be a multiple of 16 bytes")
    p = _lib.ScatterParams(device=_device_index(src), src=src.data_ptr(), dst=dst.data_ptr(),
                           indices=indices.data_ptr(), rows=src.shape[0], dst_rows=dst.shape[0],
                           row_bytes=row_bytes)
    with torch.cuda.device(src.device):
        _lib.call("pb2_scatter_rows", p, _stream(src.device), "scatter_rows")


def noisy_gemm_grouped(
    A, B, EAL, EAL_fp16, EBR, EBR_fp16, EAR_R_major, EBL_R_major, EAR_K_major, EBL_K_major,
    AxEBL_fp16, EARxBpEB_fp16, ApEA, BpEB, A_scales, B_scales, C, expert_rows,
    host_signal_headers, host_signal_syncs, pow_target, pow_key, *, hits=None, transcripts=None,
    digests=None, run_noising_A: bool = True, run_noising_B: bool = True, tile_size_m: int = 128,
    tile_size_n: int = 256, tile_size_k: int = 128, c_row_index=None,
):
    """The mined GEMM1 of every expert of a MoE layer in one call: for expert
    e, exactly ``noisy_gemm`` (run_noising_A/B, reduction and denoising on) of
    its rows of A against its rows of B -- the loop of
    pearl_moe_experts.py:304-343 -- as one noising launch and one persistent
    mined launch (per 16 experts).

    A-side tensors (A, EAL, EAL_fp16, ApEA, AxEBL_fp16, A_scales, C) hold
    every expert's rows in expert order, ``expert_rows[e]`` of them for expert
    e (0 allowed); B-side tensors (B, EBR, EBR_fp16, BpEB, EARxBpEB_fp16,
    B_scales) hold n rows per expert, expert e at rows [e n, e n + n); the
    K-side factors EAR_* / EBL_* are shared.  ``host_signal_headers`` /
    ``host_signal_syncs`` (and the optional ``hits`` / ``transcripts`` /
    ``digests``) are per-expert lists, used as for that expert's own
    noisy_gemm.

    ``c_row_index`` (optional, int32 (m,) on the device) fuses the slot-order
    write-back that follows the reference's loop (pearl_moe_experts.py:347,
    ``cache_flat[idx] = out``) into the epilogue: row i of the experts' C
    goes to row c_row_index[i] of ``C``, which then has at least m rows."""
    from .pearl_gemm_interface import _check_matmul_config, _check_tensor, _gemm_params, _ptr

    E = len(expert_rows)
    if E == 0:
        _fail("expert_rows must not be empty")
    m, k = A.shape
    n_all = B.shape[0]
    if n_all % E:
        _fail("B must hold the same number of rows for every expert")
    n = n_all // E
    r = EAL.shape[1]
    if sum(int(v) for v in expert_rows) != m or any(int(v) < 0 for v in expert_rows):
        _fail(f"expert_rows must be non-negative and add up to A's {m} rows")
    _check_matmul_config("noisy_gemm", tile_size_m, tile_size_n, tile_size_k, 1, 1, None, r)
    for t, shape, dt, name in (
            (A, (m, k), torch.int8, "A"), (EAL, (m, r), torch.int8, "EAL"),
            (EAL_fp16, (m, r), torch.float16, "EAL_fp16"), (ApEA, (m, k), torch.int8, "ApEA"),
            (AxEBL_fp16, (m, r), torch.float16, "AxEBL_fp16"), (A_scales, (m,), torch.float32, "A_scales"),
            (C, (C.shape[0] if c_row_index is not None else m, n), torch.bfloat16, "C"),
            (B, (n_all, k), torch.int8, "B"),
            (EBR, (n_all, r), torch.int8, "EBR"), (EBR_fp16, (n_all, r), torch.float16, "EBR_fp16"),
            (BpEB, (n_all, k), torch.int8, "BpEB"), (EARxBpEB_fp16, (n_all, r), torch.float16, "EARxBpEB_fp16"),
            (B_scales, (n_all,), torch.float32, "B_scales"), (EAR_R_major, (k, r), torch.int8, "EAR_R_major"),
            (EBL_R_major, (k, r), torch.int8, "EBL_R_major"), (EAR_K_major, (r, k), torch.int8, "EAR_K_major"),
            (EBL_K_major, (r, k), torch.int8, "EBL_K_major")):
        _check_tensor(t, shape, dt, name)
    for t, name in ((pow_target, "pow_target"), (pow_key, "pow_key")):
        _check_tensor(t, (8,), torch.uint32, name)
    if c_row_index is not None:
        _check_tensor(c_row_index, (m,), torch.int32, "c_row_index")
        if C.shape[0] < m:
            _fail(f"C must have at least {m} rows with c_row_index")
    if len(host_signal_headers) != E or len(host_signal_syncs) != E:
        _fail("one host signal header and one sync buffer per expert")
    p = _gemm_params(m, n, k, r, _device_index(A), tile_size_m, tile_size_n, tile_size_k, 1, 1, None, None,
                     True)
    p.A, p.B, p.EAL, p.EBR = _ptr(A), _ptr(B), _ptr(EAL), _ptr(EBR)
    p.EAR_R_major, p.EBL_R_major = _ptr(EAR_R_major), _ptr(EBL_R_major)
    p.EAR_K_major, p.EBL_K_major = _ptr(EAR_K_major), _ptr(EBL_K_major)
    p.ApEA, p.BpEB = _ptr(ApEA), _ptr(BpEB)
    p.EAL_fp16, p.EBR_fp16 = _ptr(EAL_fp16), _ptr(EBR_fp16)
    p.AxEBL_fp16, p.EARxBpEB_fp16 = _ptr(AxEBL_fp16), _ptr(EARxBpEB_fp16)
    p.A_scales, p.B_scales, p.C = _ptr(A_scales), _ptr(B_scales), _ptr(C)
    p.pow_target, p.pow_key = _ptr(pow_target), _ptr(pow_key)
    p.run_noising_a, p.run_noising_b = int(bool(run_noising_A)), int(bool(run_noising_B))
    p.k_blocks_per_split_noising_a = p.k_blocks_per_split_noising_b = -1
    table = (_lib.ExpertGemm * E)()
    row0 = 0
    for e in range(E):
        q = table[e]
        q.m, q.a_row0 = int(expert_rows[e]), row0
        row0 += int(expert_rows[e])
        hdr, sync = host_signal_headers[e], host_signal_syncs[e]
        if q.m > 0:
            if sync is None or not sync.is_cuda or sync.numel() != _lib.HOST_SIGNAL_SYNC_SIZE:
                _fail(f"expert {e}: host_signal_sync must be a {_lib.HOST_SIGNAL_SYNC_SIZE}-byte CUDA buffer")
            if hdr is not None and (hdr.is_cuda or not hdr.is_pinned()):
                _fail(f"expert {e}: host_signal_header_pinned must be a pinned CPU tensor")
        q.host_signal_sync = _ptr(sync)
        q.host_signal_header_pinned = _ptr(hdr)
        if hits is not None and hits[e] is not None:
            q.hits, q.hit_capacity = _ptr(hits[e]), hits[e].shape[0]
        for lst, words, field in ((transcripts, 16, "transcripts"), (digests, 8, "digests")):
            if lst is not None and lst[e] is not None:
                _check_tensor(lst[e], ((q.m // 2) * (n // 64), words), (torch.int32, torch.uint32),
                              f"{field}[{e}]")
                setattr(q, field, _ptr(lst[e]))
    g = _lib.GroupedGemmParams()
    g.shared, g.num_experts, g.experts = p, E, table
    if c_row_index is not None:
        g.c_row_index, g.c_rows = _ptr(c_row_index), C.shape[0]
    with torch.cuda.device(A.device):
        _lib.call("pb2_noisy_gemm_grouped", g, _stream(A.device), "noisy_gemm_grouped")


# ------------------------------------------------------- un-mined operators --
# No reference counterpart: the reference takes these steps of the layer from
# vLLM (pearl_moe_experts.py:377-434 runs them around its GEMM2).
def route_tokens(logits, topk_weights, topk_ids, *, scoring: str = "softmax", bias=None, num_groups: int = 1,
                 topk_groups: int = 1, renormalize: bool = True, scaling: float = 1.0) -> None:
    """The experts of every token: ``topk_ids`` (m, top_k) int32 in
    descending order, ties to the lowest index, and ``topk_weights`` (m,
    top_k) float32, from ``logits`` (m, num_experts) float32 / bf16 / fp16.

    Scores s are the row's softmax or sigmoids.  ``bias`` (num_experts,)
    float32 is added for the choice only.  With ``num_groups`` > 1 only the
    ``topk_groups`` best groups of experts take part; a group is worth its
    best expert, or with a bias the sum of its two best.  The weights are s
    of the chosen experts, divided by their sum when ``renormalize``, times
    ``scaling``.  A logit of -inf or NaN masks its expert (score 0, chosen
    last); a row that masks every expert gets weights 0.  ``topk_ids`` is
    what build_routing_data takes."""
    if logits.dim() != 2 or topk_ids.dim() != 2:
        _fail("logits and topk_ids must be 2D (m, num_experts) and (m, top_k)")
    m, experts = logits.shape
    top_k = topk_ids.shape[1]
    at = logits.get_device()
    if scoring not in _SCORING:
        _fail(f"scoring must be 'softmax' or 'sigmoid', got {scoring!r}")
    if not 1 <= experts <= MAX_EXPERTS:
        _fail(f"num_experts must be in 1..{MAX_EXPERTS}, got {experts}")
    if num_groups < 1 or experts % num_groups or not 1 <= topk_groups <= num_groups:
        _fail(f"num_groups must divide {experts} experts and topk_groups be in 1..num_groups, got "
              f"{num_groups} and {topk_groups}")
    if not 1 <= top_k <= min(MAX_TOP_K, topk_groups * (experts // num_groups)):
        _fail(f"top_k must be in 1..{min(MAX_TOP_K, topk_groups * (experts // num_groups))}, got {top_k}")
    _call_on(at, "pb2_route_tokens", _PACK_ROUTE(
        at, _operand(logits, "logits", (m, experts), _LOGIT_TYPES, at), _TYPES[logits.dtype], m, experts, top_k,
        _SCORING[scoring], 0 if bias is None else _operand(bias, "bias", (experts,), _FLOAT, at), num_groups,
        topk_groups, bool(renormalize), scaling,
        _operand(topk_weights, "topk_weights", (m, top_k), _FLOAT, at),
        _operand(topk_ids, "topk_ids", (m, top_k), _INT32, at)), "route_tokens")


def gemm_grouped(A, B, A_scales, B_scales, C, routing_offsets, *, c_row_index=None, host_signal_sync=None) -> None:
    """The un-mined product of every expert in one launch: rows of ``A``
    (m, k) int8 in expert order, expert e's ending at ``routing_offsets[e]``
    (build_routing_data's, read on the device: no host copy of the counts),
    against ``B`` (E, n, k) int8; A_scales (m,), B_scales (E, n) float32;

        C[i] = A_scales[i] * B_scales[e] * (A[i] . B[e]^T)   (float32, bf16 or fp16)

    With ``c_row_index`` ((m,) int32, e.g. slot_indices) row i goes to row
    c_row_index[i] of C instead; rows outside C are skipped.  Rows past the
    last expert's end are not written.  k a multiple of 16, E <= 256; sums as in
    gemm_epilogue."""
    if A.dim() != 2 or B.dim() != 3 or C.dim() != 2:
        _fail("A and C must be 2-D and B 3-D (num_experts, n, k)")
    m, k = A.shape
    experts, n, _ = B.shape
    at = A.get_device()
    if k % 16:
        _fail(f"k must be a multiple of 16, got {k}")
    if not 1 <= experts <= MAX_EXPERTS:
        _fail(f"num_experts must be in 1..{MAX_EXPERTS}, got {experts}")
    rows = m if c_row_index is None else C.shape[0]
    _call_on(at, "pb2_gemm_grouped", _PACK_GROUPED(
        at, m, n, k, _operand(A, "A", (m, k), _INT8, at), _operand(B, "B", (experts, n, k), _INT8, at),
        _operand(A_scales, "A_scales", (m,), _FLOAT, at), _operand(B_scales, "B_scales", (experts, n), _FLOAT, at),
        _operand(C, "C", (rows, n), tuple(_TYPES), at), _TYPES[C.dtype], experts,
        _operand(routing_offsets, "routing_offsets", (experts,), _INT32, at),
        0 if c_row_index is None else _operand(c_row_index, "c_row_index", (m,), _INT32, at), rows,
        _sync_word(host_signal_sync, at)), "gemm_grouped")


def combine_slots(slots, topk_weights, out, *, residual=None) -> None:
    """out[t] = residual[t] + sum_j topk_weights[t, j] * slots[t * top_k + j]:
    the token's experts added up in float32 in the order of j, rounded once.
    slots (m * top_k, n), out and ``residual`` (m, n), all bf16 or all fp16, or
    the slots float32; topk_weights (m, top_k) float32.  What a slot of weight 0 holds does
    not count; ``residual`` may be out itself."""
    if topk_weights.dim() != 2 or out.dim() != 2:
        _fail("topk_weights and out must be 2D (m, top_k) and (m, n)")
    m, top_k = topk_weights.shape
    n = out.shape[1]
    at = out.get_device()
    half = _half_type(out, "out")
    _call_on(at, "pb2_combine_slots", _PACK_COMBINE(
        at, _operand(slots, "slots", (m * top_k, n), (out.dtype, torch.float32), at), _TYPES[slots.dtype],
        _operand(topk_weights, "topk_weights", (m, top_k), _FLOAT, at),
        0 if residual is None else _operand(residual, "residual", (m, n), (out.dtype,), at),
        _operand(out, "out", (m, n), (out.dtype,), at), half, m, top_k, n), "combine_slots")


def get_gated_experts_workspace_bytes(slots: int, inner: int, hidden: int, one_pass: bool = False) -> int:
    """Workspace bytes that gated_experts needs for ``slots`` routed slots, or
    with ``one_pass`` those with which it always takes all columns at once
    (the least is enough for half of them where their float32 products are
    over 32 MB; the result is the same)."""
    return int(_lib.load().pb2_gated_experts_workspace_bytes(int(slots), int(inner), int(hidden) * (2 if one_pass else 1)))


def gated_experts(x, w, w_scales, out, slot_indices, routing_offsets, topk_weights, *, residual=None,
                  smooth_scale=None, activation: str = "silu", max_val: int = 127, block_size: int = 0,
                  workspace=None, host_signal_sync=None) -> None:
    """The second half of the experts' MLP: ``x`` (m * top_k, 2 inner), the
    first product's rows in slot order (gate values, then up values), through
    quantize_gated into expert order, gemm_grouped with ``w`` (E, hidden,
    inner) int8 / ``w_scales`` (E, hidden) float32 and combine_slots into
    ``out`` (m, hidden).  ``slot_indices`` (m * top_k,) and
    ``routing_offsets`` (E,) are build_routing_data's, ``topk_weights`` (m,
    top_k) route_tokens'.  x, out and ``residual`` are all bf16 or all fp16;
    ``smooth_scale`` (1, inner) or (inner,) float32.  ``workspace`` (uint8,
    get_gated_experts_workspace_bytes, for one pass or the least) is taken
    from torch's allocator, for one pass, when not given.  Before they are
    added up the slots' products are float32; in fp16, where they are over 32
    MB, those that it holds are rounded to it.  Slots past the last
    expert's end (ids outside 0..E-1, an expert that another GPU holds) add
    nothing to out."""
    if w.dim() != 3 or topk_weights.dim() != 2:
        _fail("w must be 3-D (num_experts, hidden, inner) and topk_weights 2D (m, top_k)")
    experts, hidden, inner = w.shape
    m, top_k = topk_weights.shape
    slots = m * top_k
    at = x.get_device()
    if inner % 16:
        _fail(f"inner must be a multiple of 16, got {inner}")
    if not 1 <= experts <= MAX_EXPERTS:
        _fail(f"num_experts must be in 1..{MAX_EXPERTS}, got {experts}")
    if not 0 < max_val <= 127:
        _fail(f"max_val must be in 1..127, got {max_val}")
    _check_block(block_size, inner)
    half = _half_type(x, "x")
    need = get_gated_experts_workspace_bytes(slots, inner, hidden)
    if workspace is None:
        workspace = torch.empty(get_gated_experts_workspace_bytes(slots, inner, hidden, one_pass=True), dtype=torch.uint8,
                                device=x.device)
    elif (workspace.get_device() != at or workspace.dtype != torch.uint8 or workspace.numel() < need
          or not workspace.is_contiguous()):
        _fail(f"workspace must be a contiguous uint8 tensor on {x.device} of at least {need} bytes")
    _call_on(at, "pb2_gated_experts", _PACK_EXPERTS(
        at, _operand(x, "x", (slots, 2 * inner), (x.dtype,), at), half, m, top_k, experts, inner, hidden,
        _activation(activation),
        0 if smooth_scale is None else _operand(
            smooth_scale, "smooth_scale", (1, inner) if smooth_scale.dim() == 2 else (inner,), _FLOAT, at),
        max_val, block_size, _operand(w, "w", (experts, hidden, inner), _INT8, at),
        _operand(w_scales, "w_scales", (experts, hidden), _FLOAT, at),
        _operand(slot_indices, "slot_indices", (slots,), _INT32, at),
        _operand(routing_offsets, "routing_offsets", (experts,), _INT32, at),
        _operand(topk_weights, "topk_weights", (m, top_k), _FLOAT, at),
        0 if residual is None else _operand(residual, "residual", (m, hidden), (x.dtype,), at),
        _operand(out, "out", (m, hidden), (x.dtype,), at), workspace.data_ptr(), workspace.numel(),
        _sync_word(host_signal_sync, at)), "gated_experts")
