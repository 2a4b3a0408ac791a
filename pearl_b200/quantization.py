"""Mirror of ``pearl_gemm.quantization`` (miner/pearl-gemm/src/pearl_gemm/
quantization/__init__.py, hadamard.py:530-611): the fused block-Hadamard +
smooth-scale + symmetric per-token quantization that turns a layer's bf16 /
fp16 activations into the int7 (max_val 63) or int8 (127) operand of the
mined GEMM.  Runs the B200 kernel in pearl_b200/csrc/quant.cu."""

from __future__ import annotations

import torch

from . import _lib
from .pearl_gemm_interface import _call_on, _device_index, _fail, _stream

_PACK_GATED = _lib.packer(_lib.GatedQuantParams)
DEFAULT_HADAMARD_BLOCK_SIZE = 16  # hadamard.py:520


def quantize(
    x: torch.Tensor,
    xq: torch.Tensor,
    xq_scales: torch.Tensor,
    smooth_scale: torch.Tensor | None = None,
    max_val: int = 63,
    block_size: int = DEFAULT_HADAMARD_BLOCK_SIZE,
) -> None:
    """xq = rint(v * inv) with v = Hadamard_k(x) * smooth (k = block_size,
    0 = no transform), inv = max_val * rcp.approx(amax_row(v) + 1e-30) and
    xq_scales = amax_row(v) * fl(1 / max_val): the reference's float32 steps
    (hadamard.py:443-466), so the same bytes come out.

    x: (M, N) fp16 / bf16 contiguous; xq: (M, N) int8; xq_scales: (M, 1)
    fp32; smooth_scale: (1, N) broadcast or (M, N) per token, fp32."""
    if x.dim() != 2:
        _fail("x must be 2D (M, N)")
    M, N = x.shape
    if x.dtype not in (torch.bfloat16, torch.float16):
        _fail(f"x must be float16 or bfloat16, got {x.dtype}")
    for t, name in ((x, "x"), (xq, "xq"), (xq_scales, "xq_scales")):
        if not t.is_cuda:
            _fail(f"{name} must be on CUDA")
        if not t.is_contiguous():
            _fail(f"{name} must be contiguous")
    if xq.dtype != torch.int8 or tuple(xq.shape) != (M, N):
        _fail(f"xq must be int8 of shape ({M}, {N})")
    if xq_scales.dtype != torch.float32 or xq_scales.numel() != M:
        _fail(f"xq_scales must be float32 of shape ({M}, 1)")
    per_row = 0
    if smooth_scale is not None:
        if smooth_scale.dtype != torch.float32 or not smooth_scale.is_cuda or not smooth_scale.is_contiguous():
            _fail("smooth_scale must be a contiguous float32 CUDA tensor")
        if smooth_scale.dim() != 2 or smooth_scale.shape[1] != N or smooth_scale.shape[0] not in (1, M):
            _fail(f"smooth_scale must have shape (1, {N}) or ({M}, {N})")
        per_row = int(smooth_scale.shape[0] == M and M != 1)
    if block_size > 0:
        if block_size < 2 or (block_size & (block_size - 1)) != 0:
            raise ValueError(f"block_size must be a power of 2 ≥ 2, got {block_size}")
        if N % block_size != 0:
            raise ValueError(f"N (={N}) must be divisible by block_size (={block_size})")
    p = _lib.QuantParams()
    p.device = _device_index(x)
    p.x, p.x_is_fp16, p.m, p.n = x.data_ptr(), int(x.dtype == torch.float16), M, N
    p.smooth = smooth_scale.data_ptr() if smooth_scale is not None else None
    p.smooth_per_row = per_row
    p.xq, p.scales, p.max_val, p.block_size = xq.data_ptr(), xq_scales.data_ptr(), int(max_val), int(block_size)
    with torch.cuda.device(x.device):
        _lib.call("pb2_quantize", p, _stream(x.device), "quantize")


def quantize_gated(x, xq, xq_scales, *, activation: str = "silu", row_index=None, smooth_scale=None,
                   max_val: int = 127, block_size: int = 0) -> None:
    """The quantized gated activation of an MLP (no reference counterpart):
    rows of ``x`` (rows, 2 N), bf16 or fp16, hold N gate and then N up values;
    in float32

        v = act(gate) * up, block-Hadamard transform of width block_size
            (as ``quantize``; 0 = none), times smooth_scale (1, N) or (N,)
        xq_scales = amax_row(v) * fl(1 / max_val)
        xq = rint(v * (max_val / amax_row(v))), 0 for a row of zeros

    A NaN or an infinity in a row makes its scale one; the bytes of a row with
    an infinity are +-max_val where it is infinite and 0 elsewhere, those of a
    row with a NaN all 0.

    xq (M, N) int8, xq_scales (M,) or (M, 1) float32.  With ``row_index``
    ((M,) int32) row i of the result is row row_index[i] of x -- a MoE
    layer's slots in expert order -- and an index outside x gives a row of
    zeros; without it M = rows."""
    from .linear import _FLOAT, _INT8, _INT32, _activation, _half_type, _operand

    if x.dim() != 2 or x.shape[1] % 2:
        _fail("x must be 2D (M, 2 N): gate values, then up values")
    rows, N = x.shape[0], x.shape[1] // 2
    at = x.get_device()
    half = _half_type(x, "x")
    M = rows if row_index is None else row_index.numel()
    if N % 8:
        _fail(f"the row length must be a multiple of 8, got {N}")
    if not 0 < max_val <= 127:
        _fail(f"max_val must be in 1..127, got {max_val}")
    _check_block(block_size, N)
    _call_on(at, "pb2_quantize_gated", _PACK_GATED(
        at, _operand(x, "x", (rows, 2 * N), (x.dtype,), at), half, M, N, rows, _activation(activation),
        0 if row_index is None else _operand(row_index, "row_index", (M,), _INT32, at),
        0 if smooth_scale is None else _operand(
            smooth_scale, "smooth_scale", (1, N) if smooth_scale.dim() == 2 else (N,), _FLOAT, at),
        _operand(xq, "xq", (M, N), _INT8, at),
        _operand(xq_scales, "xq_scales", (M, 1) if xq_scales.dim() == 2 else (M,), _FLOAT, at),
        max_val, block_size), "quantize_gated")


def _check_block(block_size: int, n: int) -> None:
    if block_size and (block_size not in (8, 16, 32, 64, 128, 256) or n % block_size):
        raise ValueError(f"block_size must be 0 or a power of 2 in 8..256 that divides {n}, got {block_size}")


def rcp_approx_f32(x: torch.Tensor) -> torch.Tensor:
    """rcp.approx.ftz.f32 of every element of a float32 CUDA tensor: the
    approximate reciprocal ``quantize`` takes for its inverse scale, as the
    reference's kernel does (hadamard.py:446, cute.arch.rcp_approx).  PTX
    bounds its error to 1 ulp without fixing the last bit, so a CPU
    restatement of the quantizer reads it from here (a test aid)."""
    if not x.is_cuda or x.dtype != torch.float32 or not x.is_contiguous():
        _fail("x must be a contiguous float32 CUDA tensor")
    out = torch.empty_like(x)
    with torch.cuda.device(x.device):
        st = _lib.load().pb2_rcp_approx_f32(_device_index(x), x.data_ptr(), out.data_ptr(), x.numel(),
                                            _stream(x.device))
    _lib.check(st, "rcp_approx_f32")
    return out


__all__ = ["quantize", "quantize_gated", "rcp_approx_f32", "DEFAULT_HADAMARD_BLOCK_SIZE"]
