"""The un-mined linear layer with its epilogue: int8 product, bias,
activation and residual in one kernel (pearl_b200/csrc/product.cu).  No
reference counterpart: the reference's vanilla GEMM stops at the scales
(gemm_operators.py:28-65) and leaves the rest to separate elementwise passes."""

from __future__ import annotations

import torch

from . import _lib
from .pearl_gemm_interface import _call_on, _fail

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _activation(name: str) -> int:
    code = ACTIVATIONS.get(name)
    if code is None:
        _fail(f"activation must be one of {', '.join(ACTIVATIONS)}, got {name!r}")
    return code


def _operand(t, name: str, shape: tuple, dtypes: tuple, device) -> int:
    """Address of a contiguous tensor of this shape, type and device."""
    if not t.is_cuda:
        _fail(f"{name} must be on CUDA")
    if t.device != device:
        _fail(f"{name} must be on {device}, got {t.device}")
    if not t.is_contiguous():
        _fail(f"{name} must be contiguous")
    if t.dtype not in dtypes:
        _fail(f"expected dtype: {' or '.join(str(d) for d in dtypes)} but got this dtype: {t.dtype} ({name})")
    if t.shape != shape:
        _fail(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    return t.data_ptr()


def _half_type(t, name: str) -> int:
    if t.dtype is not torch.bfloat16 and t.dtype is not torch.float16:
        _fail(f"{name} must be bfloat16 or float16, got {t.dtype}")
    return _TYPES[t.dtype]


def _sync_word(sync):
    if sync is None:
        return None
    if not sync.is_cuda or sync.numel() != _lib.HOST_SIGNAL_SYNC_SIZE:
        _fail(f"host_signal_sync must be a {_lib.HOST_SIGNAL_SYNC_SIZE}-byte CUDA buffer")
    return sync.data_ptr()


def gemm_epilogue(A, B, A_scales, B_scales, C, *, bias=None, activation: str = "none", residual=None,
                  host_signal_sync=None) -> None:
    """C = act(A_scales * B_scales * (A . B^T) + bias) + residual, written
    into ``C``: the integer sum exact, the epilogue in float32, one rounding.

    A (m, k), B (n, k) int8 with k a multiple of 16; A_scales (m,), B_scales
    (n,) float32; C and ``residual`` (m, n) bfloat16 or float16; ``bias``
    (n,) float32 or C's type; ``activation`` one of ``ACTIVATIONS``.
    ``residual`` may be C itself.  ``host_signal_sync`` (optional) receives a
    device timeout in its error word, as for the other products."""
    if A.dim() != 2 or B.dim() != 2:
        _fail("A and B must be 2-D")
    m, k = A.shape
    n = B.shape[0]
    dev = A.device
    if k % 16:
        _fail(f"k must be a multiple of 16, got {k}")
    half = _half_type(C, "C")
    p = _lib.GemmEpilogueParams()
    p.A = _operand(A, "A", (m, k), (torch.int8,), dev)
    p.B = _operand(B, "B", (n, k), (torch.int8,), dev)
    p.A_scales = _operand(A_scales, "A_scales", (m,), (torch.float32,), dev)
    p.B_scales = _operand(B_scales, "B_scales", (n,), (torch.float32,), dev)
    p.C = _operand(C, "C", (m, n), (C.dtype,), dev)
    if bias is not None:
        p.bias, p.bias_type = _operand(bias, "bias", (n,), (torch.float32, C.dtype), dev), _TYPES[bias.dtype]
    if residual is not None:
        p.residual = _operand(residual, "residual", (m, n), (C.dtype,), dev)
    p.m, p.n, p.k, p.c_type, p.activation = m, n, k, half, _activation(activation)
    p.host_signal_sync = _sync_word(host_signal_sync)
    _call_on(dev, "pb2_gemm_epilogue", p, "gemm_epilogue")


__all__ = ["ACTIVATIONS", "gemm_epilogue"]
