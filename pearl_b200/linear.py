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
_INT8, _INT32, _FLOAT = (torch.int8,), (torch.int32,), (torch.float32,)
_PACK = _lib.packer(_lib.GemmEpilogueParams)


def _activation(name: str) -> int:
    code = ACTIVATIONS.get(name)
    if code is None:
        _fail(f"activation must be one of {', '.join(ACTIVATIONS)}, got {name!r}")
    return code


def _operand(t, name: str, shape: tuple, dtypes: tuple, index: int) -> int:
    """Address of a contiguous tensor of this shape and type on device
    ``index``."""
    if t.get_device() == index >= 0 and t.is_contiguous() and t.dtype in dtypes and t.shape == shape:
        return t.data_ptr()
    if not t.is_cuda:
        _fail(f"{name} must be on CUDA")
    if t.get_device() != index:
        _fail(f"{name} must be on cuda:{index}, got {t.device}")
    if not t.is_contiguous():
        _fail(f"{name} must be contiguous")
    if t.dtype not in dtypes:
        _fail(f"expected dtype: {' or '.join(str(d) for d in dtypes)} but got this dtype: {t.dtype} ({name})")
    _fail(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _half_type(t, name: str) -> int:
    if t.dtype is not torch.bfloat16 and t.dtype is not torch.float16:
        _fail(f"{name} must be bfloat16 or float16, got {t.dtype}")
    return _TYPES[t.dtype]


def _sync_word(sync, index: int) -> int:
    if sync is None:
        return 0
    if sync.get_device() != index or sync.numel() != _lib.HOST_SIGNAL_SYNC_SIZE or not sync.is_contiguous():
        _fail(f"host_signal_sync must be a contiguous {_lib.HOST_SIGNAL_SYNC_SIZE}-byte buffer on cuda:{index}")
    return sync.data_ptr()


def gemm_epilogue(A, B, A_scales, B_scales, C, *, bias=None, activation: str = "none", residual=None,
                  host_signal_sync=None) -> None:
    """C = act(A_scales * B_scales * (A . B^T) + bias) + residual, written
    into ``C``: the integer sum exact (in int32, which any values of k up to
    131071 fit; beyond, it wraps where the values let it), the epilogue in
    float32, one rounding.

    A (m, k), B (n, k) int8 with k a multiple of 16; A_scales (m,), B_scales
    (n,) float32; C and ``residual`` (m, n) bfloat16 or float16; ``bias``
    (n,) float32 or C's type; ``activation`` one of ``ACTIVATIONS``.
    ``residual`` may be C itself.  ``host_signal_sync`` (optional) receives a
    device timeout in its error word, as for the other products."""
    if A.dim() != 2 or B.dim() != 2:
        _fail("A and B must be 2-D")
    m, k = A.shape
    n = B.shape[0]
    at = A.get_device()
    if k % 16:
        _fail(f"k must be a multiple of 16, got {k}")
    half = _half_type(C, "C")
    _call_on(at, "pb2_gemm_epilogue", _PACK(
        at, m, n, k, _operand(A, "A", (m, k), _INT8, at), _operand(B, "B", (n, k), _INT8, at),
        _operand(A_scales, "A_scales", (m,), _FLOAT, at), _operand(B_scales, "B_scales", (n,), _FLOAT, at),
        _operand(C, "C", (m, n), (C.dtype,), at), half,
        0 if bias is None else _operand(bias, "bias", (n,), (C.dtype, torch.float32), at),
        0 if bias is None else _TYPES[bias.dtype], _activation(activation),
        0 if residual is None else _operand(residual, "residual", (m, n), (C.dtype,), at),
        _sync_word(host_signal_sync, at)), "gemm_epilogue")


__all__ = ["ACTIVATIONS", "gemm_epilogue"]
