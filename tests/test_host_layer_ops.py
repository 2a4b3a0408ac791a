"""CPU tests of the un-mined layer operators' boundary: struct layouts, and
refusals of the Python entry points and of the C ABI (nothing is launched:
every C call here is rejected before it touches a device)."""

import ctypes

import pytest
import torch

import pearl_b200 as pg
from pearl_b200 import _lib
from tests.test_host_abi import _c_sizeof

BAD, UNSUPPORTED = _lib.PB2_ERR_INVALID_ARGUMENT, _lib.PB2_ERR_UNSUPPORTED_CONFIG
P = 4096  # a 16-byte aligned address that is never read


@pytest.mark.parametrize("cname,pyname", [
    ("pb2_route_params", "RouteParams"), ("pb2_gemm_epilogue_params", "GemmEpilogueParams"),
    ("pb2_gated_quant_params", "GatedQuantParams"), ("pb2_gemm_grouped_params", "GemmGroupedParams"),
    ("pb2_combine_params", "CombineParams"), ("pb2_gated_experts_params", "GatedExpertsParams")])
def test_param_struct_layout_matches_header(cname, pyname):
    assert _c_sizeof(cname) == ctypes.sizeof(getattr(_lib, pyname))


ROUTE = dict(logits=P, logits_type=0, num_tokens=4, num_experts=8, top_k=2, scoring=0, num_groups=1, topk_groups=1,
             scaling=1.0, topk_weights=P, topk_ids=P)
LINEAR = dict(m=4, n=8, k=32, A=P, B=P, A_scales=P, B_scales=P, C=P, c_type=1)
GATED = dict(x=P, x_type=1, m=4, n=8, x_rows=4, xq=P, scales=P, max_val=127)
GROUPED = dict(m=4, n=8, k=32, A=P, B=P, A_scales=P, B_scales=P, C=P, c_type=1, num_experts=2, routing_offsets=P)
COMBINE = dict(slots=P, slots_type=1, topk_weights=P, out=P, type=1, num_tokens=4, top_k=2, n=8)
EXPERTS = dict(x=P, type=1, num_tokens=4, top_k=2, num_experts=2, inner=16, hidden=8, max_val=127, w=P, w_scales=P,
               slot_indices=P, routing_offsets=P, topk_weights=P, out=P, workspace=P, workspace_bytes=1 << 20)


@pytest.mark.parametrize("entry,cls,good,change,status", [
    *[("pb2_route_tokens", _lib.RouteParams, ROUTE, c, BAD) for c in (
        dict(num_tokens=-1), dict(num_experts=0), dict(num_experts=257), dict(top_k=0), dict(top_k=9), dict(num_experts=64, top_k=33),
        dict(num_groups=3), dict(num_groups=0), dict(num_groups=2, topk_groups=3), dict(num_groups=4, topk_groups=1, top_k=3),
        dict(topk_groups=0), dict(logits_type=3), dict(logits_type=-1), dict(scoring=2), dict(logits=None),
        dict(topk_weights=None), dict(topk_ids=None))],
    *[("pb2_gemm_epilogue", _lib.GemmEpilogueParams, LINEAR, c, BAD) for c in (
        dict(m=-1), dict(n=0), dict(k=0), dict(m=1 << 31), dict(c_type=0), dict(c_type=3), dict(activation=5), dict(activation=-1),
        dict(bias=P, bias_type=2), dict(A=None), dict(B=None), dict(A_scales=None), dict(B_scales=None), dict(C=None),
        dict(A=P + 8), dict(B=P + 1))],
    ("pb2_gemm_epilogue", _lib.GemmEpilogueParams, LINEAR, dict(k=24), UNSUPPORTED),
    *[("pb2_quantize_gated", _lib.GatedQuantParams, GATED, c, BAD) for c in (
        dict(m=-1), dict(n=0), dict(x=None), dict(xq=None), dict(scales=None), dict(x_rows=5), dict(x_rows=-1, row_index=P),
        dict(max_val=0), dict(max_val=128), dict(x_type=0), dict(activation=9), dict(x=P + 8), dict(xq=P + 4), dict(smooth=P + 4))],
    *[("pb2_quantize_gated", _lib.GatedQuantParams, GATED, c, UNSUPPORTED) for c in (
        dict(n=12), dict(block_size=4), dict(block_size=16), dict(n=24, block_size=24), dict(n=512, block_size=512))],
    *[("pb2_gemm_grouped", _lib.GemmGroupedParams, GROUPED, c, BAD) for c in (
        dict(m=-1), dict(n=0), dict(num_experts=0), dict(num_experts=257), dict(n=1 << 30, num_experts=4), dict(c_type=3), dict(c_type=-1),
        dict(routing_offsets=None), dict(A=None), dict(B=P + 4), dict(c_row_index=P, c_rows=-1))],
    ("pb2_gemm_grouped", _lib.GemmGroupedParams, GROUPED, dict(k=40), UNSUPPORTED),
    *[("pb2_combine_slots", _lib.CombineParams, COMBINE, c, BAD) for c in (
        dict(num_tokens=-1), dict(top_k=0), dict(n=0), dict(type=0), dict(slots_type=2), dict(slots=None), dict(topk_weights=None), dict(out=None))],
    *[("pb2_gated_experts", _lib.GatedExpertsParams, EXPERTS, c, BAD) for c in (
        dict(num_tokens=-1), dict(top_k=0), dict(num_experts=0), dict(num_experts=257), dict(inner=0), dict(hidden=0), dict(type=0),
        dict(x=None), dict(w=None), dict(w=P + 8), dict(w_scales=None), dict(slot_indices=None), dict(routing_offsets=None),
        dict(topk_weights=None), dict(out=None), dict(workspace=None), dict(workspace_bytes=100), dict(max_val=0),
        dict(num_tokens=1 << 30, top_k=2), dict(activation=7))],
    ("pb2_gated_experts", _lib.GatedExpertsParams, EXPERTS, dict(inner=24), UNSUPPORTED),
    ("pb2_gated_experts", _lib.GatedExpertsParams, EXPERTS, dict(block_size=32), UNSUPPORTED)])
def test_c_abi_refuses(entry, cls, good, change, status):
    p = cls(**{**good, **change})
    assert getattr(_lib.load(), entry)(ctypes.byref(p), None) == status
    assert getattr(_lib.load(), entry)(None, None) == BAD


def test_workspace_bytes():
    f = pg.moe.get_gated_experts_workspace_bytes
    assert f(0, 16, 8) == 0 and f(-1, 16, 8) == 0
    assert f(2, 16, 8) == 3 * 256  # each part in whole 256 bytes
    assert f(1024, 512, 8192) == 1024 * 512 + 1024 * 4 + 1024 * 8192 * 4  # 32 MB of f32 products
    assert f(1025, 512, 8192) == 1025 * 512 + 17 * 256 + 1025 * 8192 * 2
    assert f(16384, 14336, 4096) == 16384 * 14336 + 16384 * 4 + 16384 * 4096 * 2
    assert f(1 << 20, 1 << 14, 1 << 13) == (1 << 34) + (1 << 22) + (1 << 34)


def test_python_entry_points_refuse_cpu_tensors_and_bad_arguments():
    i8, f, h = (lambda *s, dt=dt: torch.zeros(*s, dtype=dt) for dt in (torch.int8, torch.float32, torch.bfloat16))
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(RuntimeError, match="A must be on CUDA"):
        pg.gemm_epilogue(i8(4, 32), i8(8, 32), f(4), f(8), h(4, 8))
    with pytest.raises(RuntimeError, match="k must be a multiple of 16"):
        pg.gemm_epilogue(i8(4, 24), i8(8, 24), f(4), f(8), h(4, 8))
    with pytest.raises(RuntimeError, match="C must be bfloat16 or float16"):
        pg.gemm_epilogue(i8(4, 32), i8(8, 32), f(4), f(8), f(4, 8))
    with pytest.raises(RuntimeError, match="scoring must be"):
        pg.moe.route_tokens(f(4, 8), f(4, 2), i32(4, 2), scoring="tanh")
    with pytest.raises(RuntimeError, match="num_experts must be in"):
        pg.moe.route_tokens(f(4, 300), f(4, 2), i32(4, 2))
    with pytest.raises(RuntimeError, match="top_k must be in"):
        pg.moe.route_tokens(f(4, 8), f(4, 9), i32(4, 9))
    with pytest.raises(RuntimeError, match="num_groups must divide"):
        pg.moe.route_tokens(f(4, 8), f(4, 2), i32(4, 2), num_groups=3)
    with pytest.raises(RuntimeError, match="logits must be on CUDA"):
        pg.moe.route_tokens(f(4, 8), f(4, 2), i32(4, 2))
    with pytest.raises(RuntimeError, match="x must be 2D"):
        pg.quantization.quantize_gated(h(4, 15), i8(4, 8), f(4))
    with pytest.raises(RuntimeError, match="x must be on CUDA"):
        pg.quantization.quantize_gated(h(4, 16), i8(4, 8), f(4))
    with pytest.raises(RuntimeError, match="A must be on CUDA"):
        pg.moe.gemm_grouped(i8(4, 32), i8(2, 8, 32), f(4), f(2, 8), h(4, 8), i32(2))
    with pytest.raises(RuntimeError, match="num_experts must be in"):
        pg.moe.gemm_grouped(i8(4, 32), i8(257, 8, 32), f(4), f(257, 8), h(4, 8), i32(257))
    with pytest.raises(RuntimeError, match="must be on CUDA"):
        pg.moe.combine_slots(h(8, 8), f(4, 2), h(4, 8))
    with pytest.raises(RuntimeError, match="inner must be a multiple of 16"):
        pg.moe.gated_experts(h(8, 48), i8(2, 8, 24), f(2, 8), h(4, 8), i32(8), i32(2), f(4, 2))
    with pytest.raises(ValueError, match="block_size must be 0 or"):
        pg.moe.gated_experts(h(8, 64), i8(2, 8, 32), f(2, 8), h(4, 8), i32(8), i32(2), f(4, 2), block_size=12)
