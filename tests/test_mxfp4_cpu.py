"""MXFP4 refusals that need no GPU: every entry point turns bad arguments into cudaErrorInvalidValue (1) or a null plan before it
touches the device, and the Python layer into ShapeError."""
import pytest
import torch

from eider_b200 import _lib, ops
from tests import fakes

INVALID = 1
SOME = 0x1000  # an aligned address that nothing reads


def test_layout_length():
    lib = _lib.load()
    for outer, inner in ((1, 32), (128, 128), (129, 160), (300, 2880), (5, 13824)):
        assert lib.eider_b200_mxfp4_scale_layout_len(outer, inner) == ops.mxfp4_scale_layout_len(outer, inner)
        # the NVFP4 layout of half the row length
        assert ops.mxfp4_scale_layout_len(outer, inner) == lib.eider_b200_nvfp4_scale_layout_len(outer, inner // 2)


@pytest.mark.parametrize("change", [{"x": None}, {"packed": None}, {"scales": None}, {"tokens": 0}, {"k": 0}, {"k": 48}, {"stride": 32}, {"x": SOME + 1},
                                    {"packed": SOME + 2}, {"scales": SOME + 8}, {"tokens": 0xffffffff, "k": 0xffffffe0, "stride": 0xffffffe0}])
def test_quantizer_refuses(change):
    a = {"x": SOME, "stride": 64, "packed": SOME, "scales": SOME, "tokens": 4, "k": 64} | change
    assert _lib.load().eider_b200_quantize_mxfp4_on_stream(a["x"], 1, a["stride"], a["packed"], a["scales"], a["tokens"], a["k"], None) == INVALID


def test_other_quantizers_refuse():
    lib = _lib.load()
    assert lib.eider_b200_quantize_mxfp4_weight_on_stream(SOME, 1, SOME, SOME, 4, 40, None) == INVALID
    assert lib.eider_b200_quantize_mxfp4_weight_on_stream(None, 1, SOME, SOME, 4, 64, None) == INVALID
    assert lib.eider_b200_silu_mul_halves_quantize_mxfp4_on_stream(SOME + 4, SOME, SOME, 4, 64, None) == INVALID
    assert lib.eider_b200_silu_mul_halves_quantize_mxfp4_on_stream(SOME, SOME, SOME, 4, 48, None) == INVALID
    assert lib.eider_b200_dequantize_mxfp4_on_stream(SOME, SOME, SOME + 4, 1, 4, 64, None) == INVALID
    assert lib.eider_b200_dequantize_mxfp4_on_stream(SOME, SOME, SOME, 1, 0, 64, None) == INVALID
    assert lib.eider_b200_mxfp4_scales_to_tiled_on_stream(SOME, SOME, 0, 4, 64, None) == INVALID
    assert lib.eider_b200_mxfp4_scales_to_tiled_on_stream(SOME, SOME, 1, 4, 65, None) == INVALID


def test_route_quantizer_refuses():
    f = _lib.load().eider_b200_moe_quantize_routes_mxfp4_on_stream
    good = [SOME, 1, SOME, SOME, SOME, SOME, SOME, SOME, 4, 2, 64, 512, None]
    for at, value in ((0, None), (0, SOME + 8), (2, None), (5, None), (6, SOME + 2), (7, SOME + 2), (8, 0), (9, 0), (9, 65), (10, 80), (11, 256), (11, 1024)):
        args = list(good)
        args[at] = value
        assert f(*args) == INVALID, (at, value)


def test_products_refuse():
    lib = _lib.load()
    assert lib.eider_b200_mxfp4_gemm_tn_supported(5, 7, 32) == 1
    for shape in ((0, 8, 32), (8, 0, 32), (8, 8, 0), (8, 8, 48)):
        assert lib.eider_b200_mxfp4_gemm_tn_supported(*shape) == 0
        assert not lib.eider_b200_mxfp4_gemm_tn_create(*shape)
    assert lib.eider_b200_mxfp4_gemm_tn_on_stream(None, SOME, SOME, SOME, SOME, None, SOME, 1.0, 0.0, 1, None) == INVALID
    assert lib.eider_b200_mxfp4_gemm_tn_silu_quantize_on_stream(None, SOME, SOME, SOME, SOME, 1.0, SOME, SOME, None) == INVALID
    for shape in ((0, 8, 32), (65, 8, 32), (1, 0, 32), (1, 8, 40), (1, 8, 65568)):
        assert not lib.eider_b200_mxfp4_decode_create(*shape)
    assert lib.eider_b200_mxfp4_w4a16_gemv_on_stream(None, SOME, 1, 1, SOME, SOME, 16, SOME, None, SOME, 0.0, 1, SOME, 1 << 20, None) == INVALID
    assert lib.eider_b200_mxfp4_w4a16_workspace_bytes(5, 64, 1) == 128 + 5 * 64 * 2 and lib.eider_b200_mxfp4_w4a16_workspace_bytes(64, 64, 0) == 256 + 64 * 64 * 4
    assert lib.eider_b200_mxfp4_w4a16_workspace_bytes(9, 256, 1) == 2 * (2 * 16 * 128 + 512)
    assert lib.eider_b200_mxfp4_grouped_gemm_supported(96, 10, 160, 3) == 1
    for shape in ((48, 10, 64, 3), (96, 10, 80, 3), (96, 0, 64, 3), (96, 10, 64, 0), (1 << 20, 10, 64, 4096)):
        assert lib.eider_b200_mxfp4_grouped_gemm_supported(*shape) == 0
        assert not lib.eider_b200_mxfp4_grouped_gemm_create(*shape)
    assert lib.eider_b200_mxfp4_grouped_gemm_on_stream(None, SOME, SOME, SOME, SOME, SOME, SOME, SOME, 4, None) == INVALID
    assert lib.eider_b200_mxfp4_grouped_gemm_silu_quantize_on_stream(None, SOME, SOME, SOME, SOME, SOME, SOME, 4, SOME, SOME, 512, None) == INVALID


def test_python_layer_refuses_host_tensors_and_odd_shapes():
    u8 = torch.uint8
    with pytest.raises(ops.ShapeError):
        ops.quantize_mxfp4(torch.zeros(4, 64))
    with pytest.raises(ops.ShapeError):
        ops.silu_mul_halves_quantize_mxfp4(torch.zeros(4, 96))
    with pytest.raises(ops.ShapeError):
        ops.Mxfp4Weight.from_checkpoint(torch.zeros(4, 32, dtype=u8), torch.zeros(4, 3, dtype=u8))
    with pytest.raises(ops.ShapeError):
        ops.Mxfp4Weight.from_checkpoint(torch.zeros(4, 24, dtype=u8), torch.zeros(4, 1, dtype=u8))
    with pytest.raises(ops.ShapeError):
        ops.Mxfp4Weight.quantize(torch.zeros(4, 40))
    with pytest.raises(ops.ShapeError):
        ops.GroupedMxfp4Weights.from_checkpoint(torch.zeros(2, 48, 16, dtype=u8), torch.zeros(2, 48, 1, dtype=u8))
    with pytest.raises(ops.ShapeError):
        ops.MoeSortedMxfp4Rows(4, 2, 48, device="cpu")
    with pytest.raises(ops.ShapeError):
        ops.GroupedMoe(4, 2, 1, 64, 32, device="cpu", weight_format="mxfp6")


def test_gate_up_weights_know_their_order(monkeypatch):
    """Weights that have not been through interleave_gate_up() have the class and shape of those that have, and would give another layer."""
    called = fakes.without_a_device(monkeypatch)
    u8 = torch.uint8
    gate_up = ops.GroupedMxfp4Weights.from_checkpoint(torch.zeros(2, 128, 32, dtype=u8), torch.zeros(2, 128, 2, dtype=u8))
    down = ops.GroupedMxfp4Weights.from_checkpoint(torch.zeros(2, 64, 32, dtype=u8), torch.zeros(2, 64, 2, dtype=u8))
    interleaved = gate_up.interleave_gate_up()
    assert not gate_up.gate_up_interleaved and interleaved.gate_up_interleaved
    assert ops.GroupedMxfp4Weights.from_checkpoint(interleaved.packed, interleaved.scales_row_major, gate_up_interleaved=True).gate_up_interleaved
    with pytest.raises(ops.ShapeError):
        interleaved.interleave_gate_up()

    plan = object.__new__(ops.Mxfp4GroupedGemmPlan)
    plan._plan, plan.m, plan.max_n, plan.k, plan.groups, plan.device = None, 128, 4, 64, 2, torch.device("cpu")
    rows, out, routes = ops.MoeSortedMxfp4Rows(4, 2, 64, "cpu"), ops.MoeSortedMxfp4Rows(4, 2, 64, "cpu"), ops.MoeSortedRoutes(4, 2, "cpu")
    called.clear()
    with pytest.raises(ops.ShapeError):
        plan.run_silu_quantize(rows, gate_up, routes, out)
    assert not called
    plan.run_silu_quantize(rows, interleaved, routes, out)
    assert called == ["eider_b200_mxfp4_grouped_gemm_silu_quantize_on_stream"]

    moe = object.__new__(ops.GroupedMoe)
    moe.weight_format, moe.tokens, moe.experts, moe.hidden, moe.out = "mxfp4", 4, 2, 64, torch.zeros(4, 64)
    called.clear()
    for w_gate_up, w_down in ((gate_up, down), (None, down), (interleaved, interleaved)):
        with pytest.raises(ops.ShapeError):
            moe.run(torch.zeros(4, 64), torch.zeros(4, 2), gate_up, w_down, w_gate_up_interleaved=w_gate_up)
    assert not called


def test_decode_status_refuses():
    import ctypes as C
    lib = _lib.load()
    assert lib.eider_b200_mxfp4_decode_status(None, C.byref(C.c_uint32(0))) == INVALID and lib.eider_b200_mxfp4_decode_status(SOME, None) == INVALID


def test_beta_wants_something_to_add(monkeypatch):
    """Without C and without an output that holds it, what beta multiplies would be memory that nobody has written."""
    called = fakes.without_a_device(monkeypatch)
    u8 = torch.uint8
    w = ops.Mxfp4Weight.from_checkpoint(torch.zeros(8, 32, dtype=u8), torch.zeros(8, 2, dtype=u8))
    x = ops.Mxfp4Matrix(torch.zeros(4, 32, dtype=u8), torch.zeros(512, dtype=u8), 4, 64)
    gemm, decode = object.__new__(ops.Mxfp4MatmulPlan), object.__new__(ops.Mxfp4DecodePlan)
    gemm._plan, gemm.device, gemm.m, gemm.n, gemm.k = None, torch.device("cpu"), 4, 8, 64
    decode._plan, decode.device, decode.max_tokens, decode.n, decode.k = None, torch.device("cpu"), 4, 8, 64
    for plan, a in ((gemm, x), (decode, torch.zeros(4, 64))):
        called.clear()
        with pytest.raises(ops.ShapeError):
            plan.run(a, w, beta=1.0)
        assert not called
        plan.run(a, w, beta=1.0, c=torch.zeros(4, 8, dtype=torch.bfloat16))
        plan.run(a, w, beta=1.0, out=torch.zeros(4, 8))
        assert len(called) == 2
