"""Beam search refusals that need no GPU."""
import ctypes as C
import types

import pytest
import torch

from eider_b200 import _lib, ops
from tests import fakes

INVALID = 1
SOME = 0x1000


@pytest.mark.parametrize("change", [{"logits": None}, {"logits": SOME + 2}, {"scores": None}, {"out": None}, {"work": None}, {"work": SOME + 4}, {"bytes": 10},
                                    {"batch": 0}, {"beams": 0}, {"beams": 65}, {"vocab": 0}, {"k": 0}, {"k": 129}, {"k": 33, "vocab": 8}, {"stride": 99},
                                    {"pad": 100}, {"batch": 20000}, {"vocab": 0x7fffffff, "stride": 0x7fffffff}])
def test_select_refuses(change):
    a = {"logits": SOME, "stride": 100, "scores": SOME, "fin": SOME, "pad": 0, "out": SOME, "batch": 2, "beams": 4, "vocab": 100, "k": 8, "work": SOME,
         "bytes": 1 << 40} | change
    assert _lib.load().eider_b200_beam_select_on_stream(a["logits"], 0, a["stride"], a["scores"], a["fin"], a["pad"], a["out"], a["out"], a["out"],
                                                        a["batch"], a["beams"], a["vocab"], a["k"], a["work"], a["bytes"], None) == INVALID


def test_workspace():
    f = _lib.load().eider_b200_beam_select_workspace_bytes
    assert f(0, 4, 100, 0) == 0 and f(1, 65, 100, 0) == 0 and f(1, 1, 0, 0) == 0
    # a float per 64 logits of every row (and its lead to a 16-byte boundary), and a pair of floats per split
    for batch, beams, vocab in ((1, 1, 1), (1, 4, 32000), (64, 8, 151936)):
        rows = batch * beams
        assert rows * 4 * (vocab // 64) <= f(batch, beams, vocab, 1) <= rows * (4 * (vocab // 64 + 2) + 8 * 600)


def test_reorder_refuses():
    f = _lib.load().eider_b200_beam_reorder_on_stream
    ptrs, sizes = (C.c_void_p * 2), (C.c_size_t * 2)
    src, dst, rows = ptrs(0x10000, 0x20000), ptrs(0x30000, 0x40000), sizes(64, 64)
    assert f(None, dst, rows, 2, SOME, 4, 2, 4, None) == INVALID
    assert f(src, dst, rows, 0, SOME, 4, 2, 4, None) == INVALID
    assert f(src, dst, rows, 2, None, 4, 2, 4, None) == INVALID
    assert f(src, dst, rows, 2, SOME, 3, 2, 4, None) == INVALID
    assert f(src, dst, rows, 2, SOME, 4, 0, 4, None) == INVALID
    assert f(src, ptrs(0x30000, 0), rows, 2, SOME, 4, 2, 4, None) == INVALID
    assert f(src, dst, sizes(64, 0), 2, SOME, 4, 2, 4, None) == INVALID
    assert f(src, ptrs(0x30000, 0x20000 + 64), rows, 2, SOME, 4, 2, 4, None) == INVALID  # overlaps its source


def test_python_layer_refuses():
    with pytest.raises(ops.ShapeError):
        ops.beam_search_select(torch.zeros(1, 2, 8), torch.zeros(1, 2), 2)
    with pytest.raises(ops.ShapeError):
        ops.beam_search_reorder([torch.zeros(1, 2, 8)], torch.zeros(1, 2, dtype=torch.int32))


def test_reorder_refuses_outputs_over_any_state():
    """All states are copied at once, so an output may lie over no state and over no other output; states may share memory."""
    f = _lib.load().eider_b200_beam_reorder_on_stream
    ptrs, sizes = (C.c_void_p * 3), (C.c_size_t * 3)
    rows, size = sizes(64, 64, 64), 64 * 8
    a, b, c, d = (0x10000 + i * size for i in range(4))  # back to back
    for src, dst in (((a, b, c), (b, c, d)), ((a, b, c), (d, a, 0x40000)), ((a, b, c), (0x40000, 0x40000 + size - 16, 0x50000)), ((a, b, c), (0x40000, 0x50000, c + 16)),
                     ((a, a, a), (0x40000, 0x50000, 0x40000)), ((a, b, c), (0x40000, 0x50000, a - size + 1))):
        assert f(ptrs(*src), ptrs(*dst), rows, 3, SOME, 4, 2, 4, None) == INVALID, (src, dst)
    # an output that is long enough to reach over what lies behind it
    assert f(ptrs(a, b, 0x50000), ptrs(c, d, a), sizes(64, 64, 192), 3, SOME, 4, 2, 4, None) == INVALID


def test_python_reorder_refuses_outputs_over_any_state(monkeypatch):
    called = fakes.without_a_device(monkeypatch)
    parents = types.SimpleNamespace(dim=lambda: 2, is_cuda=True, dtype=torch.int32, numel=lambda: 8, stride=lambda i: (4, 1)[i], shape=(2, 4), device=torch.device("cpu"),
                                    data_ptr=lambda: SOME)
    buffer = torch.zeros(4, 2, 4, 16)
    a, b, c, d = buffer
    for states, out in (([a, b], [b, c]), ([a, b], [c, a]), ([a, b], [c, c]), ([a], [a]), ([a, b], [c, buffer.flatten()[8:136].view(2, 4, 16)])):
        with pytest.raises(ops.ShapeError):
            ops.beam_search_reorder(states, parents, out=out)
    assert not called
    ops.beam_search_reorder([a, c], parents, out=[b, d])
    ops.beam_search_reorder([a, a], parents, out=[b, d])
    assert called == ["eider_b200_beam_reorder_on_stream"] * 2
