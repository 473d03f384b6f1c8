"""Beam search refusals that need no GPU."""
import ctypes as C

import pytest
import torch

from eider_b200 import _lib, ops

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
