"""What the Python layer of the routed layers refuses before anything is launched."""
import pytest
import torch

from eider_b200 import ops
from tests import fakes


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_combine_takes_what_fits(monkeypatch, dtype):
    called = fakes.without_a_device(monkeypatch)
    rows, weights = torch.zeros(8, 64, dtype=torch.bfloat16), torch.zeros(8)
    for out in (torch.zeros(4, 64, dtype=dtype), *([None] if dtype == torch.float32 else [])):
        y = ops.moe_weighted_accumulate(fakes.routes(8), weights, rows, 4, 2, out=out)
        assert y.shape == (4, 64) and y.dtype == dtype and (out is None or y is out)
    kernel = "infer_moe_weighted_accumulate_sorted_bf16_batch_on_stream" if dtype == torch.float32 else "eider_b200_moe_weighted_accumulate_sorted_to_bf16_on_stream"
    assert set(called) == {kernel}


@pytest.mark.parametrize("change", [{"out": torch.zeros(4, 64, dtype=torch.float16)}, {"out": torch.zeros(3, 64)}, {"out": torch.zeros(3, 64, dtype=torch.bfloat16)},
                                    {"out": torch.zeros(4, 63)}, {"out": torch.zeros(256)}, {"out": torch.zeros(64, 4).t()}, {"out": torch.zeros(4, 64, dtype=torch.float64)},
                                    {"weights": torch.zeros(7)}, {"rows": torch.zeros(7, 64, dtype=torch.bfloat16)}, {"rows": torch.zeros(512, dtype=torch.bfloat16)},
                                    {"routes": fakes.routes(7)}])
def test_combine_refuses(monkeypatch, change):
    """An output of another type, shape or layout would be written past its end, missing weights, rows or routes read past theirs."""
    called = fakes.without_a_device(monkeypatch)
    a = {"out": torch.zeros(4, 64), "weights": torch.zeros(8), "rows": torch.zeros(8, 64, dtype=torch.bfloat16), "routes": fakes.routes(8)} | change
    with pytest.raises(ops.ShapeError):
        ops.moe_weighted_accumulate(a["routes"], a["weights"], a["rows"], 4, 2, out=a["out"])
    assert not called
