"""CPU stand-ins that show what the Python layer would launch."""
from types import SimpleNamespace

from eider_b200 import _lib, ops


def without_a_device(monkeypatch):
    """Lets CPU tensors through ops' device checks, its other checks as they are; returns the list of entry points that were called."""
    called = []

    class Recorder:
        def __getattr__(self, name):
            def entry(*args):
                called.append(name)
                return 0
            return entry

    def need(t, dtype, label):
        if not t.is_contiguous() or t.dtype != dtype:
            raise ops.ShapeError(f"{label}: expected contiguous {dtype}, got {t.dtype}")

    monkeypatch.setattr(_lib, "load", Recorder)
    monkeypatch.setattr(ops, "_need", need)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(ops.torch.cuda, "current_device", lambda: None)  # (a CPU tensor's device has no index)
    return called


def routes(count, device="cpu"):
    import torch
    return SimpleNamespace(route_to_sorted=torch.zeros(count, dtype=torch.int32, device=device))
