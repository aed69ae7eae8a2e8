"""The sequence-model operators on a backend whose device is not the current one: every call of the library, the copies
of views that it cannot read included, is made with that device current.  No GPU: a library that only notes."""
import pytest
import torch

from dlf_amd import frontend as F
from dlf_amd.hip_backend import HipBackend


class Notes:
    def __init__(self, state):
        self.state, self.calls = state, []

    def __getattr__(self, name):
        def call(*args):
            if name.endswith("_bytes"):
                return 0
            self.calls.append((name, self.state["device"]))
            return 0
        return call


@pytest.fixture
def elsewhere(monkeypatch):
    state = {"device": 1}

    class Device:
        def __init__(self, device):
            pass

        def __enter__(self):
            self.before, state["device"] = state["device"], 0

        def __exit__(self, *_):
            state["device"] = self.before
    monkeypatch.setattr(torch.cuda, "current_device", lambda: state["device"])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: type("Stream", (), {"cuda_stream": 0}))
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 0, raising=False)
    b = HipBackend.__new__(HipBackend)
    b.torch, b.device, b.lib, b._from_torch_dtype = torch, torch.device("cpu"), Notes(state), None
    return b


def test_copies_of_views_and_calls(elsewhere):
    D = elsewhere.from_torch
    x, t, v = torch.zeros(8, 6).t(), torch.zeros(12, dtype=torch.int64)[::2], torch.zeros(12)[::2]
    F.cross_entropy_grad(D(x), D(t), D(v))
    F.route(D(x), 2, bias=D(torch.zeros(16)[::2]))
    F.route_grad(D(x), D(torch.zeros(2, 6, dtype=torch.int32).t()), D(torch.zeros(2, 6).t()))
    F.gated_scan(D(x), D(x), 0)
    names = [name for name, _ in elsewhere.lib.calls]
    assert names.count("dlfx_copy") == 3 + 2 + 3 and len(set(names)) == 5
    assert {device for _, device in elsewhere.lib.calls} == {0}
