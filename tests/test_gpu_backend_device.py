"""A backend named without a device number is that of the current one."""
import pytest

pytestmark = pytest.mark.gpu


def test_a_backend_of_the_current_device():
    import torch
    from dlf_amd.hip_backend import HipBackend
    hip = HipBackend("cuda")
    t = torch.arange(6, device="cuda", dtype=torch.float32)
    assert hip.device == t.device and hip.from_torch(t).numpy().tolist() == [0, 1, 2, 3, 4, 5]
