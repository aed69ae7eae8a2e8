"""from_torch and torch's autograd: no GPU (the views are made of host arithmetic alone)."""
import pytest
import torch

from dlf_amd.hip_backend import HipBackend


@pytest.fixture
def backend():
    b = HipBackend.__new__(HipBackend)
    b.torch, b.device, b._from_torch_dtype = torch, torch.device("cpu"), None
    return b


def test_a_tensor_that_requires_a_gradient(backend):
    leaf = torch.ones(3, 4, requires_grad=True)
    for t in (leaf, leaf[1:], 2 * leaf, torch.nn.Parameter(torch.zeros(2))):
        with pytest.raises(ValueError, match="detach"):
            backend.from_torch(t)
        for off in (torch.no_grad, torch.inference_mode):
            with off():
                T = backend.from_torch(t)
                assert T.shape.extents == tuple(t.shape) and T.storage.data_ptr() == t.data_ptr()
        assert not backend.to_torch(backend.from_torch(t.detach())).requires_grad


def test_inside_an_autograd_function(backend):
    class Twice(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return 2 * backend.to_torch(backend.from_torch(x))

        @staticmethod
        def backward(ctx, dy):
            return 2 * backend.to_torch(backend.from_torch(dy))
    x = torch.ones(5, requires_grad=True)
    Twice.apply(x).sum().backward()
    assert torch.equal(x.grad, torch.full((5,), 2.0))
