"""The sequence-model operators at the ends of their ranges: offsets past 32 bits, more rows than one
axis of a grid has workgroups, first calls inside a recording, lazily conjugated torch views.  Every
result is held to the bounds of the operators' own tests."""
import numpy as np
import pytest

import sequence_oracle as O
import test_gpu_cross_entropy as loss_tests
import test_gpu_gated_scan as scan_tests
import test_gpu_route as route_tests
from dlf_amd import frontend as F
from dlf_amd.frontend import Tensor
from dlf_amd.shape import Shape
from helpers import normal, randint

pytestmark = pytest.mark.gpu

class Far(Tensor):
    def numpy(self):
        return self.contiguous().numpy()         # (not by way of the whole storage)


def spread(hip, values, axis, stride, start, storage):
    """A view of `storage` whose extent along `axis` is walked at `stride`, the others dense from
    `start` on, with the values written to it."""
    import torch
    e = values.shape
    dense = Shape.dense(e[:axis] + e[axis + 1:]).strides
    strides = tuple(dense[:axis]) + (stride,) + tuple(dense[axis:])
    T = Far(hip, Shape.of(e, strides, start), storage, values.dtype)
    flat = np.ascontiguousarray(values)
    host = torch.from_numpy(flat.view(np.int16)).view(torch.bfloat16) if values.dtype == F.BFLOAT16 else torch.from_numpy(flat)
    hip.to_torch(T).copy_(host)
    return T


@pytest.fixture(scope="module")
def far(hip_backend):
    """12.9 GB of bfloat16, reused by every test."""
    import torch
    return torch.empty(3 * 2 ** 31, dtype=torch.bfloat16, device=hip_backend.device)


# (extents, scanned axis, the axis that is walked at `stride`, stride in elements)
FAR = [((3, 40, 70), 1, 0, 2 ** 31 + 3), ((3, 300, 70), 1, 0, 2 ** 31 + 2), ((3, 12, 9), 1, 0, 2 ** 31 + 3), ((3, 5, 600), 2, 0, 2 ** 31 + 1),
       ((23, 66), 0, 0, 2 ** 28 + 1), ((300, 64), 0, 0, 20000003), ((3, 5, 2), 1, 2, 2 ** 31 + 7)]


@pytest.mark.parametrize("extents,axis,far_axis,stride", FAR)
@pytest.mark.parametrize("kind", ["gated", "gated_blend"])
def test_gated_scan_past_32_bits(hip_backend, far, extents, axis, far_axis, stride, kind):
    a = [scan_tests.stored(kind, 40 + i, extents, "bf16", gate=i == 0) for i in range(3)]
    G, X, dY = (spread(hip_backend, v, far_axis, stride, 50000 * i, far) for i, v in enumerate(a))
    out = spread(hip_backend, a[1], far_axis, stride, 50000 * 3, far)
    for reverse in (False, True):
        Y, _ = scan_tests.check_forward(hip_backend, kind, "bf16", (G, a[0]), (X, a[1]), axis, reverse, out=out)
        scan_tests.check_grad(hip_backend, kind, "bf16", (G, a[0]), (X, a[1]), (Y, Y.numpy()), (dY, a[2]), axis, reverse)


def test_rows_past_32_bits(hip_backend, far):
    x = route_tests.logits(3, 3, 60, "bf16")
    X = spread(hip_backend, x, 0, 2 ** 31 + 5, 11, far)
    route_tests.check(hip_backend, "bf16", x, 4, "softmax", X=X, renormalise=True)
    for n in (7, 1000, 20001):
        x = loss_tests.logits(4, 3, n, "bf16")
        t = np.array([n - 1, -1, 0])
        X = spread(hip_backend, x, 0, 2 ** 31 + 5, 11, far)
        T, _, want, grad, lb, gb = loss_tests.check(hip_backend, "bf16", x, t, 1e-4, X=X)
        loss, dX = F.cross_entropy_grad(X, T, None, 1e-4, out=X)                      # in place, far apart
        hip_backend.synchronize()
        assert O.close(dX.numpy(), grad, gb, "bf16") and O.close(loss.numpy(), want, lb, "f32")


@pytest.mark.parametrize("m,n,dtype", [((1 << 20) + 5, 9, "bf16"), ((1 << 21) + 1, 3, "f32")])
def test_more_rows_than_an_axis_of_a_grid(hip_backend, m, n, dtype):
    # the same few rows over and over, so that the oracle computes only those
    few = 1000
    x, t = loss_tests.logits(5, few, n, dtype), loss_tests.targets_of(6, few, n)
    pick = np.arange(m) % few
    values = O.load(x)
    want, grad = O.cross_entropy(values, t)
    lb, gb = loss_tests.loss_bound(values, np.where(np.isfinite(want), want, 0), 0.0), loss_tests.grad_bound(values, grad, t, np.ones(few), 0.0)
    X, T = Tensor.from_numpy(hip_backend, np.ascontiguousarray(x[pick])), Tensor.from_numpy(hip_backend, t[pick])
    state = F.cross_entropy_piece(X, T, 0)
    results = [(F.cross_entropy(X, T), None), F.cross_entropy_grad(X, T),
               (F.cross_entropy_join(state, T), F.cross_entropy_piece_grad(X, T, 0, state))]
    hip_backend.synchronize()
    for loss, dX in results:
        assert O.close(loss.numpy(), want[pick], lb[pick] + 2 * O.U, "f32")
        if dX is not None:
            assert O.close(dX.numpy(), grad[pick], gb[pick] * (1 + 1e-6) + 2 * O.U * (1 + np.abs(grad[pick])), dtype)


def test_first_calls_inside_a_recording(hip_backend):
    # sizes of this test alone: kernels may be loaded, and their occupancy asked for, while recording
    import torch
    x = [normal(7 + i, 300 * n).astype(np.float16).reshape(300, n) for i, n in enumerate((90000, 130000))]
    t = [randint(9, 300, 0, v.shape[1]) for v in x]
    D = [(Tensor.from_numpy(hip_backend, a), Tensor.from_numpy(hip_backend, b)) for a, b in zip(x, t)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = [F.cross_entropy_grad(X, T) for X, T in D]
    for _ in range(3):
        for loss, dX in recorded:
            loss.storage.zero_()
            dX.storage.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for (X, T), (loss, dX) in zip(D, recorded):
            l, d = F.cross_entropy_grad(X, T)
            hip_backend.synchronize()
            assert torch.equal(l.storage, loss.storage) and torch.equal(d.storage, dX.storage)
    want, _ = O.cross_entropy(O.load(x[0][:8]), t[0][:8])
    assert np.abs(recorded[0][0].numpy()[:8] - want).max() < 1e-3


def test_views_that_torch_changes_when_read_are_refused(hip_backend):
    import torch
    z = torch.zeros(4, dtype=torch.complex64, device=hip_backend.device)
    with pytest.raises(ValueError):
        hip_backend.from_torch(z.conj())
    with pytest.raises(ValueError):
        hip_backend.from_torch(z.conj().imag)
    assert hip_backend.from_torch(z.conj().resolve_conj()).size == 4


# (extents, scanned axis): rows in pairs, on whole cache lines and off them, odd; two, four, eight wavefronts to them
MANY = [((19, 131072), 0), ((37, 131074), 0), ((5, 131073), 0), ((70, 131073), 0), ((3, 17, 65536), 1), ((2, 33, 65601), 1), ((130, 131075), 0),
        ((5, 70), 0), ((33, 70), 0), ((90, 70), 0), ((129, 130), 0), ((200, 70), 0), ((256, 66), 0), ((257, 66), 0)]


@pytest.mark.parametrize("extents,axis", MANY)
@pytest.mark.parametrize("kind,dtype", [("gated_blend", "bf16"), ("gated_exp", "f16"), ("gated_sigmoid", "f32")])
def test_many_columns_and_every_width(hip_backend, extents, axis, kind, dtype):
    a = [scan_tests.stored(kind, 60 + i, extents, dtype, gate=i == 0) for i in range(3)]
    G, X, dY = (scan_tests.pair(hip_backend, v) for v in a)
    kept = extents[:axis] + extents[axis + 1:]
    initial = normal(63, int(np.prod(kept))).astype(np.float32).reshape(kept)
    for reverse in (False, True):
        Y, _ = scan_tests.check_forward(hip_backend, kind, dtype, G, X, axis, reverse, initial)
        scan_tests.check_grad(hip_backend, kind, dtype, G, X if kind == "gated_blend" else None, (Y, Y.numpy()), dY, axis, reverse, initial, initial)
