"""gated_scan where products of its gates leave fp32's or fp64's range and the states do not.

Every number is a product of few powers of two, or zero, so the 64-bit recurrence gives it exactly in
every type and the comparisons are for equality."""
import numpy as np
import pytest

import sequence_oracle as O
from dlf_amd import frontend as F
from dlf_amd.frontend import Tensor
from test_gpu_gated_scan import back, columns, state, stored

pytestmark = pytest.mark.gpu

# (extents, scanned axis): rows along memory by 4, 16, 32 lanes, by one, four and sixteen wavefronts, cut;
# rows side by side by sixteen wavefronts, cut, and whole by 2, 4, 8 and 16
LAYOUTS = [((9, 100), 1), ((5, 200), 1), ((5, 400), 1), ((2100, 700), 1), ((3, 5000), 1), ((2, 9001), 1), ((2, 40000), 1), ((4096, 70), 0),
           ((40, 130), 0), ((100, 130), 0), ((250, 130), 0), ((600, 8200), 0), ((1, 900, 4099), 1)]


def run(hip, kind, dtype, g, x, initial, axis, reverse):
    """The states and the last ones of a call, and the 64-bit ones."""
    extents = g.shape
    kept = extents[:axis] + extents[axis + 1:]
    h0 = np.full(kept, initial, np.float32)
    G, X = O.store(g, dtype), O.store(x, dtype)
    want, _ = O.gated_scan(kind, columns(G, axis, reverse), columns(X, axis, reverse), h0.astype(np.float64).reshape(-1))
    Y, L = F.gated_scan(Tensor.from_numpy(hip, G), Tensor.from_numpy(hip, X), axis, kind, reverse=reverse, initial=state(hip, h0))
    hip.synchronize()
    return O.load(Y.numpy()), L.numpy().reshape(-1), back(want, extents, axis, reverse), want[-1]


def run_grad(hip, kind, dtype, g, dy, dlast, axis, reverse):
    extents = g.shape
    kept = extents[:axis] + extents[axis + 1:]
    G, dY, Y = O.store(g, dtype), O.store(dy, dtype), O.store(np.ones(extents), dtype)
    dl, h0 = np.full(kept, dlast, np.float32), np.ones(kept, np.float32)
    want, _ = O.gated_scan_grad(kind, columns(G, axis, reverse), None, columns(Y, axis, reverse), columns(dY, axis, reverse),
                                h0.astype(np.float64).reshape(-1), dl.astype(np.float64).reshape(-1))
    got = F.gated_scan_grad(Tensor.from_numpy(hip, G), None, Tensor.from_numpy(hip, Y), Tensor.from_numpy(hip, dY), axis, kind, reverse=reverse,
                            initial=state(hip, h0), dlast=state(hip, dl))
    hip.synchronize()
    return [O.load(v.numpy()) for v in got[:2]] + [got[2].numpy().reshape(-1)], [back(w, extents, axis, reverse) for w in want[:2]] + [want[2]]


def along(values, extents, axis, reverse):
    """[n] in scanning order spread over every row."""
    v = values[::-1] if reverse else values
    shape = [1] * len(extents)
    shape[axis] = -1
    return np.broadcast_to(v.reshape(shape), extents).copy()


@pytest.mark.parametrize("extents,axis", LAYOUTS)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_growth_behind_a_reset(hip_backend, extents, axis, reverse, dtype):
    # a gate of 0, then growth by 64 a step (2^1024 after 171 steps) of a state that is 0; a second reset ten
    # steps before the end lets a state of 1 in, which halves
    n = extents[axis]
    g, x = np.full(n, 64.0), np.zeros(n)
    g[0] = g[n // 3] = g[n - 10] = 0.0
    x[n - 10] = 1.0
    g[n - 9:] = 0.5
    y, last, want, want_last = run(hip_backend, "gated", dtype, along(g, extents, axis, reverse), along(x, extents, axis, reverse), 1.0, axis, reverse)
    assert np.array_equal(y, want) and np.array_equal(last, want_last)
    # and from the last step to the first
    got, want = run_grad(hip_backend, "gated", dtype, along(g[::-1], extents, axis, reverse), along(x[::-1], extents, axis, reverse), 1.0, axis, reverse)
    for a, b in zip(got, want):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("extents,axis", LAYOUTS + [((19, 131072), 0)])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_growth_past_fp32_in_a_few_steps(hip_backend, extents, axis, reverse, dtype):
    # factors of 2^20: ten of them take a state from 2^-100 to 2^100, seven overflow a product in fp32; before that a
    # state of 0 under the same factors.  Every fortieth step starts over.
    n = extents[axis]
    t = (np.arange(n) + 7) % 40
    g = np.where(t == 0, 0.0, np.where(t <= 10, 2.0 ** 20, 1.0))
    x = np.where((t == 0) & (np.arange(n) >= 60), 2.0 ** -100, 0.0)
    y, last, want, want_last = run(hip_backend, "gated", dtype, along(g, extents, axis, reverse), along(x, extents, axis, reverse), 0.0, axis, reverse)
    assert np.array_equal(y, want) and np.array_equal(last, want_last)
    # (backwards the state is multiplied after it is added to: lam = 2^-100 at the step before a growth)
    got, want = run_grad(hip_backend, "gated", dtype, along(g[::-1], extents, axis, reverse), along(np.roll(x, 1)[::-1], extents, axis, reverse), 0.0,
                         axis, reverse)
    for a, b in zip(got, want):
        assert np.isfinite(b).all() and np.array_equal(a, b)


@pytest.mark.parametrize("extents,axis", LAYOUTS + [((19, 131072), 0), ((3, 60), 0)])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("kind", ["gated", "gated_sigmoid"])
def test_a_gate_of_nan_shows(hip_backend, extents, axis, reverse, kind):
    # also where the state that it meets is 0: NaN from there on
    n = extents[axis]
    for at in sorted({0, 1, n // 2, n // 2 // 16 * 16, n // 2 // 2048 * 2048, n - 2}):
        g = np.full(n, 0.5)
        g[at] = np.nan
        full, zeros = along(g, extents, axis, reverse), np.zeros(extents)
        y, last, want, want_last = run(hip_backend, kind, "f32", full, zeros, 0.0, axis, reverse)
        assert np.isnan(want).sum() == want.size // n * (n - at)
        assert np.array_equal(y, want, equal_nan=True) and np.array_equal(last, want_last, equal_nan=True), at
        got, want = run_grad(hip_backend, kind, "f32", full, zeros, 0.0, axis, reverse)
        for a, b in zip(got, want):
            assert np.array_equal(np.isnan(a), np.isnan(b)), at


@pytest.mark.parametrize("extents,axis", LAYOUTS + [((37, 131072), 0), ((16, 4100), 0)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_neighbours_of_such_a_row_keep_their_bits(hip_backend, extents, axis, dtype):
    # every seventh row leaves fp32's range within a pass (or fp64's in a product), the others are ordinary: they give what
    # they give beside ordinary rows, and the same when the states are written over the inputs
    n = extents[axis]
    ordinary = stored("gated", 31, extents, dtype, gate=True), stored("gated", 32, extents, dtype)
    rows = int(np.prod(extents)) // n
    kept = extents[:axis] + extents[axis + 1:]
    far = (np.arange(rows) % 7 == 3).reshape(kept)
    t = (np.arange(n) + 5) % 40
    g = along(np.where(t == 0, 0.0, np.where(t <= 10, 2.0 ** 20, 64.0)), extents, axis, False)
    x = along(np.where((t == 0) & (np.arange(n) % 80 < 40), 2.0 ** -300, 0.0), extents, axis, False)      # (0 in both types)
    mask = np.expand_dims(far, axis)
    wild = np.where(mask, O.store(g, dtype), ordinary[0]), np.where(mask, O.store(x, dtype), ordinary[1])
    dY = Tensor.from_numpy(hip_backend, stored("gated", 33, extents, dtype))
    results = []
    for G, X in (ordinary, wild):
        G, X = Tensor.from_numpy(hip_backend, G), Tensor.from_numpy(hip_backend, X)
        Y, L = F.gated_scan(G, X, axis, "gated")
        grads = F.gated_scan_grad(G, None, Y, dY, axis, "gated")
        hip_backend.synchronize()
        results.append([v.numpy() for v in (Y, L) + tuple(grads)])
        over, last = F.gated_scan(G, X, axis, "gated", out=X)
        hip_backend.synchronize()
        assert over.numpy().tobytes() == results[-1][0].tobytes() and last.numpy().tobytes() == results[-1][1].tobytes()
    near = ~far
    for a, b in zip(*results):
        a, b = (np.moveaxis(v, axis, 0) if v.shape == tuple(extents) else v[None] for v in (a.view(np.uint16) if a.dtype == O.TYPES["bf16"] else a,
                                                                                           b.view(np.uint16) if b.dtype == O.TYPES["bf16"] else b))
        assert np.array_equal(a[:, near], b[:, near])
    y = np.moveaxis(O.load(results[1][0]), axis, 0)
    assert (y[:, far] == 0).all()
