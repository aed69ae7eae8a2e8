"""gated_scan and its gradient against the 64-bit recurrence (sequence_oracle.py, which derives the
bounds), over layouts, lengths around the sizes at which the kernels cut an axis, and edge values."""
import numpy as np
import pytest

import sequence_oracle as O
from dlf_amd import frontend as F
from dlf_amd.frontend import Tensor
from dlf_amd.shape import Shape
from helpers import normal, uniform01

pytestmark = pytest.mark.gpu

KINDS = F.GATE_KINDS


def gate_values(kind, seed, count):
    g = 1.5 * normal(seed, count) + 2.0
    starts = uniform01(seed + 900, count) < 0.004
    if kind == "gated":
        return np.where(starts, 0.0, np.where(uniform01(seed + 901, count) < 0.1, -0.9, 1.0) * O.sigmoid(g))
    if kind == "gated_exp":
        return np.where(starts, -np.inf, -np.log1p(np.exp(-g)))
    return np.where(starts, -np.inf, g)


def stored(kind, seed, shape, dtype, gate=False):
    count = int(np.prod(shape))
    v = gate_values(kind, seed, count) if gate else normal(seed, count)
    return O.store(v.reshape(shape), dtype)


def columns(a, axis, reverse):
    """[n, m] in 64 bits, in scanning order."""
    a = np.moveaxis(O.load(a), axis, 0)
    a = a.reshape(a.shape[0], -1)
    return a[::-1] if reverse else a


def back(c, extents, axis, reverse):
    c = c[::-1] if reverse else c
    rest = tuple(extents[:axis]) + tuple(extents[axis + 1:])
    return np.moveaxis(c.reshape((extents[axis],) + rest), 0, axis)


def check_forward(hip, kind, dtype, G, X, axis, reverse=False, initial=None, **tensors):
    """G, X: (Tensor, its values as an array of the stored type)."""
    extents = X[1].shape
    axis %= len(extents)
    kept = extents[:axis] + extents[axis + 1:]
    h0 = np.zeros(int(np.prod(kept)) if kept else 1) if initial is None else initial.astype(np.float64).reshape(-1)
    want, err = O.gated_scan(kind, columns(G[1], axis, reverse), columns(X[1], axis, reverse), h0)
    Y, L = F.gated_scan(G[0], X[0], axis, kind, reverse=reverse,
                        initial=None if initial is None else state(hip, initial), **tensors)
    hip.synchronize()
    y, last = Y.numpy(), L.numpy()
    assert y.shape == tuple(extents) and last.shape == tuple(kept)
    assert O.close(y, back(want, extents, axis, reverse), back(err, extents, axis, reverse), dtype), "states"
    assert O.close(last.reshape(-1), want[-1], err[-1], "f32"), "last state"
    return Y, L


def check_grad(hip, kind, dtype, G, X, Y, dY, axis, reverse=False, initial=None, dlast=None):
    extents = Y[1].shape
    axis %= len(extents)
    kept = extents[:axis] + extents[axis + 1:]
    zero = np.zeros(int(np.prod(kept)) if kept else 1)
    h0 = zero if initial is None else initial.astype(np.float64).reshape(-1)
    dl = zero if dlast is None else dlast.astype(np.float64).reshape(-1)
    x = columns(X[1], axis, reverse) if X is not None else None
    want, err = O.gated_scan_grad(kind, columns(G[1], axis, reverse), x, columns(Y[1], axis, reverse), columns(dY[1], axis, reverse), h0, dl)
    got = F.gated_scan_grad(G[0], X[0] if X is not None else None, Y[0], dY[0], axis, kind, reverse=reverse,
                            initial=None if initial is None else state(hip, initial),
                            dlast=None if dlast is None else state(hip, dlast))
    hip.synchronize()
    for what, g, w, e in zip(("dgate", "dx"), got, want, err):
        assert O.close(g.numpy(), back(w, extents, axis, reverse), back(e, extents, axis, reverse), dtype), what
    assert O.close(got[2].numpy().reshape(-1), want[2], err[2], "f32"), "dinitial"
    return got


def pair(hip, a):
    return Tensor.from_numpy(hip, a), a


def state(hip, a):
    """A tensor of one value per row (from_numpy gives a single value an axis)."""
    return Tensor.from_numpy(hip, a).view(Shape(a.shape))


# (extents, axis): one step; a few; around 16, 128, 256, 512, 2048; few and many columns; time innermost
SHAPES = [
    ((1,), 0), ((5,), 0), ((1, 1, 1), 1), ((3, 1, 70), 1), ((2, 2, 65), 1), ((2, 15, 64), 1), ((1, 16, 3), 1), ((2, 17, 130), 1),
    ((1, 127, 66), 1), ((3, 128, 5), 1), ((1, 257, 192), 1), ((2, 511, 31), 1), ((1, 513, 258), 1), ((1, 2049, 70), 1), ((1, 4500, 8), 1),
    ((4, 7), 1), ((3, 64), 1), ((2, 3, 509), 2), ((5, 513), 1), ((2, 2048), 1), ((3, 2051), 1), ((1, 9001), 1), ((700, 33), 0), ((40, 3, 5, 2), 0),
    ((2100, 300), 1), ((2, 300, 1100), 2), ((2, 40001), 1), ((1, 20000, 3), 1),
]


@pytest.mark.parametrize("extents,axis", SHAPES)
@pytest.mark.parametrize("kind,dtype", [("gated", "f32"), ("gated_exp", "f16"), ("gated_sigmoid", "bf16"), ("gated_blend", "f32"),
                                        ("gated_blend", "bf16")])
def test_forward_and_gradient(hip_backend, extents, axis, kind, dtype):
    seed = sum(extents) + axis
    kept = extents[:axis] + extents[axis + 1:]
    initial = normal(seed + 1, int(np.prod(kept)) if kept else 1).astype(np.float32).reshape(kept)
    dlast = normal(seed + 2, initial.size).astype(np.float32).reshape(kept)
    G, X, dY = (pair(hip_backend, stored(kind, seed + i, extents, dtype, gate=i == 3)) for i in (3, 4, 5))
    for reverse in (False, True):
        Y, _ = check_forward(hip_backend, kind, dtype, G, X, axis, reverse, initial)
        check_grad(hip_backend, kind, dtype, G, X if kind == "gated_blend" else None, (Y, Y.numpy()), dY, axis, reverse, initial, dlast)
    check_forward(hip_backend, kind, dtype, G, X, axis)
    check_grad(hip_backend, kind, dtype, G, X, (Y, Y.numpy()), dY, axis)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("extents,axis", [((2, 1400, 96), 1), ((1, 3000, 7), 1), ((6, 2500), 1), ((1, 700, 4099), 1), ((2, 40, 8200), 1), ((300, 600), 1),
                                          ((2100, 310), 1), ((3, 33000), 1), ((520, 1100), 1), ((1, 70, 66000), 1)])
def test_every_kind_and_type(hip_backend, kind, dtype, extents, axis):
    seed = 50 + sum(extents)
    kept = extents[:axis] + extents[axis + 1:]
    initial = normal(seed + 1, int(np.prod(kept))).astype(np.float32).reshape(kept)
    G, X, dY = (pair(hip_backend, stored(kind, seed + i, extents, dtype, gate=i == 3)) for i in (3, 4, 5))
    Y, _ = check_forward(hip_backend, kind, dtype, G, X, axis, initial=initial)
    check_grad(hip_backend, kind, dtype, G, X, (Y, Y.numpy()), dY, axis, initial=initial)


@pytest.mark.parametrize("kind", ["gated_exp", "gated_blend"])
def test_views(hip_backend, kind):
    # steps of 2 along time, a column slice that starts at an odd element, a transposed input, a shared gate
    dtype = "bf16"
    base = stored(kind, 71, (3, 600, 75), dtype, gate=True)
    G = (Tensor.from_numpy(hip_backend, base).slice([1, 3], [600, 73], [1, 2], [2, 1]), base[:, 1:600:2, 3:73])
    raw = stored(kind, 72, (3, 70, 300), dtype)
    X = (Tensor.from_numpy(hip_backend, raw).transpose([0, 2, 1]), raw.transpose(0, 2, 1))
    Y, _ = check_forward(hip_backend, kind, dtype, G, X, 1)
    dY = pair(hip_backend, stored(kind, 73, (3, 300, 70), dtype))
    check_grad(hip_backend, kind, dtype, G, X, (Y, Y.numpy()), dY, 1)
    # one gate for every 10 columns (stride 0): the gradient is per column, its sum the shared gate's
    shared = stored(kind, 74, (3, 300, 7), dtype, gate=True)
    T = Tensor.from_numpy(hip_backend, shared)
    G4 = T.view(Shape((3, 300, 7, 10), (2100, 7, 1, 0)))
    full = np.repeat(shared[..., None], 10, axis=-1)
    X4 = pair(hip_backend, stored(kind, 75, (3, 300, 7, 10), dtype))
    Y4, _ = check_forward(hip_backend, kind, dtype, (G4, full), X4, 1)
    dY4 = pair(hip_backend, stored(kind, 76, (3, 300, 7, 10), dtype))
    check_grad(hip_backend, kind, dtype, (G4, full), X4, (Y4, Y4.numpy()), dY4, 1)


@pytest.mark.parametrize("extents,axis", [((2, 900, 130), 1), ((1, 5000, 40), 1), ((3, 4000), 1), ((1, 1, 300), 1), ((70, 9), 1)])
def test_in_place(hip_backend, extents, axis):
    kind, dtype = "gated_blend", "f16"
    kept = extents[:axis] + extents[axis + 1:]
    g, x = stored(kind, 81, extents, dtype, gate=True), stored(kind, 82, extents, dtype)
    initial = normal(83, int(np.prod(kept))).astype(np.float32).reshape(kept)
    for over in ("x", "gate"):
        G, X, S = pair(hip_backend, g), pair(hip_backend, x), Tensor.from_numpy(hip_backend, initial)
        out = X[0] if over == "x" else G[0]
        Y, L = check_forward(hip_backend, kind, dtype, G, X, axis, initial=initial, out=out, last=S)
        assert Y is out and L is S
        # the state's own tensor is read and updated
        G, X, S = pair(hip_backend, g), pair(hip_backend, x), Tensor.from_numpy(hip_backend, initial)
        want, err = O.gated_scan(kind, columns(g, axis, False), columns(x, axis, False), initial.astype(np.float64).reshape(-1))
        F.gated_scan(G[0], X[0], axis, kind, initial=S, last=S)
        hip_backend.synchronize()
        assert O.close(S.numpy().reshape(-1), want[-1], err[-1], "f32")


@pytest.mark.parametrize("n", [15, 63, 64, 65, 257, 1023, 1025, 2049, 4097, 33001])
@pytest.mark.parametrize("start", [0, 1, 2, 3])
def test_rows_on_odd_elements(hip_backend, n, start):
    # two-byte rows along memory that start on any element, at even and odd pitches
    kind, dtype, m = "gated_blend", "f16", 5
    for pitch in (n + 3, n + 4):
        for reverse in (False, True):
            wide = [stored(kind, 400 + i, (m, pitch + start), dtype, gate=i == 0) for i in range(3)]
            T = [Tensor.from_numpy(hip_backend, w).slice([start], [start + n], [1]) for w in wide]
            v = [np.ascontiguousarray(w[:, start:start + n]) for w in wide]
            initial = normal(410, m).astype(np.float32)
            rest = Tensor.from_numpy(hip_backend, np.zeros((m, pitch + start), np.float16))
            out = rest.slice([start], [start + n], [1])
            Y, _ = check_forward(hip_backend, kind, dtype, (T[0], v[0]), (T[1], v[1]), 1, reverse, initial, out=out)
            got = rest.numpy()
            assert (got[:, :start] == 0).all() and (got[:, start + n:] == 0).all()          # nothing beside the rows
            check_grad(hip_backend, kind, dtype, (T[0], v[0]), (T[1], v[1]), (Y, Y.numpy()), (T[2], v[2]), 1, reverse, initial)


def test_decoding_equals_the_long_call(hip_backend):
    kind, dtype, shape = "gated_sigmoid", "f32", (5, 12, 33)
    G, X = pair(hip_backend, stored(kind, 91, shape, dtype, gate=True)), pair(hip_backend, stored(kind, 92, shape, dtype))
    whole, last = F.gated_scan(G[0], X[0], 1, kind)
    S = Tensor.from_numpy(hip_backend, np.zeros((5, 33), np.float32))
    for t in range(12):
        y, _ = F.gated_scan(G[0].slice([t], [t + 1], [1]), X[0].slice([t], [t + 1], [1]), 1, kind, initial=S, last=S)
        hip_backend.synchronize()
        # both round the same steps in the same order: equal bit for bit
        assert np.array_equal(y.numpy()[:, 0], whole.numpy()[:, t])
    assert np.array_equal(S.numpy(), last.numpy())


def test_growing_states_stay_finite(hip_backend):
    # factors of 2 from a state of 1e-30: after 200 steps 1.6e30, although the product of the gates
    # alone passes the largest fp32 number; zeros under any growth stay zeros
    n, m = 1500, 3
    g = np.full((n, m), 1.0, np.float32)
    g[300:500] = 2.0
    g[900:, 1] = 3.0
    x = np.zeros((n, m), np.float32)
    x[10, 0] = 1e-30
    for arrays, axis in (((g, x), 0), ((g.T.copy(), x.T.copy()), 1)):
        Y, _ = F.gated_scan(Tensor.from_numpy(hip_backend, arrays[0]), Tensor.from_numpy(hip_backend, arrays[1]), axis, "gated")
        hip_backend.synchronize()
        y = np.moveaxis(Y.numpy(), axis, 0)
        assert np.isfinite(y).all() and (y[:, 1:] == 0).all()
        want = np.float64(np.float32(1e-30)) * 2.0 ** 200
        assert abs(y[-1, 0] - want) <= 1600 * 2 * O.U * want          # a rounding a step at most


@pytest.mark.parametrize("kind", KINDS)
def test_gradient_against_differences(hip_backend, kind):
    # derivative of sum(wy y) + sum(wl last) along a random direction, from the 64-bit recurrence by
    # central differences: a step of 1e-5 leaves 1e-10 of truncation and 1e-11 of cancellation
    n, m = 37, 6
    g0, x0 = gate_values(kind, 301, n * m).reshape(n, m), normal(302, n * m).reshape(n, m)
    g0 = np.where(np.isfinite(g0), g0, 1.0)
    g, x = (O.load(O.store(v, "f32")) for v in (g0, x0))
    h0, wl = normal(303, m).astype(np.float32), normal(304, m).astype(np.float32)
    wy = normal(305, n * m).astype(np.float32).reshape(n, m)
    y = O.gated_scan(kind, g, x, h0.astype(np.float64))[0]
    T = lambda a: Tensor.from_numpy(hip_backend, np.asarray(a, np.float32))       # noqa: E731
    dg, dx, dh = (v.numpy().astype(np.float64) for v in
                  F.gated_scan_grad(T(g), T(x), T(y), T(wy), 0, kind, initial=T(h0), dlast=T(wl)))

    def loss(e, a, b, c):
        h = O.gated_scan(kind, g + e * a, x + e * b, h0 + e * c)[0]
        return (h * wy).sum() + (h[-1] * wl).sum()
    for seed in range(4):
        a, b, c = (normal(310 + 3 * seed + i, s).reshape(-1, m) for i, s in enumerate((n * m, n * m, m)))
        c = c[0]
        want = (loss(1e-5, a, b, c) - loss(-1e-5, a, b, c)) / 2e-5
        got = (dg * a).sum() + (dx * b).sum() + (dh * c).sum()
        scale = np.abs(dg * a).sum() + np.abs(dx * b).sum() + np.abs(dh * c).sum()
        # fp32 gradients: under 40 steps with under 16 u each
        assert abs(got - want) <= (40 * 16 * O.U + 1e-8) * scale


def test_refusals(hip_backend):
    T = lambda *e, t=np.float32: Tensor.empty(hip_backend, e, t)                  # noqa: E731
    with pytest.raises(ValueError, match="kind"):
        F.gated_scan(T(2, 3), T(2, 3), 1, "gru")
    with pytest.raises(TypeError):
        F.gated_scan(T(2, 3, t=np.float64), T(2, 3, t=np.float64), 1)
    with pytest.raises(TypeError):
        F.gated_scan(T(2, 3, t=np.float16), T(2, 3), 1)
    with pytest.raises(ValueError, match="gate"):
        F.gated_scan(T(2, 4), T(2, 3), 1)
    with pytest.raises(ValueError, match="initial"):
        F.gated_scan(T(2, 3), T(2, 3), 1, initial=T(3))
    with pytest.raises(TypeError, match="last"):
        F.gated_scan(T(2, 3), T(2, 3), 1, last=T(2, t=np.float16))
    with pytest.raises(ValueError):
        F.gated_scan(T(2, 3), T(2, 3), 2)
    with pytest.raises(ValueError, match="X is needed"):
        F.gated_scan_grad(T(2, 3), None, T(2, 3), T(2, 3), 1, "gated_blend")
    with pytest.raises(RuntimeError, match="invalid argument"):
        F.gated_scan(T(2, 3), T(2, 3), 1, out=T(1, 3).view(Shape((2, 3), (0, 1))))
