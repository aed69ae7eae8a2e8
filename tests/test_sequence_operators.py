"""Refusals of the sequence-model operators' C entry points: host arithmetic, no GPU."""
import ctypes

import numpy as np
import pytest

from dlf_amd import frontend as F
from dlf_amd import hip_backend

FAKE = ctypes.c_void_p(0x1000)
INVALID, DTYPE, UNKNOWN, SCRATCH, RANK, LARGE = -1, -2, -3, -4, -5, -7


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def scan(lib, name=b"gated", dtype=0, m=4, n=8, rank=2, dims=(4, 8), g=FAKE, x=FAKE, y=FAKE, st=(8, 1), ys=(8, 1), initial=None, ist=None,
         last=None, lst=None):
    return lib.dlfx_gated_scan(None, name, dtype, m, n, rank, i64(*dims), g, 0, i64(*st), x, 0, i64(*st), initial, 0, ist, y, 0, i64(*ys),
                               last, 0, lst, None, 0)


def scan_grad(lib, name=b"gated", dtype=0, m=4, n=8, x=None, xs=None, g=FAKE, y=FAKE, dy=FAKE, dg=FAKE, dx=FAKE, ds=(8, 1), dinitial=None, dist=None):
    st = i64(8, 1)
    return lib.dlfx_gated_scan_grad(None, name, dtype, m, n, 2, i64(4, 8), g, 0, st, x, 0, xs, None, 0, None, y, 0, st, dy, 0, st, None, 0, None,
                                    dg, 0, st, dx, 0, i64(*ds), dinitial, 0, dist, None, 0)


def test_gated_scan_refusals():
    lib = hip_backend.load_library()
    assert scan(lib, name=b"gru") == UNKNOWN
    assert scan(lib, name=None) == INVALID
    for dtype in (1, 2, 3, 5, 6, 7, 8, 10):
        assert scan(lib, dtype=dtype) == DTYPE
    for missing in ("g", "x", "y"):
        assert scan(lib, **{missing: None}) == INVALID
    assert scan(lib, n=7) == INVALID and scan(lib, m=5) == INVALID and scan(lib, m=0) == INVALID and scan(lib, n=0, dims=(4, 0)) == INVALID
    assert scan(lib, rank=0) == INVALID
    assert scan(lib, ys=(0, 1)) == INVALID and scan(lib, ys=(8, 0)) == INVALID
    assert scan(lib, initial=FAKE) == INVALID and scan(lib, last=FAKE) == INVALID           # without strides
    assert scan(lib, last=FAKE, lst=i64(0)) == INVALID
    nine = (2,) * 9 + (3,)
    far = tuple(1000 ** 0 * 7 * (11 ** i) for i in range(10))
    assert scan(lib, m=512, n=3, rank=10, dims=nine, st=far, ys=far) == RANK
    assert scan_grad(lib, name=b"gated_blend") == INVALID                                    # x is needed
    assert scan_grad(lib, name=b"none") == UNKNOWN
    assert scan_grad(lib, dtype=1) == DTYPE
    for missing in ("g", "y", "dy", "dg", "dx"):
        assert scan_grad(lib, **{missing: None}) == INVALID
    assert scan_grad(lib, ds=(0, 1)) == INVALID and scan_grad(lib, n=9) == INVALID
    assert scan_grad(lib, dinitial=FAKE) == INVALID and scan_grad(lib, dinitial=FAKE, dist=i64(0)) == INVALID


def route(lib, name=b"softmax", dtype=0, m=4, n=64, x=FAKE, stride=64, groups=1, kept=1, best=1, k=8, w=FAKE, i=FAKE):
    return lib.dlfx_route(None, name, dtype, m, n, x, 0, stride, None, groups, kept, best, k, 0, 1.0, w, i, None)


def test_route_refusals():
    lib = hip_backend.load_library()
    assert route(lib, name=b"tanh") == UNKNOWN and route(lib, name=None) == INVALID
    for dtype in (1, 2, 3, 5, 8, 10):
        assert route(lib, dtype=dtype) == DTYPE
    for bad in (dict(m=0), dict(n=0), dict(k=0), dict(k=65), dict(stride=63), dict(x=None), dict(w=None), dict(i=None), dict(groups=0),
                dict(groups=3), dict(groups=4, kept=5), dict(groups=4, kept=0), dict(best=0), dict(best=3), dict(groups=16, kept=1, k=5)):
        assert route(lib, **bad) == INVALID, bad
    assert route(lib, n=1025, stride=1025) == LARGE and route(lib, n=512, stride=512, k=65) == LARGE
    grad = lambda **a: lib.dlfx_route_grad(None, a.get("name", b"softmax"), a.get("dtype", 0), 4, 64, a.get("x", FAKE), 0, a.get("stride", 64),   # noqa: E731
                                           a.get("k", 8), a.get("i", FAKE), a.get("dw", FAKE), 0, 1.0, a.get("dx", FAKE), 0, a.get("ds", 64))
    assert grad(name=b"x") == UNKNOWN and grad(dtype=2) == DTYPE
    for bad in (dict(x=None), dict(i=None), dict(dw=None), dict(dx=None), dict(ds=63), dict(stride=1), dict(k=0), dict(k=65)):
        assert grad(**bad) == INVALID, bad


def test_cross_entropy_refusals():
    lib = hip_backend.load_library()

    def whole(dtype=0, index=2, m=4, n=100, x=FAKE, stride=100, t=FAKE, loss=FAKE):
        return lib.dlfx_cross_entropy(None, dtype, index, m, n, x, 0, stride, t, 0.0, loss, None, 0)

    def grad(dtype=0, index=2, m=4, n=100, x=FAKE, stride=100, t=FAKE, dx=FAKE, ds=100):
        return lib.dlfx_cross_entropy_grad(None, dtype, index, m, n, x, 0, stride, t, None, 0.0, None, dx, 0, ds, None, 0)

    def piece(dtype=0, index=2, m=4, n=100, x=FAKE, stride=100, t=FAKE, first=0, state=FAKE):
        return lib.dlfx_cross_entropy_piece(None, dtype, index, m, n, x, 0, stride, t, first, 0, state, None, 0)

    def piece_grad(dtype=0, index=2, m=4, n=100, x=FAKE, stride=100, t=FAKE, first=0, state=FAKE, dx=FAKE, ds=100):
        return lib.dlfx_cross_entropy_piece_grad(None, dtype, index, m, n, x, 0, stride, t, first, state, None, 0.0, dx, 0, ds)

    for call in (whole, grad, piece, piece_grad):
        assert call(dtype=1) == DTYPE and call(dtype=10) == DTYPE and call(index=0) == DTYPE and call(index=5) == DTYPE
        for bad in (dict(m=0), dict(n=0), dict(x=None), dict(t=None), dict(stride=99)):
            assert call(**bad) == INVALID, (call, bad)
        assert call(m=1 << 31) == LARGE and call(n=1 << 31, stride=1 << 31, **({"ds": 1 << 31} if call in (grad, piece_grad) else {})) == LARGE
    assert whole(loss=None) == INVALID and piece(state=None) == INVALID and piece(first=-1) == INVALID
    assert grad(dx=None) == INVALID and grad(ds=99) == INVALID
    assert piece_grad(state=None) == INVALID and piece_grad(first=-1) == INVALID and piece_grad(dx=None) == INVALID and piece_grad(ds=99) == INVALID
    join = lib.dlfx_cross_entropy_join
    assert join(None, 2, 0, FAKE, FAKE, 0.0, FAKE) == INVALID and join(None, 2, 4, None, FAKE, 0.0, FAKE) == INVALID
    assert join(None, 2, 4, FAKE, None, 0.0, FAKE) == INVALID and join(None, 2, 4, FAKE, FAKE, 0.0, None) == INVALID
    assert join(None, 0, 4, FAKE, FAKE, 0.0, FAKE) == DTYPE and join(None, 2, 1 << 31, FAKE, FAKE, 0.0, FAKE) == LARGE


def test_other_operators_refuse_bfloat16():
    lib = hip_backend.load_library()
    dims, st, one, s1 = i64(4, 8), i64(8, 1), i64(4), i64(1)
    assert lib.dlfx_scan(None, b"cumsum", 9, 4, 8, 0, 2, dims, FAKE, 0, st, FAKE, 0, st, None, 0) == DTYPE
    assert lib.dlfx_sort(None, 0, 9, 2, dims, FAKE, 0, st, FAKE, 0, st, None, 0) == DTYPE
    assert lib.dlfx_softmax(None, b"softmax", 9, 4, 8, FAKE, 0, FAKE, 0, None, 0) == DTYPE
    assert lib.dlfx_reduce(None, b"reduce_sum", 9, 4, 8, 2, dims, st, FAKE, 0, 1, one, s1, FAKE, 0, None, 0) == DTYPE


def test_bfloat16_arrays():
    v = np.array([1.0, -2.5, 0.0, -0.0, np.inf, -np.inf, 3.0e38, 3.3961775e38, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, 1e-40, np.nan], np.float32)
    b = F.to_bfloat16(v)
    assert b.dtype == F.BFLOAT16 and b.shape == v.shape
    back = F.from_bfloat16(b)
    assert np.isnan(back[-1])
    # ties to even: 1 + 2^-8 lies between 1 and 1 + 2^-7, 1 + 3 2^-8 between 1 + 2^-7 and 1 + 2^-6
    assert back[8] == 1.0 and back[9] == 1 + 2.0 ** -6
    fin = np.where(np.isfinite(v[:7]), v[:7], 0)
    assert (np.abs(np.where(np.isfinite(back[:7]), back[:7], 0) - fin) <= 2.0 ** -8 * np.abs(fin)).all() and back[4] == np.inf and back[5] == -np.inf
    assert back[7] == np.inf                              # halfway past the largest finite value
    assert np.array_equal(F.to_bfloat16(back[:-1]), b[:-1])


@pytest.mark.parametrize("kind", F.GATE_KINDS)
def test_oracle_gradient_of_the_recurrence(kind):
    # the oracle's own backward recurrence against central differences of its forward one
    import sequence_oracle as O
    from helpers import normal
    n, m = 23, 4
    g, x, wy = (normal(s, n * m).reshape(n, m) * 0.7 for s in (1, 2, 3))
    h0, wl = normal(4, m), normal(5, m)
    y = O.gated_scan(kind, g, x, h0)[0]
    (dg, dx, dh), _ = O.gated_scan_grad(kind, g, x, y, wy, h0, wl)

    def loss(e, a, b, c):
        h = O.gated_scan(kind, g + e * a, x + e * b, h0 + e * c)[0]
        return (h * wy).sum() + (h[-1] * wl).sum()
    a, b, c = normal(6, n * m).reshape(n, m), normal(7, n * m).reshape(n, m), normal(8, m)
    want = (loss(1e-5, a, b, c) - loss(-1e-5, a, b, c)) / 2e-5
    got = (dg * a).sum() + (dx * b).sum() + (dh * c).sum()
    assert abs(got - want) <= 1e-7 * (np.abs(dg * a).sum() + np.abs(dx * b).sum() + np.abs(dh * c).sum())
