"""cross_entropy, whole and in pieces, and its gradient against 64 bits (sequence_oracle.py).

Bounds: with d = max - x the fp32 exponential of a term is off by (d + 4) u of itself (the
difference's rounding, the function, and for two-byte elements the hardware's 2^x of a rounded
product: another d u); a sum of n <= 2^18 terms, joined in trees of lanes and wavefronts over runs
of at most n / 256 terms added one by one in 8 strands, is off by (n / 2048 + 40) u.  The loss adds
roundings at the size of its two terms and of z lse^2."""
import numpy as np
import pytest

import sequence_oracle as O
from dlf_amd import frontend as F
from dlf_amd.frontend import Tensor
from dlf_amd.shape import Shape
from helpers import normal, randint, uniform01

pytestmark = pytest.mark.gpu


def logits(seed, m, n, dtype, std=2.0, masked=0.0):
    x = std * normal(seed, m * n).reshape(m, n)
    return O.store(np.where(uniform01(seed + 1, m * n).reshape(m, n) < masked, -np.inf, x), dtype)


def targets_of(seed, m, n, ignored=0.1):
    t = randint(seed, m, 0, n)
    return np.where(uniform01(seed + 2, m) < ignored, -100, t)


def sum_error(n):
    return (n / 2048 + 48) * O.U


def loss_bound(x, want, z):
    mx = np.where(np.isfinite(x).any(1), x.max(1, initial=-np.inf), 0.0)
    lse = np.abs(mx) + np.log(x.shape[1])
    # terms far below the maximum add nothing that their own error could show: d exp(-d) <= 1 / e on
    # average, so the sum's relative error is within the bound for d = 8
    e = sum_error(x.shape[1]) + 24 * O.U
    return e * (1 + 2 * z * lse) + 8 * O.U * (np.abs(want) + 2 * lse + z * lse ** 2)


def grad_bound(x, want, targets, w, z):
    with np.errstate(invalid="ignore"):
        mx = x.max(1, keepdims=True)
        d = np.where(np.isfinite(x), mx - x, 0.0)
    lse = np.abs(np.where(np.isfinite(mx), mx, 0.0)) + np.log(x.shape[1])
    factor = 1 + 2 * z * lse
    p = np.where(np.isfinite(x), np.exp(-d), 0.0)
    p = p / np.maximum(p.sum(1, keepdims=True), 1e-300) * factor
    one = np.zeros_like(x)
    ok = (targets >= 0) & (targets < x.shape[1])
    one[np.nonzero(ok)[0], targets[ok]] = 1.0
    return np.abs(w)[:, None] * (p * (2 * d * O.U + sum_error(x.shape[1]) + 40 * O.U) + 4 * O.U * one)


def check(hip, dtype, x, t, z=0.0, w=None, X=None, index=np.int64):
    """The loss alone, loss and gradient in one call, and the same in pieces, all against the oracle."""
    m, n = x.shape
    values = O.load(x)
    want, grad = O.cross_entropy(values, t, float(np.float32(z)), None if w is None else w.astype(np.float64))
    weights = np.ones(m) if w is None else w.astype(np.float64)
    lb, gb = loss_bound(values, np.where(np.isfinite(want), want, 0), z), grad_bound(values, grad, t, weights, z)
    X = X or Tensor.from_numpy(hip, x)
    T = Tensor.from_numpy(hip, t.astype(index))
    W = None if w is None else Tensor.from_numpy(hip, w)
    loss = F.cross_entropy(X, T, z)
    both = F.cross_entropy_grad(X, T, W, z)
    hip.synchronize()
    assert O.close(loss.numpy(), want, lb, "f32"), "loss"
    assert O.close(both[0].numpy(), want, lb, "f32"), "loss beside the gradient"
    assert O.close(both[1].numpy(), grad, gb, dtype), "gradient"
    return T, W, want, grad, lb, gb


def check_pieces(hip, dtype, x, t, cuts, z=0.0, w=None, order=None, in_place=False):
    m, n = x.shape
    T, W, want, grad, lb, gb = check(hip, dtype, x, t, z, w)
    spans = list(zip([0] + cuts, cuts + [n]))
    pieces = [(a, Tensor.from_numpy(hip, np.ascontiguousarray(x[:, a:b]))) for a, b in spans]
    state = None
    for i in order or range(len(pieces)):
        state = F.cross_entropy_piece(pieces[i][1], T, pieces[i][0], state)
    loss = F.cross_entropy_join(state, T, z)
    # every piece joins two sums: another two roundings of the sum
    more = 2 * len(pieces) * O.U
    for (a, b), (first, P) in zip(spans, pieces):
        g = F.cross_entropy_piece_grad(P, T, first, state, W, z, out=P if in_place else None)
        hip.synchronize()
        assert O.close(g.numpy(), grad[:, a:b], gb[:, a:b] * (1 + 1e-6) + more * np.abs(grad[:, a:b]) + more * O.U, dtype), (a, b)
    assert O.close(loss.numpy(), want, lb + more, "f32")
    # the state: maxima are exact, so are the targets' logits
    s = state.numpy()
    live = t >= 0
    values = O.load(x)
    assert np.array_equal(s[0][live], values[live].max(1).astype(np.float32))
    inside = live & (t < n)
    assert np.array_equal(s[2][inside], values[np.nonzero(inside)[0], t[inside]].astype(np.float32))


SIZES = [(1, 1), (3, 2), (5, 7), (1, 8), (64, 33), (130, 64), (17, 255), (9, 256), (33, 1000), (6, 2049), (12, 4099), (300, 5000), (5, 8192), (3, 8193),
         (7, 16385), (4, 32000), (2, 32771), (260, 33000), (3, 50257), (2, 65537), (1, 131072), (2, 200003)]


@pytest.mark.parametrize("m,n", SIZES)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_loss_and_gradient(hip_backend, m, n, dtype):
    x = logits(m + n, m, n, dtype)
    t = targets_of(m + 3, m, n)
    check(hip_backend, dtype, x, t, 1e-4, (normal(m, m) / m).astype(np.float32))
    check(hip_backend, dtype, x, t.astype(np.int32), index=np.int32)


@pytest.mark.parametrize("m,n,cuts", [(5, 100, [1, 40]), (33, 3000, [1024, 2048]), (6, 20011, [8191, 8192, 17000]), (2, 150000, [70001]), (300, 9001, [4500]),
                                      (1, 1, []), (4, 60, [59])])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_pieces(hip_backend, m, n, cuts, dtype):
    x = logits(m + n, m, n, dtype)
    t = targets_of(m + 4, m, n)
    w = (normal(m + 9, m) * 4).astype(np.float32)
    check_pieces(hip_backend, dtype, x, t, cuts, 1e-4, w)
    check_pieces(hip_backend, dtype, x, t, cuts, order=list(range(len(cuts), -1, -1)), in_place=True)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,n", [(40, 50), (12, 3001), (4, 40000), (2, 140001)])
def test_masks_empty_rows_and_targets(hip_backend, m, n, dtype):
    m = max(m, 8)
    x = logits(m, m, n, dtype, masked=0.7)
    t = targets_of(5, m, n, 0.0)
    x[0] = O.store(np.full(n, -np.inf), dtype)                   # nothing left: loss inf, gradient 0
    t[1] = -1                                                    # taken out, whatever the row holds
    x[1, ::3] = O.store(np.full(len(x[1, ::3]), np.nan), dtype)
    x[2, 1:] = O.store(np.full(n - 1, -np.inf), dtype)           # one left
    t[2] = 0
    x[3] = O.store(np.full(n, -np.inf), dtype)
    x[3, n - 1] = O.store(np.float32(3.0), dtype)
    t[3] = 0                                                     # a masked target: loss inf, gradient finite
    t[4] = n                                                     # beyond the vocabulary: loss NaN
    x[5] = O.store(np.full(n, O.LOWEST[dtype]), dtype)           # the lowest value everywhere: uniform
    x[6, : n // 2] = O.store(np.full(n // 2, O.LOWEST[dtype]), dtype)
    x[6, n // 2] = O.store(np.float32(1.0), dtype)
    t[6] = n // 2
    values = O.load(x)
    y = values.copy()
    y[1] = 0.0
    want, grad = O.cross_entropy(y, t)
    # rows at the lowest value: the difference is exact, the bound that of a row of zeros
    flat = np.where(np.abs(y) > 1e4, np.where(np.isfinite(y), 0.0, y), y)
    lb, gb = loss_bound(flat, np.where(np.isfinite(want), want, 0), 0.0), grad_bound(flat, grad, t, np.ones(m), 0.0)
    X, T = Tensor.from_numpy(hip_backend, x), Tensor.from_numpy(hip_backend, t)
    loss, g = F.cross_entropy_grad(X, T)
    alone = F.cross_entropy(X, T)
    half = n // 2
    parts = [(a, Tensor.from_numpy(hip_backend, np.ascontiguousarray(x[:, a:b]))) for a, b in ((0, half), (half, n))]
    state = None
    for first, P in parts:
        state = F.cross_entropy_piece(P, T, first, state)
    joined = F.cross_entropy_join(state, T)
    grads = [F.cross_entropy_piece_grad(P, T, first, state) for first, P in parts]
    hip_backend.synchronize()
    for got in (loss, alone, joined):
        assert O.close(got.numpy(), want, lb + 8 * O.U, "f32")
    assert np.isinf(loss.numpy()[0]) and loss.numpy()[1] == 0 and np.isinf(loss.numpy()[3]) and np.isnan(loss.numpy()[4])
    assert O.close(g.numpy(), grad, gb, dtype)
    assert O.close(np.concatenate([p.numpy() for p in grads], 1), grad, gb + 8 * O.U * np.abs(grad), dtype)
    assert (O.load(g.numpy())[:2] == 0).all()


def test_nan_and_infinite_logits_show(hip_backend):
    x = logits(8, 6, 700, "f32")
    x[1, 300], x[2, 5], x[3, 699] = np.nan, np.inf, np.inf
    t = np.array([1, 2, 3, 699, 5, -7])
    loss, g = F.cross_entropy_grad(Tensor.from_numpy(hip_backend, x), Tensor.from_numpy(hip_backend, t))
    hip_backend.synchronize()
    l = loss.numpy()
    assert np.isfinite(l[[0, 4, 5]]).all() and np.isnan(l[1]) and l[2] == np.inf and np.isnan(l[3])
    assert np.isnan(g.numpy()[1]).any() and np.isfinite(g.numpy()[[0, 4, 5]]).all()


@pytest.mark.parametrize("n", [61, 5001, 40001])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_views_ranks_and_in_place(hip_backend, n, dtype):
    m = 12
    wide = logits(n, m, n + 20, dtype)
    x = np.ascontiguousarray(wide[:, 7:7 + n])
    t = targets_of(3, m, n)
    want, grad = O.cross_entropy(O.load(x), t)
    gb = grad_bound(O.load(x), grad, t, np.ones(m), 0.0)
    B = Tensor.from_numpy(hip_backend, wide)
    X = B.slice([7], [7 + n], [1])                               # rows at a stride, off a vector's boundary
    check(hip_backend, dtype, x, t, X=X)
    T = Tensor.from_numpy(hip_backend, t)
    F.cross_entropy_grad(X, T, out=X)                            # in place; what lies beside the rows stays
    hip_backend.synchronize()
    after = B.numpy()
    assert O.close(after[:, 7:7 + n], grad, gb, dtype)
    assert np.array_equal(after[:, :7].tobytes(), wide[:, :7].tobytes()) and np.array_equal(after[:, 7 + n:].tobytes(), wide[:, 7 + n:].tobytes())
    cube = Tensor.from_numpy(hip_backend, x.reshape(3, 4, n))
    loss = F.cross_entropy(cube, Tensor.from_numpy(hip_backend, t.reshape(3, 4)))
    column = Tensor.from_numpy(hip_backend, np.ascontiguousarray(x.T)).transpose()
    loss2, g2 = F.cross_entropy_grad(column, T)
    hip_backend.synchronize()
    # the loss alone and the loss beside a gradient add up in different orders: each within the bound
    lb = loss_bound(O.load(x), want, 0.0)
    assert loss.numpy().shape == (3, 4) and O.close(loss.numpy().reshape(-1), want, lb, "f32") and O.close(loss2.numpy(), want, lb, "f32")
    assert O.close(g2.numpy(), grad, gb, dtype)
    one = F.cross_entropy(Tensor.from_numpy(hip_backend, x[0]), Tensor.from_numpy(hip_backend, t[:1]).view(Shape(())))
    hip_backend.synchronize()
    assert one.numpy().shape == ()


@pytest.mark.parametrize("z", [0.0, 1e-3])
def test_gradient_against_differences(hip_backend, z):
    m, n = 4, 30
    x = logits(61, m, n, "f32")
    t = np.array([3, 29, 0, 7])
    w = normal(62, m).astype(np.float32)
    _, g = F.cross_entropy_grad(Tensor.from_numpy(hip_backend, x), Tensor.from_numpy(hip_backend, t), Tensor.from_numpy(hip_backend, w), z)
    g = g.numpy().astype(np.float64)
    d = normal(63, m * n).reshape(m, n)
    z = float(np.float32(z))
    f = lambda e: (O.cross_entropy(O.load(x) + e * d, t, z)[0] * w).sum()        # noqa: E731
    want = (f(1e-5) - f(-1e-5)) / 2e-5
    assert abs((g * d).sum() - want) <= (100 * O.U + 1e-8) * (np.abs(w)[:, None] * np.abs(d)).sum()


def test_refusals(hip_backend):
    T = lambda *e, t=np.float32: Tensor.empty(hip_backend, e, t)                  # noqa: E731
    with pytest.raises(TypeError, match="targets"):
        F.cross_entropy(T(2, 8), T(2))
    with pytest.raises(ValueError, match="targets"):
        F.cross_entropy(T(2, 8), T(3, t=np.int32))
    with pytest.raises(TypeError):
        F.cross_entropy(T(2, 8, t=np.int32), T(2, t=np.int32))
    with pytest.raises(ValueError, match="weights"):
        F.cross_entropy_grad(T(2, 8), T(2, t=np.int32), T(8))
    with pytest.raises(TypeError, match="weights"):
        F.cross_entropy_grad(T(2, 8), T(2, t=np.int32), T(2, t=np.float64))
    with pytest.raises(ValueError, match="state"):
        F.cross_entropy_piece(T(2, 8), T(2, t=np.int32), 0, T(2, 3))
    with pytest.raises(RuntimeError, match="invalid argument"):
        F.cross_entropy_piece(T(2, 8), T(2, t=np.int32), -1)
    with pytest.raises(ValueError, match="out"):
        F.cross_entropy_grad(T(2, 8), T(2, t=np.int32), out=T(8, 2).transpose())
    with pytest.raises(ValueError, match="state"):
        F.cross_entropy_join(T(3, 3), T(2, t=np.int32))
