"""route and its gradient against a row-by-row 64-bit form (sequence_oracle.py).

Weights are fp32 results of scores in 64 bits or fp32: a softmax of up to 1024 terms sums with at
most 10 levels of roundings on top of sums of 16 in a lane, its exponentials carry |x - max| u from
the difference and 2 u from the function, the renormalisation sums k <= 64 scores and divides:
under 64 u with logits within +-12."""
import numpy as np
import pytest

import sequence_oracle as O
from dlf_amd import frontend as F
from dlf_amd.frontend import Tensor
from helpers import normal, uniform01

pytestmark = pytest.mark.gpu
BOUND = 64 * O.U


def logits(seed, m, n, dtype, std=1.5, masked=0.0, lowest=0.0):
    x = np.clip(std * normal(seed, m * n).reshape(m, n), -6, 6)
    x = np.where(uniform01(seed + 500, m * n).reshape(m, n) < masked, -np.inf, x)
    a = O.store(x, dtype)
    if lowest:
        low = O.store(np.full((m, n), O.LOWEST[dtype]), dtype)
        a = np.where(uniform01(seed + 501, m * n).reshape(m, n) < lowest, low, a)
    return a


def check(hip, dtype, x, k, score, X=None, bias=None, loads=False, grad=True, **how):
    m, n = x.shape
    named = dict(groups=how.get("groups", 1), kept=how.get("kept_groups"), best=how.get("group_best", 1), renormalise=how.get("renormalise", False),
                 scale=np.float64(np.float32(how.get("scale", 1.0))))
    values = O.load(x)
    W0, I0, _ = O.route(score, values, O.LOWEST[dtype], k, None if bias is None else bias.astype(np.float64), **named)
    X = X or Tensor.from_numpy(hip, x)
    L = Tensor.from_numpy(hip, np.full(n, 7, np.int32)) if loads else None
    W, I = F.route(X, k, score, bias=None if bias is None else Tensor.from_numpy(hip, bias), loads=L, **how)
    hip.synchronize()
    assert W.numpy().shape == (m, k) and W.dtype == np.float32 and I.dtype == np.int32
    assert np.array_equal(I.numpy(), I0)
    assert O.close(W.numpy(), W0, BOUND * np.abs(W0), "f32")
    if loads:
        assert np.array_equal(L.numpy(), 7 + np.bincount(I0.reshape(-1), minlength=n))
    if grad:
        dw = normal(m + n, m * k).astype(np.float32).reshape(m, k)
        check_grad(hip, dtype, X, values, I0, dw, score, named["renormalise"], how.get("scale", 1.0))
    return W, I


def check_grad(hip, dtype, X, values, indices, dw, score, renormalise, scale, out=None):
    want = O.route_grad(score, values, O.LOWEST[dtype], indices, dw.astype(np.float64), renormalise, np.float64(np.float32(scale)))
    got = F.route_grad(X, Tensor.from_numpy(hip, indices.astype(np.int32)), Tensor.from_numpy(hip, dw), score, renormalise=renormalise,
                       scale=scale, out=out)
    hip.synchronize()
    # every term of the gradient is a product of scores and of sums of scale dw s over the choices
    _, _, s = O.route(score, values, O.LOWEST[dtype], 1)
    m, n = values.shape
    size = np.zeros_like(s)
    for r in range(m):
        ok = (indices[r] >= 0) & (indices[r] < n)
        q, d = s[r, indices[r][ok]], np.abs(dw[r][ok].astype(np.float64) * scale)
        d, mean = (d / q.sum(), (d * q).sum() / q.sum() ** 2) if renormalise and q.sum() else (d, 0.0 if renormalise else (d * q).sum())
        if renormalise and not q.sum():
            continue
        size[r] = s[r] * mean * (1.0 if score == "softmax" or renormalise else 0.0)
        if renormalise:
            # without a choice the exact value is 0 for the logistic score; the softmax one cancels to 0 as well
            chosen = np.zeros(n, bool)
            chosen[indices[r][ok]] = True
            size[r] *= chosen
        np.add.at(size[r], indices[r][ok], s[r, indices[r][ok]] * d)
    # renormalised softmax: an expert that was not chosen has no gradient; 64 bits leave their own rounding
    assert O.close(got.numpy(), want, 2 * BOUND * size + 2.0 ** -48, dtype)


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 8, 2), (3, 5, 5), (17, 16, 4), (64, 60, 4), (257, 64, 6), (1000, 128, 8), (33, 129, 3), (65, 256, 8),
                                   (9, 257, 16), (5, 512, 64), (4, 1000, 10), (3, 1024, 64), (40, 33, 1)])
@pytest.mark.parametrize("score,dtype", [("softmax", "f32"), ("softmax", "bf16"), ("sigmoid", "f32"), ("sigmoid", "f16")])
def test_choices_and_weights(hip_backend, m, n, k, score, dtype):
    x = logits(m + n + k, m, n, dtype)
    check(hip_backend, dtype, x, k, score, loads=True)
    check(hip_backend, dtype, x, k, score, renormalise=True, scale=2.5)
    bias = (0.05 * normal(m + 7, n)).astype(np.float32)
    check(hip_backend, dtype, x, k, score, bias=bias, renormalise=True, grad=False)


@pytest.mark.parametrize("n,groups,kept,best,k", [(8, 2, 1, 1, 3), (64, 8, 3, 2, 6), (256, 8, 4, 2, 8), (160, 8, 3, 1, 6), (60, 4, 2, 2, 4), (35, 5, 2, 2, 14),
                                                  (512, 16, 2, 2, 8), (1024, 32, 4, 2, 8), (12, 12, 5, 2, 5), (256, 256, 9, 1, 9), (96, 3, 2, 2, 64),
                                                  (64, 64, 64, 2, 8), (128, 4, 4, 2, 8)])
@pytest.mark.parametrize("score", F.SCORE_KINDS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_groups(hip_backend, n, groups, kept, best, k, score, dtype):
    m = 67
    x = logits(n + groups, m, n, dtype)
    bias = (0.1 * normal(n + 3, n)).astype(np.float32)
    check(hip_backend, dtype, x, k, score, bias=bias, groups=groups, kept_groups=kept, group_best=best, renormalise=True, scale=2.5, loads=True)
    check(hip_backend, dtype, x, k, score, groups=groups, kept_groups=kept, group_best=best, grad=False)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("score", F.SCORE_KINDS)
@pytest.mark.parametrize("groups,kept,best", [(1, 1, 1), (4, 2, 2), (8, 3, 1)])
def test_masked_experts(hip_backend, dtype, score, groups, kept, best):
    m, n, k = 120, 32, 7
    for masked, lowest in ((0.5, 0.0), (0.0, 0.6), (0.5, 0.45)):
        x = logits(5, m, n, dtype, masked=masked, lowest=lowest)
        x[3] = O.store(np.full(n, -np.inf), dtype)                       # nothing left
        x[4] = O.store(np.full(n, O.LOWEST[dtype]), dtype)
        x[5, 1:] = O.store(np.full(n - 1, -np.inf), dtype)               # one left
        x[6, :n // groups] = O.store(np.full(n // groups, -np.inf), dtype)   # a whole group gone
        bias = (0.3 * normal(6, n)).astype(np.float32)
        bias[2] = 5.0                                                    # a bias never brings a masked expert in
        for b in (None, bias):
            for renormalise in (False, True):
                W, I = check(hip_backend, dtype, x, k, score, bias=b, groups=groups, kept_groups=kept, group_best=best, renormalise=renormalise,
                             loads=True)
                w = W.numpy()
                assert (w[3] == 0).all() and (w[4] == 0).all() and np.isfinite(w).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_equal_values_take_the_lower_index(hip_backend, dtype):
    m, n, k = 300, 96, 9
    x = O.store(np.round(normal(11, m * n).reshape(m, n) * 2) / 2, dtype)      # few different values
    x[0] = O.store(np.zeros(n), dtype)
    x[1] = O.store(np.where(np.arange(n) % 2, 0.0, -0.0), dtype)               # one value of two signs
    for score in F.SCORE_KINDS:
        check(hip_backend, dtype, x, k, score)
        check(hip_backend, dtype, x, k, score, groups=6, kept_groups=3, group_best=2)
        check(hip_backend, dtype, x, k, score, bias=np.zeros(n, np.float32), groups=6, kept_groups=2)
        check(hip_backend, dtype, x, k, score, bias=np.repeat(np.float32([0.5, 0.25, 0.5]), n // 3), renormalise=True)


def test_choices_closer_than_fp32_tells(hip_backend):
    # scores + bias that differ by less than an fp32 rounding are still told apart, in either order
    m, n, k = 64, 16, 8
    x = np.zeros((m, n), np.float32)
    x += (np.arange(n) * 3e-8)[None, :].astype(np.float32)
    x = np.where(np.arange(m)[:, None] % 2, x, x[:, ::-1])
    bias = np.full(n, 1.0, np.float32)
    for score in F.SCORE_KINDS:
        W, I = check(hip_backend, "f32", np.ascontiguousarray(x), k, score, bias=bias, grad=False)
        assert I.numpy()[1, 0] == n - 1 and I.numpy()[0, 0] == 0


def test_nan_rows_have_valid_different_choices(hip_backend):
    m, n, k = 50, 40, 12
    x = logits(21, m, n, "f32")
    x[::2, 5] = np.nan
    x[4] = np.nan
    x[6, 3] = np.inf
    for score in F.SCORE_KINDS:
        for how in (dict(), dict(groups=4, kept_groups=2, group_best=2), dict(bias=True)):
            if how.pop("bias", False):
                how["bias"] = Tensor.from_numpy(hip_backend, np.zeros(n, np.float32))
            W, I = F.route(Tensor.from_numpy(hip_backend, x), k, score, **how)
            hip_backend.synchronize()
            i = I.numpy()
            assert ((i >= 0) & (i < n)).all() and all(len(set(r)) == k for r in i.tolist())
            clean = [r for r in range(1, m, 2)]
            assert np.isfinite(W.numpy()[clean]).all()


def test_views_and_ranks(hip_backend):
    dtype = "f16"
    wide = logits(31, 30, 100, dtype)
    X = Tensor.from_numpy(hip_backend, wide).slice([3], [64], [1])                 # rows at a stride, odd start
    check(hip_backend, dtype, np.ascontiguousarray(wide[:, 3:64]), 5, "softmax", X=X, renormalise=True)
    T = Tensor.from_numpy(hip_backend, np.ascontiguousarray(wide.T)).transpose()    # not contiguous along the experts
    check(hip_backend, dtype, wide, 5, "sigmoid", X=T)
    cube = wide.reshape(5, 6, 100)
    W, I = F.route(Tensor.from_numpy(hip_backend, cube), 4)
    W2, I2 = F.route(Tensor.from_numpy(hip_backend, wide), 4)
    hip_backend.synchronize()
    assert W.numpy().shape == (5, 6, 4) and np.array_equal(I.numpy().reshape(30, 4), I2.numpy()) and np.array_equal(W.numpy().reshape(30, 4), W2.numpy())
    one, at = F.route(Tensor.from_numpy(hip_backend, wide[0]), 4)
    hip_backend.synchronize()
    assert one.numpy().shape == (4,) and np.array_equal(at.numpy(), I2.numpy()[0])


@pytest.mark.parametrize("score", F.SCORE_KINDS)
@pytest.mark.parametrize("renormalise", [False, True])
def test_gradient_of_repeated_and_foreign_indices_in_place(hip_backend, score, renormalise):
    m, n, k = 41, 70, 6
    x = logits(41, m, n, "f32")
    idx = (uniform01(42, m * k) * n).astype(np.int64).reshape(m, k)
    idx[:, 1] = idx[:, 0]                                     # the same expert twice
    idx[::3, 2] = -1
    idx[1::3, 2] = n
    idx[2::3, 2] = 2 ** 31 - 1
    idx[7] = -5                                               # no choice at all
    dw = normal(43, m * k).astype(np.float32).reshape(m, k)
    X = Tensor.from_numpy(hip_backend, x)
    check_grad(hip_backend, "f32", X, O.load(x), idx, dw, score, renormalise, 1.5)
    check_grad(hip_backend, "f32", X, O.load(x), idx, dw, score, renormalise, 1.5, out=X)


@pytest.mark.parametrize("score", F.SCORE_KINDS)
@pytest.mark.parametrize("renormalise", [False, True])
def test_gradient_against_differences(hip_backend, score, renormalise):
    m, n, k = 6, 24, 4
    x = logits(51, m, n, "f32")
    dw = normal(52, m * k).astype(np.float32).reshape(m, k)
    values = O.load(x)
    _, I0, _ = O.route(score, values, O.LOWEST["f32"], k)
    got = F.route_grad(Tensor.from_numpy(hip_backend, x), Tensor.from_numpy(hip_backend, I0.astype(np.int32)), Tensor.from_numpy(hip_backend, dw),
                       score, renormalise=renormalise, scale=2.0).numpy().astype(np.float64)

    def loss(v):
        s = O.scores(score, v, np.ones_like(v, bool))
        w = np.take_along_axis(s, I0, 1)
        return (2.0 * w / (w.sum(1, keepdims=True) if renormalise else 1.0) * dw).sum()
    d = normal(53, m * n).reshape(m, n)
    want = (loss(values + 1e-5 * d) - loss(values - 1e-5 * d)) / 2e-5
    assert abs((got * d).sum() - want) <= (BOUND + 1e-8) * 4 * (np.abs(dw).sum() + np.abs(got * d).sum())


def test_refusals(hip_backend):
    T = lambda *e, t=np.float32: Tensor.empty(hip_backend, e, t)                  # noqa: E731
    with pytest.raises(ValueError, match="score"):
        F.route(T(2, 8), 2, "tanh")
    with pytest.raises(TypeError):
        F.route(T(2, 8, t=np.float64), 2)
    with pytest.raises(RuntimeError, match="invalid argument"):
        F.route(T(2, 8), 9)
    with pytest.raises(RuntimeError, match="invalid argument"):
        F.route(T(2, 8), 3, groups=4, kept_groups=1)
    with pytest.raises(RuntimeError, match="too large"):
        F.route(T(2, 2000), 3)
    with pytest.raises(ValueError, match="bias"):
        F.route(T(2, 8), 3, bias=T(7))
    with pytest.raises(TypeError, match="loads"):
        F.route(T(2, 8), 3, loads=T(8))
    with pytest.raises(ValueError, match="indices"):
        F.route_grad(T(2, 8), T(3, 2, t=np.int32), T(2, 2))
    with pytest.raises(TypeError, match="dweights"):
        F.route_grad(T(2, 8), T(2, 2, t=np.int32), T(2, 2, t=np.float16))
