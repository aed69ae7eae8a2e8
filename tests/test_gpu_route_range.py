"""route at the ends of its range: sums of choices that cancel, chosen scores near and below 2^-126."""
import numpy as np
import pytest

import sequence_oracle as O
import test_gpu_route as T
from dlf_amd import frontend as F
from dlf_amd.frontend import Tensor
from helpers import normal, uniform01

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,spread,score", [(1024, 0.25, "softmax"), (512, 0.5, "softmax"), (256, 1.0, "softmax"), (64, 4.0, "softmax"),
                                            (512, 4.0, "sigmoid"), (32, 64.0, "sigmoid")])
def test_groups_whose_biases_cancel(hip_backend, n, spread, score):
    # pairs of biases t and -t far above the scores: a group's value is the sum of two scores, about as large as the
    # rounding of its choices
    m, groups = 4000, n // 2
    kept = groups // 2
    k = 4
    x = O.store(0.01 * normal(n, m * n).reshape(m, n) - (0.0 if score == "softmax" else 8.0), "f32")
    t = spread * (0.5 + 0.5 * uniform01(n + 1, groups))
    bias = np.stack([t, -t], 1).reshape(-1).astype(np.float32)
    values = O.load(x)
    s = O.scores(score, values, np.ones(x.shape, bool))
    by = (s + bias.astype(np.float64)).reshape(m, groups, 2)
    total = by.sum(2)
    order = np.argsort(-total, axis=1, kind="stable")[:, :kept]
    open_ = np.zeros((m, groups), bool)
    np.put_along_axis(open_, order, True, 1)
    want = np.argsort(-np.where(open_[:, :, None], by, -np.inf).reshape(m, n), axis=1, kind="stable")[:, :k]
    W, I = F.route(Tensor.from_numpy(hip_backend, x), k, score, bias=Tensor.from_numpy(hip_backend, bias), groups=groups, kept_groups=kept, group_best=2)
    hip_backend.synchronize()
    # (64 bits cannot order groups whose sums differ by less than their own rounding: left out)
    ranked = np.sort(-total, axis=1)
    clear = ranked[:, kept] - ranked[:, kept - 1] > 64 * 2.0 ** -53 * spread
    assert clear.mean() > 0.99
    assert np.array_equal(I.numpy()[clear], want[clear])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,k", [(16, 4), (300, 6), (64, 20)])
@pytest.mark.parametrize("low", [-82.0, -88.0, -100.0, -5000.0])
def test_renormalised_scores_near_and_below_the_end_of_fp32(hip_backend, dtype, n, k, low):
    # logistic scores of about exp(low): only their ratios count
    m = 33
    x = O.store(low - 3.0 * uniform01(7, m * n).reshape(m, n) if low > -1000 else np.round(low - 3.0 * uniform01(7, m * n).reshape(m, n)), dtype)
    X, values = Tensor.from_numpy(hip_backend, x), O.load(x)
    # ratios from exp(x - top) / (1 + exp(x)): the second factor is 1 in 64 bits
    I0 = np.argsort(-values, axis=1, kind="stable")[:, :k]
    v = np.take_along_axis(values, I0, 1)
    q = np.exp(v - v[:, :1])
    q /= q.sum(1, keepdims=True)
    W, I = F.route(X, k, "sigmoid", renormalise=True, scale=2.5)
    hip_backend.synchronize()
    assert np.array_equal(I.numpy(), I0)
    assert O.close(W.numpy(), 2.5 * q, T.BOUND * 2.5 * q, "f32")
    # the gradient under a loss scaled by 2^16: d(w)/dx = q (d - sum d q) with 1 - s = 1
    dw = (65536 * normal(8, m * k)).astype(np.float32).reshape(m, k)
    G = F.route_grad(X, Tensor.from_numpy(hip_backend, I0.astype(np.int32)), Tensor.from_numpy(hip_backend, dw), "sigmoid", renormalise=True, scale=2.5)
    hip_backend.synchronize()
    d = 2.5 * dw.astype(np.float64)
    mean = (d * q).sum(1, keepdims=True)
    want, size = np.zeros((m, n)), np.zeros((m, n))
    np.put_along_axis(want, I0, q * (d - mean), 1)
    np.put_along_axis(size, I0, q * (np.abs(d) + (np.abs(d) * q).sum(1, keepdims=True)), 1)
    assert np.isfinite(want).all()
    assert O.close(G.numpy(), want, 2 * T.BOUND * size, dtype)


def test_renormalised_scores_of_both_signs(hip_backend):
    # chosen logits from -120 to 120 in one row: weights and gradients from ratios to the largest score
    m, n, k = 64, 24, 10
    x = O.store(240.0 * uniform01(17, m * n).reshape(m, n) - 120.0, "f32")
    x[0], x[1] = O.store(-np.arange(n, dtype=np.float64) - 86.0, "f32"), O.store(np.arange(n, dtype=np.float64) + 90.0, "f32")
    X, values = Tensor.from_numpy(hip_backend, x), O.load(x)
    idx = np.stack([np.argsort(uniform01(100 + r, n))[:k] for r in range(m)])
    W, I = F.route(X, k, "sigmoid", renormalise=True)
    hip_backend.synchronize()
    s = O.sigmoid(np.take_along_axis(values, I.numpy().astype(np.int64), 1))
    want = s / s.sum(1, keepdims=True)
    # terms (1.5 |x| + 2) u of the exponential of a logit up to 120 below 0
    assert O.close(W.numpy(), want, (180 * O.U + T.BOUND) * want, "f32")
    dw = normal(18, m * k).astype(np.float32).reshape(m, k)
    G = F.route_grad(X, Tensor.from_numpy(hip_backend, idx.astype(np.int32)), Tensor.from_numpy(hip_backend, dw), "sigmoid", renormalise=True)
    hip_backend.synchronize()
    v = np.take_along_axis(values, idx, 1)
    s = O.sigmoid(v)
    q = s / s.sum(1, keepdims=True)
    d = dw.astype(np.float64)
    g, size = np.zeros((m, n)), np.zeros((m, n))
    np.put_along_axis(g, idx, q * (d - (d * q).sum(1, keepdims=True)) * O.sigmoid(-v), 1)
    np.put_along_axis(size, idx, q * (np.abs(d) + (np.abs(d) * q).sum(1, keepdims=True)) * O.sigmoid(-v), 1)
    assert O.close(G.numpy(), g, (4 * 180 * O.U + 2 * T.BOUND) * size, "f32")
