"""route at the ends of its range: sums of choices that cancel."""
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
