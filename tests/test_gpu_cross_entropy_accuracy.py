"""Single elements of an fp32 gradient: how exact they are far below the row's maximum, and the ends of their range."""
import numpy as np
import pytest

import sequence_oracle as O
from dlf_amd import frontend as F
from dlf_amd.frontend import Tensor
from helpers import uniform01

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [3, 300, 20000, 70000])
def test_elements_far_below_the_maximum(hip_backend, n):
    # logits in steps of 2^-10, so that differences are exact; against the row's largest element, which the sum and the
    # weight divide out of: a distance d costs d u / 22 for ln 2 as it is rounded, the function 2 u, products, the
    # difference left and its square 4 u, the largest element itself 2 u
    m = 6
    x = np.round(-60.0 * uniform01(n, m * n).reshape(m, n) * 1024) / 1024
    x[:, 0], x[:, -1] = 0.0, -50.0
    t = np.full(m, n - 1)
    X, T = Tensor.from_numpy(hip_backend, x.astype(np.float32)), Tensor.from_numpy(hip_backend, t)
    state = F.cross_entropy_piece(X, T, 0)
    for dX in (F.cross_entropy_grad(X, T)[1], F.cross_entropy_piece_grad(X, T, 0, state)):
        hip_backend.synchronize()
        g = dX.numpy().astype(np.float64)[:, :-1]
        ratio, want = g / g[:, :1], np.exp(x[:, :-1])
        assert (np.abs(ratio - want) <= (-x[:, :-1] / 22 + 8) * O.U * want).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_elements_at_the_ends_of_the_range(hip_backend, dtype):
    # -inf, the lowest value and what lies thousands below the maximum have no part in the gradient; a NaN that the state
    # has not met still shows
    n, m = 700, 4
    x = O.store(np.zeros((m, n)), dtype)
    x[:, 3:9] = O.store(np.array([-np.inf, O.LOWEST[dtype], -2.0 ** 126, -5000.0, -300.0, -110.0]), dtype)
    t = np.full(m, 1)
    X, T = Tensor.from_numpy(hip_backend, x), Tensor.from_numpy(hip_backend, t)
    state = F.cross_entropy_piece(X, T, 0)
    dirty = x.copy()
    dirty[2, 50] = O.store(np.float32(np.nan), dtype)
    whole, piece = F.cross_entropy_grad(X, T)[1], F.cross_entropy_piece_grad(Tensor.from_numpy(hip_backend, dirty), T, 0, state)
    hip_backend.synchronize()
    p = 1 / (n - 6)
    want = np.full((m, n), p)
    want[:, 3:9] = 0.0
    want[:, 1] -= 1
    for g in (O.load(whole.numpy()), O.load(piece.numpy())):
        at = np.isnan(g)
        g = np.where(at, want, g)
        assert (np.abs(g - want) <= (1 + O.HALF_STEP[dtype]) * (8 * O.U + O.HALF_STEP[dtype]) * np.abs(want) + 8 * O.U * p).all()
    assert not np.isnan(O.load(whole.numpy())).any() and np.argwhere(at).tolist() == [[2, 50]]
