"""How exact single elements of an fp32 gradient are, far below the row's maximum."""
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
