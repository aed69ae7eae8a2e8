"""The gradient of gates that several elements share: every element's own, summed over the shared extent."""
import numpy as np
import pytest

import sequence_oracle as O
from dlf_amd import frontend as F
from dlf_amd.frontend import Tensor
from dlf_amd.shape import Shape
from test_gpu_gated_scan import check_forward, check_grad, columns, pair, stored

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,width", [(7, 10), (3, 64), (2, 1)])
def test_a_gate_for_every_head(hip_backend, dtype, heads, width):
    kind, B, T = "gated_sigmoid", 2, 130
    g = stored(kind, 11, (B, T, heads), dtype, gate=True)
    base = Tensor.from_numpy(hip_backend, g)
    G = base.view(Shape((B, T, heads, width), (T * heads, heads, 1, 0)))
    full = np.repeat(g[..., None], width, axis=-1)
    X, dY = (pair(hip_backend, stored(kind, 12 + i, (B, T, heads, width), dtype)) for i in range(2))
    Y, _ = check_forward(hip_backend, kind, dtype, (G, full), X, 1)
    dG = check_grad(hip_backend, kind, dtype, (G, full), X, (Y, Y.numpy()), dY, 1)[0]
    if dtype == "bf16":
        one = Tensor.from_numpy(hip_backend, O.store(np.ones(1), dtype))
        _, shared = F.gated_scan(one.view(Shape(dG.shape.extents, (0,) * 4)), dG, 3, "gated")
    else:
        shared = F.reduce("reduce_sum", dG, [3])
    hip_backend.synchronize()
    each = O.load(dG.numpy())
    got = O.load(shared.numpy()) if shared.dtype != np.float32 else shared.numpy().astype(np.float64)
    assert got.shape == (B, T, heads)
    # a rounding per addend, and where the sum is stored in 16 bits its own
    half = O.HALF_STEP["f16"] if dtype == "f16" else 0.0
    assert (np.abs(got - each.sum(-1)) <= width * O.U * np.abs(each).sum(-1) + half * np.abs(each.sum(-1)) + O.TINY[dtype]).all()
    # and it is the gate's own gradient: the 64-bit one, every element within the stored type's rounding
    want = O.gated_scan_grad(kind, columns(full, 1, False), None, columns(Y.numpy(), 1, False), columns(dY[1], 1, False), np.zeros(B * heads * width),
                             np.zeros(B * heads * width))[0][0]
    want = np.moveaxis(want.reshape(T, B, heads, width), 0, 1)
    room = (2 * O.HALF_STEP[dtype] + 64 * O.U) * (np.abs(want).sum(-1) + np.abs(each).sum(-1)) + 2 * O.TINY[dtype] * width
    assert (np.abs(got - want.sum(-1)) <= room).all()
