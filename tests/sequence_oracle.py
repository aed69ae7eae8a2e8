"""Plain 64-bit forms of the sequence-model operators, written from their definitions, with the
bounds that the tests hold the fp32 kernels to.

u = 2^-24 is the relative size of one fp32 rounding.  An output rounded to its own type is off by at
most half a step more: 2^-24 (fp32), 2^-11 (half, below its normal range 2^-25 absolute), 2^-8
(bfloat16)."""
import numpy as np

from dlf_amd.frontend import BFLOAT16, from_bfloat16, to_bfloat16

U = 2.0 ** -24
TYPES = {"f32": np.dtype(np.float32), "f16": np.dtype(np.float16), "bf16": BFLOAT16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
# smallest magnitudes that are rounded absolutely (half the smallest subnormal; flushed fp32 / bf16 numbers)
TINY = {"f32": 2.0 ** -125, "f16": 2.0 ** -25, "bf16": 2.0 ** -125}


def store(a, kind):
    """An array in the named type, as the kernels get it."""
    return to_bfloat16(np.asarray(a, np.float32)) if kind == "bf16" else np.asarray(a).astype(TYPES[kind])


def load(a):
    """The 64-bit values of an array of any of the types."""
    return (from_bfloat16(a) if a.dtype == BFLOAT16 else a).astype(np.float64)


def sigmoid(g):
    e = np.exp(-np.abs(g))
    return np.where(g < 0, e / (1 + e), 1 / (1 + e))


def gates(kind, g):
    """(a, factor of x, derivative of a by g)"""
    one = np.ones_like(g)
    if kind == "gated":
        return g, one, one
    if kind == "gated_exp":
        return np.exp(g), one, np.exp(g)
    a, keep = sigmoid(g), sigmoid(-g)
    return a, (keep if kind == "gated_blend" else one), a * keep


def _gate_error(kind, g):
    """Relative error of a gate function in fp32, in units of u: the rounded product under the
    hardware's 2^x moves the exponent by |g| log2(e) u / 2, which is |g| u of the result (twice that
    allowed); the function, the sum, the reciprocal and a product are within 2 u each."""
    finite = np.where(np.isfinite(g), np.abs(g), 0.0)
    return 0.0 * finite if kind == "gated" else 8.0 + 2.0 * finite


def gated_scan(kind, g, x, initial):
    """g, x [n, m] in 64 bits, initial [m]: (h [n, m], bound of the fp32 state's error [n, m]).

    Every product of gates along a path from an input to a state carries, per step, the gate's own
    error and at most four roundings (its product, the sum, and where the axis is cut the product
    of the cut's gates and its joining), however it is associated: E follows the recurrence of the
    absolute values."""
    a, fx, _ = gates(kind, g)
    b = fx * x
    k = (_gate_error(kind, g) + 4.0) * U
    h, M, E = initial.copy(), np.abs(initial), np.zeros_like(initial)
    out, err = np.empty_like(x), np.empty_like(x)
    for t in range(x.shape[0]):
        E = np.abs(a[t]) * E + 2 * k[t] * (np.abs(a[t]) * M + np.abs(b[t]))
        M = np.abs(a[t]) * M + np.abs(b[t])
        h = a[t] * h + b[t]
        out[t], err[t] = h, E
    return out, err


def gated_scan_grad(kind, g, x, y, dy, initial, dlast):
    """All [n, m] in 64 bits: (dg, dx, dinitial) and the bounds of their errors before the rounding to the type."""
    a, fx, slope = gates(kind, g)
    k = (_gate_error(kind, g) + 4.0) * U
    mu, M, E = dlast.copy(), np.abs(dlast), np.zeros_like(dlast)
    lam, lam_err, lam_abs = np.empty_like(dy), np.empty_like(dy), np.empty_like(dy)
    for t in range(dy.shape[0] - 1, -1, -1):
        lam[t] = dy[t] + mu
        lam_abs[t] = np.abs(dy[t]) + M
        lam_err[t] = E + U * lam_abs[t]
        mu = a[t] * lam[t]
        M = np.abs(a[t]) * lam_abs[t]
        E = np.abs(a[t]) * lam_err[t] + 2 * k[t] * M
    before = np.concatenate([initial[None], y[:-1]])
    if kind == "gated_blend":
        before = before - x
    side = before * slope
    dg, dx = lam * side, lam * fx
    # the slope is two gate functions and their product, each factor's error relative
    dg_err = np.abs(side) * lam_err + (2 * k + 4 * U) * np.abs(side) * np.abs(lam)
    dx_err = np.abs(fx) * lam_err + (k + 2 * U) * np.abs(fx * lam)
    return (dg, dx, mu), (dg_err, dx_err, E + U * M)


def close(got, want, bound, kind):
    """Whether every element is within the bound and half a step of its type (infinities and NaN alike)."""
    got = load(got) if got.dtype in (BFLOAT16, np.dtype(np.float16), np.dtype(np.float32)) else got
    finite = np.isfinite(want)
    if not np.array_equal(np.isnan(got), np.isnan(want)) or not np.array_equal(got[~finite & ~np.isnan(want)], want[~finite & ~np.isnan(want)]):
        return False
    off = np.abs(got - want)[finite]
    room = (np.broadcast_to(bound, want.shape) * (1 + HALF_STEP[kind]) + HALF_STEP[kind] * np.abs(want) + TINY[kind])[finite]
    return bool((off <= room).all())


# ---------------------------------------------------------------- route

LOWEST = {"f32": -np.finfo(np.float32).max.astype(np.float64), "f16": -65504.0, "bf16": -float(from_bfloat16(np.array([0x7f7f], np.uint16).view(BFLOAT16))[0])}


def scores(kind, x, present):
    if kind == "sigmoid":
        return np.where(present, sigmoid(np.where(present, x, 0.0)), 0.0)
    s = np.zeros_like(x)
    for r in range(x.shape[0]):
        p = present[r]
        if p.any():
            e = np.exp(x[r, p] - x[r, p].max())
            s[r, p] = e / e.sum()
    return s


def route(kind, x, lowest, k, bias=None, groups=1, kept=None, best=1, renormalise=False, scale=1.0):
    """Row by row, by sorting: (weights, indices, scores)."""
    m, n = x.shape
    kept = groups if kept is None else kept
    size = n // groups
    present = ~(x <= lowest)
    s = scores(kind, x, present)
    by = s + (0.0 if bias is None else bias[None, :]) if bias is not None or kept < groups else x
    W, I = np.zeros((m, k)), np.zeros((m, k), np.int64)
    for r in range(m):
        open_ = list(range(groups))
        if kept < groups:
            def value(g):
                c = sorted((by[r, e] for e in range(g * size, (g + 1) * size) if present[r, e]), reverse=True)[:best]
                return (0, 0.0) if not c else (1, sum(c))
            open_ = sorted(range(groups), key=lambda g: (-value(g)[0], -value(g)[1], g))[:kept]
        pool = [e for g in open_ for e in range(g * size, (g + 1) * size)]
        pool.sort(key=lambda e: (not present[r, e], -by[r, e] if present[r, e] else 0.0, e))
        I[r] = pool[:k]
        w = s[r, I[r]]
        if renormalise:
            w = w / w.sum() if w.sum() else 0 * w
        W[r] = scale * w
    return W, I, s


def route_grad(kind, x, lowest, indices, dw, renormalise=False, scale=1.0):
    m, n = x.shape
    present = ~(x <= lowest)
    s = scores(kind, x, present)
    ds = np.zeros_like(s)
    for r in range(m):
        ok = (indices[r] >= 0) & (indices[r] < n)
        idx, d = indices[r][ok], dw[r][ok] * scale
        q = s[r, idx]
        if renormalise:
            d = (d - (d * q).sum() / q.sum()) / q.sum() if q.sum() else 0 * d
        np.add.at(ds[r], idx, d)
    if kind == "softmax":
        return s * (ds - (ds * s).sum(1, keepdims=True))
    return ds * s * (1 - s)


# ---------------------------------------------------------------- cross entropy

def cross_entropy(x, targets, z=0.0, weights=None):
    """(loss, gradient of the weighted sum) with the module's rules for rows without a target or a logit."""
    m, n = x.shape
    w = np.ones(m) if weights is None else weights
    loss, grad = np.zeros(m), np.zeros((m, n))
    for r in range(m):
        t = int(targets[r])
        if t < 0:
            continue
        mx = x[r].max()
        if mx == -np.inf:
            loss[r] = np.inf
            continue
        e = np.exp(x[r] - mx)
        lse = mx + np.log(e.sum())
        loss[r] = np.nan if t >= n else np.log(e.sum()) + (mx - x[r, t]) + z * lse * lse
        p = e / e.sum() * (1 + 2 * z * lse)
        if t < n:
            p[t] -= 1
        grad[r] = w[r] * p
    return loss, grad
