"""Timed cases of the sequence-model operators: gated_scan and its gradient, route and its gradient,
cross_entropy whole and in pieces of the vocabulary.

Every case has a plain form in elementary torch operations (32 bits, 64 where two candidates can lie
closer than 32 bits tell apart) and the call a user makes of this package (`own`)."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one new token for each of 48 sequences: the state is updated, latency is all
        dict(name="scan_decode", op="scan", kind="gated_blend", dtype="bf16", batch=48, steps=1, channels=2560, inner="channels"),
        # a training batch's forward pass, channels innermost
        dict(name="scan_batch", op="scan", kind="gated_blend", dtype="bf16", batch=8, steps=4096, channels=2048, inner="channels"),
        # one long document, few channels: the time axis has to be shared out
        dict(name="scan_long", op="scan", kind="gated_exp", dtype="f32", batch=1, steps=65536, channels=1000, inner="channels"),
        # time innermost (channels-first layers), rows of no whole cache lines
        dict(name="scan_rows", op="scan", kind="gated_sigmoid", dtype="f16", batch=4, steps=5001, channels=1536, inner="steps"),
        # the batch's backward pass
        dict(name="scan_grad_batch", op="scan_grad", kind="gated_sigmoid", dtype="bf16", batch=8, steps=4096, channels=2048, inner="channels"),
        # odd sizes in single precision, as a small model is fine-tuned
        dict(name="scan_grad_odd", op="scan_grad", kind="gated_blend", dtype="f32", batch=3, steps=1777, channels=515, inner="channels"),
        # a decode step's router
        dict(name="route_decode", op="route", score="softmax", dtype="bf16", tokens=24, experts=64, k=6, groups=1, kept=1, best=1, bias=False, renormalise=True, scale=1.0),
        # a prefill's router: sigmoid scores, bias for balance, groups
        dict(name="route_grouped", op="route", score="sigmoid", dtype="f32", tokens=32768, experts=256, k=8, groups=8, kept=4, best=2, bias=True, renormalise=True, scale=2.5),
        # a training step's router with its gradient, an odd number of tokens
        dict(name="route_train", op="route_grad", score="softmax", dtype="bf16", tokens=65537, experts=128, k=8, groups=1, kept=1, best=1, bias=False, renormalise=True, scale=1.0),
        # scoring a short text: the loss alone, few rows
        dict(name="loss_eval", op="loss", dtype="f32", rows=64, vocabulary=32000, z=0.0),
        # a training step's loss and gradient over a large vocabulary
        dict(name="loss_train", op="loss_grad", dtype="bf16", rows=8192, vocabulary=128000, z=1e-4),
        # the same in pieces of the vocabulary, rows of odd length
        dict(name="loss_pieces", op="loss_pieces", dtype="f16", rows=4096, vocabulary=50257, piece=8192, z=0.0),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, evenly over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["scan", "scan", "scan_grad", "route", "route_grad", "loss", "loss_grad", "loss_pieces"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op in ("scan", "scan_grad"):
        steps = 1 if op == "scan" and rng.random() < 0.15 else _spread(rng, 2, 65536)
        channels = _spread(rng, 3, 4096)
        batch = _spread(rng, 1, max(1, min(64, 50_000_000 // (steps * channels))))
        return dict(op=op, kind=rng.choice(["gated", "gated_exp", "gated_sigmoid", "gated_blend"]), dtype=dtype, batch=batch,
                    steps=steps, channels=channels, inner=rng.choice(["channels", "channels", "steps"]))
    if op in ("route", "route_grad"):
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _spread(rng, 4, 512 // groups)
        kept = rng.randint(1, groups)
        return dict(op=op, score=rng.choice(["softmax", "sigmoid"]), dtype=dtype, tokens=_spread(rng, 1, 65536), experts=experts,
                    k=rng.randint(1, min(16, kept * experts // groups)), groups=groups, kept=kept, best=rng.choice([1, 2]),
                    bias=rng.random() < 0.5, renormalise=rng.random() < 0.6, scale=rng.choice([1.0, 2.5]))
    vocabulary = _spread(rng, 500, 256000)
    rows = _spread(rng, 1, max(1, min(16384, 500_000_000 // vocabulary)))
    case = dict(op=op, dtype=dtype, rows=rows, vocabulary=vocabulary, z=rng.choice([0.0, 1e-4]))
    if op == "loss_pieces":
        case["piece"] = max(64, vocabulary // rng.randint(2, 8))
    return case


# ---------------------------------------------------------------- inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def prepare(case, seed):
    gen, dtype = _generator(seed), DTYPES[case["dtype"]]

    def normal(*shape, mean=0.0, std=1.0, to=torch.float32):
        return (torch.randn(*shape, generator=gen, device="cuda") * std + mean).to(to)

    if case["op"] in ("scan", "scan_grad"):
        b, t, c = case["batch"], case["steps"], case["channels"]
        shape = (b, t, c) if case["inner"] == "channels" else (b, c, t)
        axis = 1 if case["inner"] == "channels" else 2
        gate = normal(*shape, mean=2.0, std=1.5)
        # packed sequences: the state starts anew about every 1500 steps
        starts = torch.rand(b, t, generator=gen, device="cuda") < 1 / 1500
        starts = starts[:, :, None] if axis == 1 else starts[:, None, :]
        if case["kind"] == "gated":
            gate = torch.sigmoid(gate).masked_fill_(starts, 0.0)
        elif case["kind"] == "gated_exp":
            gate = gate.neg_().exp_().log1p_().neg_().masked_fill_(starts, -math.inf)
        else:
            gate.masked_fill_(starts, -math.inf)
        state = dict(case=case, axis=axis, gate=gate.to(dtype), x=normal(*shape, to=dtype), initial=normal(b, c))
        if case["op"] == "scan":
            state["last"] = torch.empty(b, c, device="cuda")
        else:
            # the forward pass's states, as a training program keeps them
            state["y"] = _scan_plain(case["kind"], state["gate"], state["x"], state["initial"], axis)[0]
            state["dy"] = normal(*shape, to=dtype)
            state["dlast"] = normal(b, c)
        return state
    if case["op"] in ("route", "route_grad"):
        m, n = case["tokens"], case["experts"]
        state = dict(case=case, x=normal(m, n, std=1.5, to=dtype), bias=normal(n, std=0.05) if case["bias"] else None)
        if case["op"] == "route_grad":
            state["dweights"] = normal(m, case["k"])
        return state
    m, v = case["rows"], case["vocabulary"]
    targets = torch.randint(0, v, (m,), generator=gen, device="cuda", dtype=torch.int64)
    # padding at the batch's end counts for nothing
    targets.masked_fill_(torch.rand(m, generator=gen, device="cuda") < 0.05, -100)
    # the batch's mean; half precision trains with a scaled loss, or its gradients vanish
    weights = torch.full((m,), (16384.0 if dtype == torch.float16 else 1.0) / m, device="cuda")
    state = dict(case=case, targets=targets, weights=weights)
    if case["op"] == "loss_pieces":
        state["pieces"] = [(first, normal(m, min(case["piece"], v - first), std=2.0, to=dtype)) for first in range(0, v, case["piece"])]
    else:
        x = torch.empty(m, v, device="cuda", dtype=dtype)
        for r in range(0, m, 1024):
            x[r:r + 1024] = normal(min(1024, m - r), v, std=2.0, to=dtype)
        state["x"] = x
    return state


# ---------------------------------------------------------------- plain forms

def _gates(kind, gate):
    """a and its derivative by the gate, in 32 bits."""
    gate = gate.float()
    if kind == "gated":
        return gate, None
    if kind == "gated_exp":
        a = torch.exp(gate)
        return a, a
    a = torch.sigmoid(gate)
    return a, a * torch.sigmoid(-gate)


def _affine_scan(a, b):
    """h[t] = a[t] h[t-1] + b[t] along axis 1 from 0, joining spans of 1, 2, 4, ... steps."""
    a, b, span = a.clone(), b.clone(), 1
    while span < a.shape[1]:
        b = torch.cat([b[:, :span], b[:, span:] + a[:, span:] * b[:, :-span]], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return b


def _scan_plain(kind, gate, x, initial, axis):
    dtype = x.dtype
    a = _gates(kind, gate.movedim(axis, 1))[0]
    b = x.movedim(axis, 1).float()
    if kind == "gated_blend":
        b = b * torch.sigmoid(-gate.movedim(axis, 1).float())
    b = torch.cat([b[:, :1] + a[:, :1] * initial[:, None], b[:, 1:]], 1)
    h = _affine_scan(a, b)
    return h.to(dtype).movedim(1, axis).contiguous(), h[:, -1].contiguous()


def _scan_grad_plain(kind, gate, x, y, dy, initial, dlast, axis):
    dtype = x.dtype
    gate, x, y, dy = (v.movedim(axis, 1).float() for v in (gate, x, y, dy))
    a, da = _gates(kind, gate)
    # mu[t] = a[t] (dy[t] + mu[t+1]), from the last step to the first
    b = a * dy
    b = torch.cat([b[:, :-1], b[:, -1:] + a[:, -1:] * dlast[:, None]], 1)
    mu = _affine_scan(a.flip(1), b.flip(1)).flip(1)
    lam = dy + torch.cat([mu[:, 1:], dlast[:, None]], 1)
    before = torch.cat([initial[:, None], y[:, :-1]], 1)
    if kind == "gated_blend":
        dx, dgate = lam * torch.sigmoid(-gate), lam * (before - x)
    else:
        dx, dgate = lam, lam * before
    if da is not None:
        dgate = dgate * da
    return [v.to(dtype).movedim(1, axis).contiguous() for v in (dgate, dx)] + [mu[:, 0].contiguous()]


def _route_plain(case, x, bias):
    """Scores and choices in 64 bits: two experts' values can be closer than 32 bits tell apart."""
    s = torch.softmax(x.double(), 1) if case["score"] == "softmax" else torch.sigmoid(x.double())
    c = s if bias is None else s + bias.double()
    groups, m = case["groups"], x.shape[0]
    if case["kept"] < groups:
        by_group = c.view(m, groups, -1)
        best = min(case["best"], by_group.shape[2])
        value = by_group.sort(dim=2, descending=True).values[:, :, :best].sum(2)
        kept = value.sort(dim=1, descending=True, stable=True).indices[:, :case["kept"]]
        open_ = torch.zeros(m, groups, dtype=torch.bool, device=x.device).scatter_(1, kept, True)
        c = by_group.masked_fill(~open_[:, :, None], -math.inf).view(m, -1)
    idx = c.sort(dim=1, descending=True, stable=True).indices[:, :case["k"]]
    w = s.gather(1, idx)
    if case["renormalise"]:
        w = w / w.sum(1, keepdim=True)
    return (w * case["scale"]).float(), idx.int(), s


def _route_grad_plain(case, s, idx, dw):
    idx = idx.long()
    chosen, ds = s.gather(1, idx), dw.double() * case["scale"]
    if case["renormalise"]:
        total = chosen.sum(1, keepdim=True)
        ds = (ds - (ds * chosen).sum(1, keepdim=True) / total) / total
    full = torch.zeros_like(s).scatter_(1, idx, ds)
    if case["score"] == "softmax":
        return s * (full - (full * s).sum(1, keepdim=True))
    return full * s * (1 - s)


def _loss_plain(mx, total, target_logit, targets, z):
    log_total = torch.log(total)
    loss = log_total + (mx - target_logit)
    if z:
        loss = loss + z * (mx + log_total) ** 2
    return torch.where(targets < 0, torch.zeros_like(loss), loss)


def _loss_grad_plain(x, mx, total, targets, first, weights, z, e=None):
    e = torch.exp(x.float() - mx[:, None]) if e is None else e
    factor = 1 / total
    if z:
        factor = factor * (1 + 2 * z * (mx + torch.log(total)))
    e = e.mul_(factor[:, None])
    here = (targets >= first) & (targets < first + x.shape[1])
    at = torch.where(here, targets - first, torch.zeros_like(targets))
    e.scatter_add_(1, at[:, None], -here.float()[:, None])
    return e.mul_(torch.where(targets < 0, torch.zeros_like(weights), weights)[:, None]).to(x.dtype)


def _target_logit(x, targets, first, before):
    here = (targets >= first) & (targets < first + x.shape[1])
    at = torch.where(here, targets - first, torch.zeros_like(targets))
    return torch.where(here, x.gather(1, at[:, None])[:, 0].float(), before)


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "scan":
        return list(_scan_plain(case["kind"], s["gate"], s["x"], s["initial"], s["axis"]))
    if op == "scan_grad":
        return _scan_grad_plain(case["kind"], s["gate"], s["x"], s["y"], s["dy"], s["initial"], s["dlast"], s["axis"])
    if op == "route":
        return list(_route_plain(case, s["x"], s["bias"])[:2])
    if op == "route_grad":
        w, idx, scores = _route_plain(case, s["x"], s["bias"])
        return [w, idx, _route_grad_plain(case, scores, idx, s["dweights"]).to(s["x"].dtype)]
    targets, z = s["targets"], case["z"]
    none = torch.full(targets.shape, math.nan, device="cuda")
    if op in ("loss", "loss_grad"):
        x = s["x"]
        mx = x.max(1).values.float()
        e = torch.exp(x.float() - mx[:, None])
        total = e.sum(1)
        loss = _loss_plain(mx, total, _target_logit(x, targets, 0, none), targets, z)
        return [loss] if op == "loss" else [loss, _loss_grad_plain(x, mx, total, targets, 0, s["weights"], z, e)]
    mx, total, logit = torch.full_like(none, -math.inf), torch.zeros_like(none), none
    for first, x in s["pieces"]:
        new = torch.maximum(mx, x.max(1).values.float())
        total = total * torch.exp(mx - new) + torch.exp(x.float() - new[:, None]).sum(1)
        mx, logit = new, _target_logit(x, targets, first, logit)
    return [_loss_plain(mx, total, logit, targets, z)] + [_loss_grad_plain(x, mx, total, targets, first, s["weights"], z) for first, x in s["pieces"]]


# ---------------------------------------------------------------- the package's calls

def _run_own(s):
    from dlf_amd import frontend as F
    from dlf_amd.hip_backend import default_backend
    hip = default_backend()
    D, T = hip.from_torch, hip.to_torch
    case = s["case"]
    op = case["op"]
    if op == "scan":
        y, last = F.gated_scan(D(s["gate"]), D(s["x"]), s["axis"], case["kind"], initial=D(s["initial"]), last=D(s["last"]))
        return [T(y), T(last)]
    if op == "scan_grad":
        got = F.gated_scan_grad(D(s["gate"]), D(s["x"]), D(s["y"]), D(s["dy"]), s["axis"], case["kind"], initial=D(s["initial"]), dlast=D(s["dlast"]))
        return [T(v) for v in got]
    if op in ("route", "route_grad"):
        x, bias = D(s["x"]), None if s["bias"] is None else D(s["bias"])
        w, idx = F.route(x, case["k"], case["score"], bias=bias, groups=case["groups"], kept_groups=case["kept"], group_best=case["best"],
                         renormalise=case["renormalise"], scale=case["scale"])
        if op == "route":
            return [T(w), T(idx)]
        dx = F.route_grad(x, idx, D(s["dweights"]), case["score"], renormalise=case["renormalise"], scale=case["scale"])
        return [T(w), T(idx), T(dx)]
    targets, z = D(s["targets"]), case["z"]
    if op == "loss":
        return [T(F.cross_entropy(D(s["x"]), targets, z_loss=z))]
    weights = D(s["weights"])
    if op == "loss_grad":
        return [T(v) for v in F.cross_entropy_grad(D(s["x"]), targets, weights, z_loss=z)]
    pieces, state = [(first, D(x)) for first, x in s["pieces"]], None
    for first, x in pieces:
        state = F.cross_entropy_piece(x, targets, first, state)
    loss = F.cross_entropy_join(state, targets, z_loss=z)
    return [T(loss)] + [T(F.cross_entropy_piece_grad(x, targets, first, state, weights, z_loss=z)) for first, x in pieces]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] in ("scan", "scan_grad"):
        rows = case["batch"] * case["channels"]
        count = rows * case["steps"]
        if case["op"] == "scan":
            return {"bytes": 3 * size * count + 8 * rows, "flops": 2 * count}
        return {"bytes": (6 if case["kind"] == "gated_blend" else 5) * size * count + 12 * rows, "flops": 6 * count}
    if case["op"] in ("route", "route_grad"):
        m, n, k = case["tokens"], case["experts"], case["k"]
        if case["op"] == "route":
            return {"bytes": m * n * size + 8 * m * k + 4 * n, "flops": 4 * m * n}
        return {"bytes": 2 * m * n * size + 12 * m * k + 4 * n, "flops": 8 * m * n}
    count = case["rows"] * case["vocabulary"]
    return {"bytes": (1 if case["op"] == "loss" else 2) * size * count + 16 * case["rows"], "flops": 4 * count}


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("scan", "scan_grad"):
        to_front = lambda v: v.movedim(s["axis"], 0).double()          # noqa: E731
        gate, x = to_front(s["gate"]), to_front(s["x"])
        a = {"gated": lambda: gate, "gated_exp": lambda: torch.exp(gate)}.get(case["kind"], lambda: 1 / (1 + torch.exp(-gate)))()
        keep = 1 / (1 + torch.exp(gate)) if case["kind"] == "gated_blend" else torch.ones_like(a)
        if op == "scan":
            out, h = torch.empty_like(x), s["initial"].double()
            for t in range(x.shape[0]):
                h = torch.addcmul(keep[t] * x[t], a[t], h, out=out[t])
            return [out.movedim(0, s["axis"]), h.clone()]
        y, dy = to_front(s["y"]), to_front(s["dy"])
        carry, lam = s["dlast"].double(), torch.empty_like(x)
        for t in range(x.shape[0] - 1, -1, -1):
            torch.add(dy[t], carry, out=lam[t])
            carry = a[t] * lam[t]
        slope = {"gated": lambda: torch.ones_like(a), "gated_exp": lambda: a}.get(case["kind"], lambda: a / (1 + torch.exp(gate)))()
        slope = torch.where(a == 0, torch.zeros_like(a), slope) if case["kind"] != "gated" else slope
        before = torch.cat([s["initial"].double()[None], y[:-1]])
        dgate = lam * slope * (before - x if case["kind"] == "gated_blend" else before)
        return [dgate.movedim(0, s["axis"]), (lam * keep).movedim(0, s["axis"]), carry]
    if op in ("route", "route_grad"):
        x, m, n = s["x"].double(), case["tokens"], case["experts"]
        if case["score"] == "softmax":
            p = torch.exp(x - x.amax(1, keepdim=True))
            p = p / p.sum(1, keepdim=True)
        else:
            p = 1 / (1 + torch.exp(-x))
        c = p.clone() if s["bias"] is None else p + s["bias"].double()
        if case["kept"] < case["groups"]:
            g = c.view(m, case["groups"], n // case["groups"])
            value = g.amax(2)
            if case["best"] == 2 and g.shape[2] > 1:
                value = g.topk(2, 2).values.sum(2)
            opened = torch.zeros_like(value)
            for _ in range(case["kept"]):
                at = value.argmax(1, keepdim=True)
                opened.scatter_(1, at, 1.0)
                value = value.scatter(1, at, -math.inf)
            c = torch.where(opened.repeat_interleave(n // case["groups"], 1) > 0, c, torch.full_like(c, -math.inf))
        picks = []
        for _ in range(case["k"]):
            # the first of equal values: argmax of the truth value "is the largest"
            at = (c == c.amax(1, keepdim=True)).to(torch.int8).argmax(1, keepdim=True)
            picks.append(at)
            c = c.scatter(1, at, -math.inf)
        idx = torch.cat(picks, 1)
        q = p.gather(1, idx)
        norm = q.sum(1, keepdim=True) if case["renormalise"] else torch.ones(m, 1, device="cuda", dtype=torch.float64)
        w = case["scale"] * q / norm
        if op == "route":
            return [w, None]
        up = case["scale"] * s["dweights"].double() / norm
        if case["renormalise"]:
            up = up - (up * q).sum(1, keepdim=True) / norm
        slope = torch.zeros_like(p).scatter_(1, idx, up)
        if case["score"] == "softmax":
            return [w, None, p * slope - p * (p * slope).sum(1, keepdim=True)]
        return [w, None, slope * p / (1 + torch.exp(x))]
    targets = s["targets"]
    live = targets >= 0
    x = torch.cat([p for _, p in s["pieces"]], 1) if op == "loss_pieces" else s["x"]
    losses, grads = [], []
    for r in range(0, case["rows"], 512):
        part, t, on = x[r:r + 512].double(), targets[r:r + 512].clamp(min=0), live[r:r + 512]
        lse = torch.logsumexp(part, 1)
        losses.append(torch.where(on, lse - part.gather(1, t[:, None])[:, 0] + case["z"] * lse ** 2, torch.zeros_like(lse)))
        if op != "loss":
            g = torch.exp(part - lse[:, None]) * (1 + 2 * case["z"] * lse)[:, None]
            g.scatter_add_(1, t[:, None], torch.full((t.shape[0], 1), -1.0, device="cuda", dtype=torch.float64))
            grads.append(g.mul_(torch.where(on, s["weights"][r:r + 512].double(), torch.zeros_like(lse))[:, None]))
    loss = torch.cat(losses)
    if op == "loss":
        return [loss]
    grad = torch.cat(grads)
    if op == "loss_grad":
        return [loss, grad]
    return [loss] + [grad[:, first:first + p.shape[1]].contiguous() for first, p in s["pieces"]]
