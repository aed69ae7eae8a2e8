"""The sequence-model operators together: a training step through recurrence, router and loss against
64-bit automatic differentiation, a decoding loop, and the calls under graph capture, on several
streams and from several threads."""
import threading

import numpy as np
import pytest

import sequence_oracle as O
from dlf_amd import frontend as F
from dlf_amd.frontend import Tensor
from helpers import normal, randint

pytestmark = pytest.mark.gpu


def rand(seed, *shape, scale=1.0):
    return (scale * normal(seed, int(np.prod(shape)))).astype(np.float32).reshape(shape)


def test_training_step(hip_backend):
    """h = recurrence(g, x); w, i = route(h R); y = h * sum_j w_j E[i_j]; loss of y V^T in three pieces.

    Tolerance of the gradients, relative in the 2-norm: the recurrence's 40 steps with under 16 u each
    way, products of 48 to 200 terms with as many u, the router's 64 u and the loss's 60 u, every one of
    them on the way back too: under 2 (40 * 16 + 200 + 64 + 60) u < 2048 u, doubled for what they
    amplify in each other."""
    import torch
    B, T, C, N, K, V = 3, 40, 48, 12, 3, 200
    m = B * T
    g, x = rand(1, B, T, C) + 1.0, rand(2, B, T, C)
    R, E, U = rand(3, C, N, scale=0.3), rand(4, N, C), rand(5, V, C, scale=0.3)
    h0 = rand(6, B, C)
    targets = randint(7, m, 0, V)
    targets[::11] = -1
    weights = np.full(m, 1.0 / m, np.float32)

    # 64 bits, on the host
    p = {k: torch.tensor(v, dtype=torch.float64, requires_grad=True) for k, v in dict(g=g, x=x, R=R, E=E, U=U, h0=h0).items()}
    a = torch.sigmoid(p["g"])
    h, hs = p["h0"], []
    for t in range(T):
        h = a[:, t] * h + (1 - a[:, t]) * p["x"][:, t]
        hs.append(h)
    hm = torch.stack(hs, 1).reshape(m, C)
    s = torch.softmax(hm @ p["R"], 1)
    idx = torch.sort(s, dim=1, descending=True, stable=True).indices[:, :K]
    w = s.gather(1, idx)
    w = w / w.sum(1, keepdim=True)
    y = hm * (w[:, :, None] * p["E"][idx]).sum(1)
    logits = y @ p["U"].T
    live = torch.tensor(targets >= 0)
    tt = torch.tensor(np.maximum(targets, 0))
    loss = torch.where(live, torch.logsumexp(logits, 1) - logits.gather(1, tt[:, None])[:, 0], 0.0)
    (loss * torch.tensor(weights, dtype=torch.float64)).sum().backward()

    # the device
    D, A = (lambda v: Tensor.from_numpy(hip_backend, v)), hip_backend.to_torch
    wrap = hip_backend.from_torch
    dev = lambda v: torch.tensor(v, device=hip_backend.device)                    # noqa: E731
    G, X, S, Td, Wd = D(g), D(x), D(h0), D(targets), D(weights)
    Rd, Ed, Ud = dev(R), dev(E), dev(U)
    Y, _ = F.gated_scan(G, X, 1, "gated_blend", initial=S)
    H = A(Y).reshape(m, C)
    router = H @ Rd
    Wt, It = F.route(wrap(router), K, "softmax", renormalise=True)
    mix = (A(Wt)[:, :, None] * Ed[A(It).long()]).sum(1)
    y_dev = H * mix
    cuts = [(0, 64), (64, 129), (129, V)]
    state = None
    for lo, hi in cuts:
        state = F.cross_entropy_piece(wrap(y_dev @ Ud[lo:hi].T.contiguous()), Td, lo, state)
    loss_dev = F.cross_entropy_join(state, Td)
    dy, dU = torch.zeros_like(y_dev), torch.zeros_like(Ud)
    for lo, hi in cuts:
        piece = wrap(y_dev @ Ud[lo:hi].T.contiguous())
        dp = A(F.cross_entropy_piece_grad(piece, Td, lo, state, Wd, out=piece))
        dy += dp @ Ud[lo:hi]
        dU[lo:hi] = dp.T.contiguous() @ y_dev
    dmix = dy * H
    dW = (dmix[:, None, :] * Ed[A(It).long()]).sum(2)
    dE = torch.zeros_like(Ed).index_add_(0, A(It).long().reshape(-1), (A(Wt)[:, :, None] * dmix[:, None, :]).reshape(-1, C))
    drouter = A(F.route_grad(wrap(router), It, wrap(dW.contiguous()), "softmax", renormalise=True))
    dH = dy * mix + drouter @ Rd.T.contiguous()
    dG, dX, dS = F.gated_scan_grad(G, X, Y, wrap(dH.reshape(B, T, C).contiguous()), 1, "gated_blend", initial=S)
    hip_backend.synchronize()

    assert np.array_equal(A(It).cpu().numpy(), idx.numpy())
    room = 4096 * O.U
    for got, want in ((loss_dev.numpy(), loss.detach().numpy()), (dG.numpy(), p["g"].grad.numpy()), (dX.numpy(), p["x"].grad.numpy()),
                      (dS.numpy(), p["h0"].grad.numpy()), ((H.T.contiguous() @ drouter).cpu().numpy(), p["R"].grad.numpy()),
                      (dE.cpu().numpy(), p["E"].grad.numpy()), (dU.cpu().numpy(), p["U"].grad.numpy())):
        assert np.linalg.norm(got.astype(np.float64) - want) <= room * np.linalg.norm(want)


def every_call(D):
    """One call of everything, in shapes that take scratch, a second launch or several."""
    out = []
    y, last = F.gated_scan(D["g"], D["x"], 1, "gated_sigmoid", initial=D["h0"])                 # cut into segments
    out += [y, last, *F.gated_scan_grad(D["g"], None, y, D["dy"], 1, "gated_sigmoid", initial=D["h0"])]
    yr, lr = F.gated_scan(D["gr"], D["xr"], 1, "gated_blend")                                   # rows cut into segments
    out += [yr, lr]
    w, i = F.route(D["logits"], 4, "sigmoid", bias=D["bias"], groups=4, kept_groups=2, group_best=2, renormalise=True)
    out += [w, i, F.route_grad(D["logits"], i, w, "sigmoid", renormalise=True)]
    out += [F.cross_entropy(D["v"], D["t"]), *F.cross_entropy_grad(D["v"], D["t"], z_loss=1e-3)]     # tiles and records
    out += list(F.cross_entropy_grad(D["many"], D["tm"]))                                       # rows held in registers
    state = F.cross_entropy_piece(D["v"], D["t"], 0)
    state = F.cross_entropy_piece(D["v"], D["t"], 70000, state)
    out += [F.cross_entropy_join(state, D["t"]), F.cross_entropy_piece_grad(D["v"], D["t"], 0, state)]
    return out


def inputs(seed):
    g = rand(seed, 1, 3000, 70) + 1.5
    return dict(g=g, x=rand(seed + 1, 1, 3000, 70), dy=rand(seed + 2, 1, 3000, 70), h0=rand(seed + 3, 1, 70),
                gr=rand(seed + 4, 2, 40000), xr=rand(seed + 5, 2, 40000), logits=rand(seed + 6, 700, 64), bias=np.round(rand(seed + 7, 64), 1),
                v=rand(seed + 8, 3, 70000), t=np.array([5, 69999, -1]), many=rand(seed + 9, 300, 9000), tm=randint(seed + 10, 300, 0, 9000))


def test_capture_and_replay(hip_backend):
    # two recorded graphs with their own inputs, replayed in turn with eager calls between
    import torch
    sets = [inputs(1000), inputs(2000)]
    dev = [{k: Tensor.from_numpy(hip_backend, v) for k, v in s.items()} for s in sets]
    for D in dev:
        every_call(D)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for D in dev:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(every_call(D))
        graphs.append(graph)
    for r in range(3):
        for k, D in enumerate(dev):
            fresh = inputs(3000 + 100 * r + 10 * k)
            for name, T in D.items():
                T.storage.copy_(torch.from_numpy(np.ascontiguousarray(fresh[name]).reshape(-1)))
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for D, recorded in zip(dev, outs):
            got = [o.numpy() for o in recorded]
            want = [o.numpy() for o in every_call(D)]          # the same calls, eagerly: nothing depends on the order of atomics
            for i, (a, b) in enumerate(zip(got, want)):
                assert np.array_equal(a, b, equal_nan=True), (r, i)


def test_streams_and_threads(hip_backend):
    # the same calls from two threads, each on a stream of its own, give what one call after the other gives
    import torch
    sets = [inputs(5000), inputs(6000)]
    dev = [{k: Tensor.from_numpy(hip_backend, v) for k, v in s.items()} for s in sets]
    want = [[o.numpy() for o in every_call(D)] for D in dev]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(k):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(4):
                    out = every_call(dev[k])
            stream.synchronize()
            got[k] = [o.numpy() for o in out]
        except Exception as e:                                 # shown by the assertion below
            errors.append(e)
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for k in range(2):
        for i, (a, b) in enumerate(zip(got[k], want[k])):
            assert np.array_equal(a, b, equal_nan=True), (k, i)


def test_loads_add_up_over_calls(hip_backend):
    x = rand(71, 5000, 96)
    X = Tensor.from_numpy(hip_backend, x)
    loads = Tensor.from_numpy(hip_backend, np.zeros(96, np.int32))
    for _ in range(3):
        _, I = F.route(X, 5, loads=loads)
    hip_backend.synchronize()
    assert np.array_equal(loads.numpy(), 3 * np.bincount(I.numpy().reshape(-1), minlength=96))


def test_torch_views(hip_backend):
    import torch
    t = torch.arange(60, device=hip_backend.device, dtype=torch.float32).view(3, 4, 5)
    for v in (t, t[1], t[:, 1:3], t.transpose(0, 2), t[:, :, 2], t[0, 0, :1]):
        T = hip_backend.from_torch(v)
        assert np.array_equal(T.numpy(), v.cpu().numpy()) and torch.equal(hip_backend.to_torch(T), v)
    T = hip_backend.from_torch(t)
    assert torch.equal(hip_backend.to_torch(T.slice([1], [3], [1])), t[:, 1:3])
    with pytest.raises(ValueError):
        hip_backend.to_torch(T.flip([0]))
    with pytest.raises(ValueError):
        hip_backend.from_torch(torch.zeros(3))
    with pytest.raises(ValueError):
        hip_backend.from_torch(t[:0])
    b = torch.tensor([1.5, -2.0, 3.0], device=hip_backend.device, dtype=torch.bfloat16)
    assert np.array_equal(F.from_bfloat16(hip_backend.from_torch(b).numpy()), np.float32([1.5, -2.0, 3.0]))
    c = hip_backend.from_torch(b.expand(4, 3).contiguous()).transpose().contiguous()            # dlfx_copy of bfloat16
    assert np.array_equal(F.from_bfloat16(c.numpy()), np.repeat(np.float32([1.5, -2.0, 3.0]), 4).reshape(3, 4))
    z = Tensor.empty(hip_backend, (5,), F.BFLOAT16)
    hip_backend.fill(9, z.shape.extents, z.shape.strides, z.storage, 0, -0.75)
    hip_backend.synchronize()
    assert np.array_equal(F.from_bfloat16(z.numpy()), np.full(5, -0.75, np.float32))
