"""The normalised layer and the orthogonalised update through the C++ front-end: Tensor::group_norm on the tape,
muon_step_all, newton_schulz, and the demo network trained with both."""
import ctypes as C

import numpy as np
import pytest

import norm_oracle as N
import update_oracle as O
from support import HostLayer, f32, fp, write_mnist_dir

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def host():
    h = HostLayer()
    for n in ("group_norm", "muon_step", "newton_schulz"):
        getattr(h.cdll, "cth_" + n).restype = C.c_long
    return h


def _dims(shape):
    return (C.c_long * len(shape))(*shape), len(shape)


def _group_norm(host, x, groups, w, b, act, up=None, eps=1e-5):
    d, n = _dims(x.shape)
    y, dx, dw, db = np.empty_like(x), np.empty_like(x), np.empty_like(w), np.empty_like(b)
    rc = host.cdll.cth_group_norm(fp(x), d, n, C.c_long(groups), fp(w), fp(b), N.ACTS[act], C.c_float(eps), fp(y), None if up is None else fp(up),
                                  fp(dx), fp(dw), fp(db))
    return rc, y, dx, dw, db


@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("shape,groups", [((128, 64), 8), ((5, 6), 1), ((3, 7, 9, 24), 6), ((2, 40, 40, 64), 4), ((1, 10), 10)], ids=str)
def test_group_norm_and_its_tape_gradients(host, shape, groups, act):
    print("case host group norm", shape, groups, act, flush=True)
    r = np.random.default_rng(3)
    c = shape[-1]
    x, up = f32(r.standard_normal(shape) + 0.2), f32(r.standard_normal(shape))
    w, b = f32(r.uniform(0.5, 1.5, c)), f32(0.3 * r.standard_normal(c))
    rc, y, dx, dw, db = _group_norm(host, x, groups, w, b, act, up)
    assert rc == x.size
    flat = x.reshape(shape[0], -1, c)
    wy, wst, ey, _ = N.forward(flat, w, b, groups, act, 1e-5)
    assert np.all(np.abs(y.reshape(flat.shape) - wy) <= ey)
    # The tape's statistics are the kernel's, within DEPTH roundings of the 64-bit ones; the gradient's bound takes
    # them as given.  They move xhat, s1 and s2 by that relative amount each: 4 DEPTH roundings of the terms.
    want, err = N.backward(flat, w, b, wst.astype(np.float32), groups, act, up.reshape(flat.shape))
    g, rstd = np.abs(up.reshape(flat.shape)).astype(np.float64), np.repeat(wst[..., 1], c // groups, 1)[:, None]
    h = np.abs((flat - np.repeat(wst[..., 0], c // groups, 1)[:, None]) * rstd) + 1
    # An element whose z lies within the forward bound of 0 may take either side of ReLU: its whole term is open
    z, _, ez, _ = N.forward(flat, w, b, groups, "none", 1e-5)
    open_ = (g if act == "relu" else 0 * g) * (np.abs(z) <= ez)
    loose = 4 * N.DEPTH * N.U * g + open_
    mean = lambda v: np.broadcast_to(v.reshape(shape[0], -1, groups, c // groups).mean((1, 3), keepdims=True),  # noqa: E731
                                     (shape[0], flat.shape[1], groups, c // groups)).reshape(flat.shape)
    extra = (rstd * (w * loose + mean(w * loose) + h * mean(w * loose * h) + 4 * N.DEPTH * N.U * h * h * mean(w * g * h)), (loose * h).sum((0, 1)),
             loose.sum((0, 1)))
    for got, v, e, x_, name in zip((dx.reshape(flat.shape), dw, db), want, err, extra, ("dx", "dweight", "dbias")):
        assert np.all(np.abs(got - v) <= e + x_), (name, float(np.max(np.abs(got - v) - e - x_)))


def test_group_norm_refuses(host):
    print("case host group norm refusals", flush=True)
    x, w = np.ones((4, 6), np.float32), np.ones(6, np.float32)
    assert _group_norm(host, x, 4, w, w, "none")[0] == -1                     # 6 channels, 4 groups
    assert _group_norm(host, x, 0, w, w, "none")[0] == -1
    d, n = _dims((6,))
    y = np.empty(6, np.float32)
    assert host.cdll.cth_group_norm(fp(w), d, n, C.c_long(2), fp(w), fp(w), 0, C.c_float(1e-5), fp(y), None, None, None, None) == -1   # 1-D
    assert host.cdll.cth_group_norm(fp(x), _dims((4, 6))[0], 2, C.c_long(2), fp(w), fp(w), 9, C.c_float(1e-5), fp(np.empty_like(x)), None, None, None,
                                    None) == -1


def test_more_groups_than_channels_are_refused_before_their_statistics_are_allocated(host):
    print("case host group norm, 2^40 groups", flush=True)
    x, w = np.ones((4, 6), np.float32), np.ones(6, np.float32)
    assert _group_norm(host, x, 1 << 40, w, w, "none", up=x)[0] == -1
    assert _group_norm(host, x, 12, w, w, "none")[0] == -1
    assert _group_norm(host, x, 3, w, w, "none")[0] == x.size                  # and the next call is served


def _grad(rows, cols, seed):
    r = np.random.default_rng(seed)
    return f32(1e-3 * r.standard_normal((rows, cols)))


@pytest.mark.parametrize("nesterov", [0, 1])
def test_muon_step_in_place(host, nesterov):
    print("case host muon", nesterov, flush=True)
    shapes = [(128, 64), (64, 10), (70, 300)]
    p, g, m = ([f32(10 * _grad(*s, k + o)) if o != 50 else _grad(*s, k + o) for k, s in enumerate(shapes)] for o in (1, 50, 90))
    want = [O.muon(a, b, c, np.float32(0.2) * np.sqrt(np.float32(max(a.shape))), 0.02, 0.95, 0.01, bool(nesterov), 5) for a, b, c in zip(p, g, m)]
    ptrs = lambda v: (C.POINTER(C.c_float) * 3)(*[fp(a) for a in v])  # noqa: E731
    dims = (C.c_long * 6)(*sum(([*s] for s in shapes), []))
    before = [a.copy() for a in p]
    assert host.cdll.cth_muon_step(3, dims, ptrs(p), ptrs(g), ptrs(m), C.c_float(0.02), C.c_float(0.01), nesterov, 5, 1) == -1      # shapes differ
    assert all(np.array_equal(a, b) for a, b in zip(p, before))
    assert host.cdll.cth_muon_step(3, dims, ptrs(p), ptrs(g), ptrs(m), C.c_float(0.02), C.c_float(0.01), nesterov, 5, 0) == 3
    for a, c, (wp, wm, ep, em) in zip(p, m, want):
        assert np.all(np.abs(a - wp) <= ep) and np.all(np.abs(c - wm) <= em)


def test_newton_schulz_of_a_matrix_and_of_a_batch(host):
    print("case host newton schulz", flush=True)
    for shape in ((40, 90), (3, 65, 20)):
        g = f32(np.random.default_rng(5).standard_normal(shape))
        out = np.empty_like(g)
        d, n = _dims(shape)
        assert host.cdll.cth_newton_schulz(fp(g), d, n, 5, fp(out)) == g.size
        for a, b in zip(g.reshape(-1, *shape[-2:]), out.reshape(-1, *shape[-2:])):
            assert np.linalg.norm(b - O.newton_schulz(a)) <= O.newton_schulz_bound(a.shape, 5)
    d, n = _dims((8,))
    assert host.cdll.cth_newton_schulz(fp(np.ones(8, np.float32)), d, n, 5, fp(np.empty(8, np.float32))) == -1


def _train_oracle(x, labels, params, batch, steps, lr, groups=8, muon_lr=0.02):
    """The network of the demo in 64 bits: matmul + bias, group norm, ReLU, twice; logits; summed cross entropy;
    weight matrices by their orthogonalised momentum, the rest by gradient descent."""
    P = [p.astype(np.float64) for p in params]
    norm = [np.ones(P[1].size), np.zeros(P[1].size), np.ones(P[3].size), np.zeros(P[3].size)]
    mom = [np.zeros_like(P[k]) for k in (0, 2, 4)]
    losses = []
    def fwd(z, w, b):
        n, c = z.shape
        zg = z.reshape(n, groups, -1)
        mean, rstd = zg.mean(2, keepdims=True), 1 / np.sqrt(zg.var(2, keepdims=True) + 1e-5)
        h = ((zg - mean) * rstd).reshape(n, c)
        return np.maximum(h * w + b, 0), h, rstd
    def bwd(g, y, h, rstd, w):
        n, c = g.shape
        dz = g * (y > 0)
        d, hg = (dz * w).reshape(n, groups, -1), h.reshape(n, groups, -1)
        return ((d - d.mean(2, keepdims=True) - hg * (d * hg).mean(2, keepdims=True)) * rstd).reshape(n, c), (dz * h).sum(0), dz.sum(0)
    for s in range(steps):
        at = (s % (len(x) // batch)) * batch
        xb, yb = x[at:at + batch].astype(np.float64), labels[at:at + batch].astype(int)
        h1, n1, r1 = fwd(xb @ P[0] + P[1], norm[0], norm[1])
        h2, n2, r2 = fwd(h1 @ P[2] + P[3], norm[2], norm[3])
        z = h2 @ P[4] + P[5]
        e = np.exp(z - z.max(1, keepdims=True))
        q = e / e.sum(1, keepdims=True)
        losses.append(float(-np.log(np.maximum(q[np.arange(batch), yb], 1e-10)).sum()))
        dz = q.copy()
        dz[np.arange(batch), yb] -= 1
        gW3, gb3 = h2.T @ dz, dz.sum(0)
        d2, gn2w, gn2b = bwd(dz @ P[4].T, h2, n2, r2, norm[2])
        gW2, gb2 = h1.T @ d2, d2.sum(0)
        d1, gn1w, gn1b = bwd(d2 @ P[2].T, h1, n1, r1, norm[0])
        gW1, gb1 = xb.T @ d1, d1.sum(0)
        for k, (i, g) in enumerate(((0, gW1), (2, gW2), (4, gW3))):
            mom[k] = 0.95 * mom[k] + g
            P[i] = P[i] - muon_lr * 0.2 * np.sqrt(max(g.shape)) * O.newton_schulz(g + 0.95 * mom[k])
        for i, g in ((1, gb1), (3, gb2), (5, gb3)):
            P[i] = P[i] - lr * g
        for k, g in enumerate((gn1w, gn1b, gn2w, gn2b)):
            norm[k] = norm[k] - lr * g
    return np.array(losses), P


def test_the_network_trained_with_normalised_layers_and_orthogonalised_updates(host):
    """Three steps against the same network in 64 bits, operator by operator; fused layers and a step recorded into a
    graph and replayed give the same bits; the one-pass head agrees as it does without them."""
    print("case train with norm and muon", flush=True)
    r = np.random.default_rng(11)
    I, H1, H2, classes, batch, steps, lr = 60, 64, 48, 10, 32, 3, 1e-3
    x, y = f32(r.uniform(0, 1, (4 * batch, I))), f32(r.integers(0, classes, 4 * batch))
    params = [f32(r.uniform(-1, 1, s) / np.sqrt(s[0])) for s in ((I, H1), (H1,), (H1, H2), (H2,), (H2, classes), (classes,))]
    losses, P = host.mnist_train(x, y, params, batch, steps, lr, reference_tape=32 + 64)
    want_l, want_p = _train_oracle(x, y, params, batch, steps, lr)
    # A step's update is off by the iteration's own bound, and by the gradient's relative error (sums of at most
    # 64 terms in fp32 behind four operators: 256 roundings) magnified like any error of X_0; both times the step's
    # size.  A later step starts from that, and its gradient moves by at most as much again.
    unit = max(O.newton_schulz_bound(p.shape, 5) + 485 * 256 * N.U for p in params if p.ndim == 2)
    tol = 0.02 * 0.2 * 8 * unit * (2 ** steps - 1)
    for a, b in zip(P, want_p):
        assert np.abs(a - b).max() <= tol, (a.shape, float(np.abs(a - b).max()), tol)
    assert np.abs(losses - want_l).max() <= batch * I * tol
    assert losses[0] != losses[1]
    for mode in (2, 4, 6):
        l2, p2 = host.mnist_train(x, y, params, batch, steps, lr, reference_tape=32 + 64 + mode)
        assert np.array_equal(l2, losses) and all(np.array_equal(a, b) for a, b in zip(p2, P)), mode
    l3, p3 = host.mnist_train(x, y, params, batch, steps, lr, reference_tape=32 + 64 + 12)
    assert all(np.abs(a - b).max() <= tol for a, b in zip(p3, P))
    # each of the two by itself
    l4, _ = host.mnist_train(x, y, params, batch, steps, lr, reference_tape=32)
    assert l4[0] == losses[0]
    l5, p5 = host.mnist_train(x, y, params, batch, steps, lr, reference_tape=64)
    plain, pp = host.mnist_train(x, y, params, batch, steps, lr, reference_tape=0)
    assert l5[0] == plain[0] and not np.array_equal(p5[0], pp[0])


def test_the_demo_runs_with_both(host, tmp_path):
    print("case demo with norm and muon", flush=True)
    write_mnist_dir(str(tmp_path))
    rc, losses, acc, _ = host.mnist_demo(str(tmp_path), epochs=2, lr=1e-3, reference_tape=32 + 64 + 4)
    rc2, losses2, acc2, _ = host.mnist_demo(str(tmp_path), epochs=2, lr=1e-3, reference_tape=32 + 64 + 4 + 2)
    assert rc == rc2 == 8 and np.isfinite(losses).all() and np.array_equal(acc, acc2) and np.allclose(losses, losses2, rtol=1e-6, atol=0)
