"""Group normalisation with an activation (ctamd_group_norm_f32) and its gradient through the C ABI, against
the formulas in 64 bits with bounds counted in roundings (tests/norm_oracle.py)."""
import ctypes as C

import numpy as np
import pytest

import norm_oracle as O

pytestmark = pytest.mark.gpu


def _run_forward(G, x, w, b, groups, act, eps=1e-5, stats=True, y=None):
    import torch
    n, p, c = x.shape
    y = torch.empty_like(x) if y is None else y
    st = torch.full((n, groups, 2), float("nan"), device=G.DEV) if stats else None
    G.call("ctamd_group_norm_f32", G.ptr(x), G.ptr(w), G.ptr(b), C.c_float(eps), O.ACTS[act], G.ptr(y), G.ptr(st), n, p, c, groups, G.stream())
    return y, st


def _run_backward(G, x, w, b, st, groups, act, g, want=(True, True, True), dx=None):
    import torch
    n, p, c = x.shape
    dx = (torch.full_like(x, float("nan")) if dx is None else dx) if want[0] else None
    dw = torch.full((c,), float("nan"), device=G.DEV) if want[1] else None
    db = torch.full((c,), float("nan"), device=G.DEV) if want[2] else None
    G.call("ctamd_group_norm_backward_f32", G.ptr(x), G.ptr(w), G.ptr(b), G.ptr(st), O.ACTS[act], G.ptr(g), G.ptr(dx), G.ptr(dw), G.ptr(db),
           n, p, c, groups, G.stream())
    return dx, dw, db


def _inputs(n, p, c, seed, mean=0.3):
    r = np.random.default_rng(seed)
    x = (r.standard_normal((n, p, c)) * r.uniform(0.3, 2.0, (n, 1, 1)) + mean).astype(np.float32)
    return (x, r.uniform(0.5, 1.5, c).astype(np.float32), (0.5 * r.standard_normal(c)).astype(np.float32),
            r.standard_normal((n, p, c)).astype(np.float32))


def _near(got, want, err, what):
    got = got.detach().cpu().numpy().astype(np.float64).reshape(want.shape)
    bad = ~(np.abs(got - want) <= err)
    assert not bad.any(), (what, int(bad.sum()), float(np.max(np.abs(got - want)[bad])), float(np.max(err[bad])), np.argwhere(bad)[:4].tolist())


# n, positions, channels, groups: a layer's activations (one position), maps that stay in a block's registers,
# and maps that are split; widths that take vectors of 4, 2 and 1; groups wider than a block
SHAPES = [
    (1, 1, 1, 1), (3, 1, 4, 4), (5, 1, 6, 2), (256, 1, 256, 8), (7, 1, 330, 11), (2, 1, 4096, 1), (9, 1, 1021, 1), (3, 1, 514, 1), (33, 1, 2048, 1),
    (300, 1, 96, 96), (2, 1, 9001, 1), (1, 1, 40000, 2), (4, 1, 8224, 1), (70, 1, 12, 3),
    (2, 2, 3, 1), (3, 5, 8, 2), (4, 49, 64, 8), (2, 64, 512, 32), (1, 100, 30, 10), (3, 17, 1024, 4), (2, 256, 40, 5), (5, 333, 66, 11),
    (6, 3, 7, 7), (40, 8, 36, 3), (2, 1024, 32, 1), (2, 900, 16, 4),
    (1, 5000, 64, 8), (2, 4096, 128, 32), (3, 3001, 30, 3), (1, 2, 3000, 2), (2, 7, 5000, 1), (1, 40001, 4, 1), (2, 10007, 1, 1), (1, 3000, 770, 7),
    (65, 301, 256, 2),
]


@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_against_64_bits(shape, act):
    import gpu_support as G
    n, p, c, groups = shape
    x, w, b, g = _inputs(n, p, c, 7 + c + p)
    y, st = _run_forward(G, G.dev(x), G.dev(w), G.dev(b), groups, act)
    wy, wst, ey, est = O.forward(x, w, b, groups, act, 1e-5)
    _near(st, wst, est, "stats")
    _near(y, wy, ey, "y")
    stats = wst.astype(np.float32)
    got = _run_backward(G, G.dev(x), G.dev(w), G.dev(b), G.dev(stats), groups, act, G.dev(g))
    want, err = O.backward(x, w, b, stats, groups, act, g)
    for a, v, e, what in zip(got, want, err, ("dx", "dweight", "dbias")):
        _near(a, v, e, what)


@pytest.mark.parametrize("shape", [(6, 1, 64, 4), (3, 20, 32, 4), (2, 3000, 64, 4)], ids=str)
def test_without_weight_bias_or_statistics(shape):
    """NULL weight and bias are ones and zeros, bit for bit; the statistics are optional; each gradient is."""
    import gpu_support as G
    import torch
    n, p, c, groups = shape
    x, _, _, g = (G.dev(v) for v in _inputs(n, p, c, 3))
    one, zero = torch.ones(c, device=G.DEV), torch.zeros(c, device=G.DEV)
    y, st = _run_forward(G, x, one, zero, groups, "silu")
    y2, _ = _run_forward(G, x, None, None, groups, "silu", stats=False)
    assert torch.equal(y, y2)
    full = _run_backward(G, x, one, zero, st, groups, "silu", g)
    bare = _run_backward(G, x, None, None, st, groups, "silu", g)
    for a, b in zip(full, bare):
        assert torch.equal(a, b)
    for k in range(3):
        want = [k == j for j in range(3)]
        got = _run_backward(G, x, one, zero, st, groups, "silu", g, want)
        assert torch.equal(got[k], full[k])
    assert [v is None for v in _run_backward(G, x, one, zero, st, groups, "silu", g, (False, True, True))] == [True, False, False]


@pytest.mark.parametrize("shape", [(6, 1, 64, 4), (3, 20, 32, 4), (2, 3000, 64, 4)], ids=str)
@pytest.mark.parametrize("shift", [1, 2])
def test_tensors_off_a_16_byte_boundary_and_in_place(shape, shift):
    import gpu_support as G
    import torch
    n, p, c, groups = shape
    x, w, b, g = _inputs(n, p, c, 5)
    size = n * p * c
    def off(a):
        t = torch.empty(a.size + 8, device=G.DEV)
        v = t[shift:shift + a.size].view(*a.shape)
        v.copy_(G.dev(a))
        return v
    wy, wst, ey, est = O.forward(x, w, b, groups, "relu", 1e-5)
    xo = off(x)
    guard = torch.full((size + 16,), 7.5, device=G.DEV)
    y, st = _run_forward(G, xo, off(w), off(b), groups, "relu", y=guard[8 + shift:8 + shift + size].view(n, p, c))
    _near(y, wy, ey, "y")
    assert bool((guard[:8 + shift] == 7.5).all()) and bool((guard[8 + shift + size:] == 7.5).all())
    stats = wst.astype(np.float32)
    want, err = O.backward(x, w, b, stats, groups, "relu", g)
    go = off(g)
    got = _run_backward(G, xo, off(w), off(b), G.dev(stats), groups, "relu", go, dx=go)       # dx over g
    for a, v, e, what in zip(got, want, err, ("dx", "dweight", "dbias")):
        _near(a, v, e, what)
    y2, _ = _run_forward(G, xo, off(w), off(b), groups, "relu", y=xo)                        # y over x
    assert torch.equal(y2, y)


@pytest.mark.parametrize("shape", [(4, 1, 256, 2), (2, 60, 64, 2), (2, 5000, 64, 2)], ids=str)
def test_a_mean_far_from_zero_keeps_the_variance(shape):
    """x = 1000 + noise of 0.01 .. : a difference of sums of squares would lose all of the variance (1000^2 u = 0.06)."""
    import gpu_support as G
    n, p, c, groups = shape
    r = np.random.default_rng(2)
    x = (1000 + 0.05 * r.standard_normal((n, p, c))).astype(np.float32)
    one, zero = np.ones(c, np.float32), np.zeros(c, np.float32)
    _, st = _run_forward(G, G.dev(x), G.dev(one), G.dev(zero), groups, "none")
    _, want, _, _ = O.forward(x, one, zero, groups, "none", 1e-5)
    got = st.cpu().numpy().astype(np.float64)
    # deviations of 0.05 from a mean that 32 bits hold to 1000 u = 6e-5: they shift the variance by that squared,
    # and the sum of the deviations, which a mean in 64 bits would have zero, by nothing else
    assert np.all(np.abs(got[..., 1] / want[..., 1] - 1) <= 1e-3)
    assert np.all(np.abs(got[..., 0] - want[..., 0]) <= 1000 * 64 * O.U)


@pytest.mark.parametrize("shape", [(4, 1, 64, 4), (3, 24, 64, 4), (2, 4000, 64, 4)], ids=str)
def test_constant_groups_and_values_that_are_no_numbers(shape):
    import gpu_support as G
    import torch
    n, p, c, groups = shape
    x, w, b, g = _inputs(n, p, c, 9)
    x[0, :, :16] = 3.25                                  # variance 0: xhat is 0, y = act(bias)
    x[-1, -1, 20] = np.nan                               # group 1 of the last sample
    x[-1, 0, 40] = np.inf                                # group 2 of the last sample
    y, st = _run_forward(G, G.dev(x), G.dev(w), G.dev(b), groups, "none")
    y, st = y.cpu().numpy(), st.cpu().numpy()
    assert np.array_equal(y[0, :, :16], np.broadcast_to(b[:16], (p, 16)))
    assert st[0, 0, 0] == np.float32(3.25) and abs(st[0, 0, 1] / np.sqrt(1e5) - 1) < 1e-6
    assert np.isnan(y[-1, :, 16:48]).all()
    clean = np.ones_like(y, bool)
    clean[-1, :, 16:48] = False
    x2 = np.where(np.isfinite(x), x, 0).astype(np.float32)
    wy, _, ey, _ = O.forward(x2, w, b, groups, "none", 1e-5)
    assert np.all((np.abs(y - wy) <= ey)[clean])
    # a group that is not a number stays by itself in dx too
    stats = torch.from_numpy(st).to(G.DEV)
    dx, _, _ = _run_backward(G, G.dev(x), G.dev(w), G.dev(b), stats, groups, "none", G.dev(g))
    dx = dx.cpu().numpy()
    assert np.isfinite(dx[clean]).all() and np.isnan(dx[-1, :, 16:32]).all()


def test_groups_of_one_value_have_no_gradient():
    import gpu_support as G
    x, w, b, g = _inputs(50, 1, 24, 4)
    y, st = _run_forward(G, G.dev(x), G.dev(w), G.dev(b), 24, "none")
    assert np.array_equal(y.cpu().numpy(), np.broadcast_to(b, x.shape))
    dx, dw, db = _run_backward(G, G.dev(x), G.dev(w), G.dev(b), st, 24, "none", G.dev(g))
    assert float(dx.abs().max()) == 0 and float(dw.abs().max()) == 0
    assert np.allclose(db.cpu().numpy(), g.astype(np.float64).sum((0, 1)), rtol=0, atol=50 * 64 * O.U)


@pytest.mark.parametrize("shape", [(8, 1, 48, 3), (2, 12, 48, 3), (1, 2500, 24, 3)], ids=str)
@pytest.mark.parametrize("act", ["none", "silu"])
def test_gradient_against_differences(shape, act):
    """(L(v + h d) - L(v - h d)) / 2h for L = sum y g, by the kernel's own forward pass, against <gradient, d>."""
    import gpu_support as G
    n, p, c, groups = shape
    x, w, b, g = _inputs(n, p, c, 21)
    _, st = _run_forward(G, G.dev(x), G.dev(w), G.dev(b), groups, act)
    grads = [v.cpu().numpy().astype(np.float64) for v in _run_backward(G, G.dev(x), G.dev(w), G.dev(b), st, groups, act, G.dev(g))]
    r = np.random.default_rng(1)
    for k, (v, grad) in enumerate(zip((x, w, b), grads)):
        d = r.standard_normal(v.shape)
        h = 2.0 ** -6
        loss, noise = [], 0.0
        for sign in (1, -1):
            args = [x, w, b]
            args[k] = (v + sign * h * d).astype(np.float32)
            y, _ = _run_forward(G, *(G.dev(a) for a in args), groups, act)
            _, _, ey, _ = O.forward(*args, groups, act, 1e-5)
            loss.append(float((y.cpu().numpy().astype(np.float64) * g).sum()))
            noise += float(np.sqrt((ey ** 2 * g ** 2).sum()))
        # the third derivative's term, h^2 / 6 L''', is taken from the 64-bit formulas at twice the step
        exact = []
        for step in (h, 2 * h):
            pair = []
            for sign in (1, -1):
                args = [x, w, b]
                args[k] = v + sign * step * d
                pair.append(float((O.forward(*args, groups, act, 1e-5)[0] * g).sum()))
            exact.append((pair[0] - pair[1]) / (2 * step))
        curvature = abs(exact[1] - exact[0])                 # 3 h^2 / 6 L''' and above: more than the h^2 / 6 L''' at h
        got, want = (loss[0] - loss[1]) / (2 * h), float((grad * d).sum())
        assert abs(got - want) <= curvature + 4 * noise / (2 * h) + 1e-5 * float(np.abs(grad * d).sum()), (k, got, want, curvature, noise)


@pytest.mark.parametrize("shape", [(500, 1, 64, 4), (3, 100, 64, 4), (2, 6000, 64, 4)], ids=str)
def test_the_same_call_gives_the_same_bits_on_any_stream_and_in_a_replayed_graph(shape):
    import gpu_support as G
    import torch
    n, p, c, groups = shape
    lib = G.lib()
    x, w, b, g = (G.dev(v) for v in _inputs(n, p, c, 11))
    y, st = _run_forward(G, x, w, b, groups, "silu")
    ref = _run_backward(G, x, w, b, st, groups, "silu", g)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        y2, st2 = _run_forward(G, x, w, b, groups, "silu")
        got = _run_backward(G, x, w, b, st2, groups, "silu", g)
    # on this stream at the same time: the scratch is shared, the library orders the two
    y3, _ = _run_forward(G, x, w, b, groups, "silu")
    torch.cuda.synchronize()
    assert torch.equal(y, y2) and torch.equal(y, y3) and torch.equal(st, st2)
    for a, v in zip(ref, got):
        assert torch.equal(a, v)
    stream, graph = C.c_void_p(), C.c_void_p()
    assert lib.ctamd_stream_create(C.byref(stream)) == 0
    yg, sg = torch.zeros_like(y), torch.zeros_like(st)
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    torch.cuda.synchronize()
    assert lib.ctamd_graph_begin(stream) == 0
    assert lib.ctamd_group_norm_f32(G.ptr(x), G.ptr(w), G.ptr(b), C.c_float(1e-5), 2, G.ptr(yg), G.ptr(sg), n, p, c, groups, stream) == 0
    assert lib.ctamd_group_norm_backward_f32(G.ptr(x), G.ptr(w), G.ptr(b), G.ptr(sg), 2, G.ptr(g), G.ptr(dx), G.ptr(dw), G.ptr(db), n, p, c, groups,
                                             stream) == 0
    assert lib.ctamd_graph_end(stream, C.byref(graph)) == 0
    for turn in range(3):
        for t in (yg, sg, dx, dw, db):
            t.zero_()
        x.mul_(1.0 + 0.5 * turn)                            # the replay reads the data of now
        y, st = _run_forward(G, x, w, b, groups, "silu")
        ref = _run_backward(G, x, w, b, st, groups, "silu", g)
        torch.cuda.synchronize()
        assert lib.ctamd_graph_launch(graph, stream) == 0 and lib.ctamd_sync(stream) == 0
        assert torch.equal(yg, y) and torch.equal(sg, st)
        for a, v in zip(ref, (dx, dw, db)):
            assert torch.equal(a, v)
    assert lib.ctamd_graph_destroy(graph) == 0 and lib.ctamd_stream_destroy(stream) == 0


def test_offsets_past_32_bits():
    """2^32 + elements: the last sample lies behind a 32-bit element offset."""
    import gpu_support as G
    import torch
    n, p, c, groups = 17, 1 << 16, 4096, 8                 # 17 x 2^28 elements, 17 GiB
    x = torch.zeros(n, p, c, device=G.DEV)
    last, w, b, g = _inputs(1, p, 8, 6)
    tile = G.dev(last).repeat(1, 1, c // 8)
    x[-1] = tile[0]
    x[0, 0, 0] = 5.0
    wt, bt = G.dev(w).repeat(c // 8), G.dev(b).repeat(c // 8)
    y, st = _run_forward(G, x, wt, bt, groups, "relu")
    # every group of the last sample holds the same 8 channels over and over
    wy, wst, ey, est = O.forward(last, w, b, 1, "relu", 1e-5)
    _near(st[-1], np.broadcast_to(wst[0], (groups, 2)), np.broadcast_to(est[0], (groups, 2)), "stats")
    _near(y[-1, :, :8], wy[0], ey[0], "y")
    _near(y[-1, :, -8:], wy[0], ey[0], "y end")
    assert torch.equal(y[-2, -1], torch.relu(bt))
    dy = x                                                 # any values
    dx, dw, db = _run_backward(G, x, wt, bt, st, groups, "relu", dy)
    sub = last
    want, err = O.backward(sub, w, b, np.asarray(st[-1:, :1].cpu()), 1, "relu", last)
    _near(dx[-1, :, -8:], want[0][0], err[0][0], "dx")
