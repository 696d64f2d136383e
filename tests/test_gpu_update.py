"""Orthogonalised updates through the C ABI: ctamd_newton_schulz_f32 and ctamd_muon_step_f32 against the iteration
in 64 bits, with the bounds of tests/update_oracle.py."""
import ctypes as C

import numpy as np
import pytest

import update_oracle as O

pytestmark = pytest.mark.gpu


def _gradient(rows, cols, seed, batch=None):
    r = np.random.default_rng(seed)
    rank = max(1, min(rows, cols) // 4)
    lead = () if batch is None else (batch,)
    g = r.standard_normal((*lead, rows, rank)) @ r.standard_normal((*lead, rank, cols)) / np.sqrt(rank)
    return ((g + 0.5 * r.standard_normal((*lead, rows, cols))) * 1e-3).astype(np.float32)


def _workspace(G, nbytes):
    """filled with NaN patterns: nothing may be read that the call has not written"""
    import torch
    return torch.full((max(1, (nbytes + 3) // 4),), -1, dtype=torch.int32, device=G.DEV)


def _ns(G, g, steps=5, coefficients=None, eps=1e-7, out=None, work=None, stream=None):
    import torch
    lib = G.lib()
    batch, rows, cols = g.shape if g.dim() == 3 else (1, *g.shape)
    size = C.c_size_t()
    assert lib.ctamd_newton_schulz_workspace(rows, cols, batch, C.byref(size)) == 0
    work = _workspace(G, size.value) if work is None else work
    out = torch.full_like(g, float("nan")) if out is None else out
    c = None if coefficients is None else (C.c_float * 3)(*coefficients)
    G.call("ctamd_newton_schulz_f32", G.ptr(g), G.ptr(out), rows, cols, batch, steps, c, C.c_float(eps), G.ptr(work), size.value,
           stream or G.stream())
    return out


def _check(got, g, steps=5, coefficients=O.COEFFICIENTS, eps=1e-7):
    got = got.detach().cpu().numpy().astype(np.float64)
    want = O.newton_schulz(g, steps, coefficients, eps)
    err = float(np.linalg.norm(got - want))
    bound = O.newton_schulz_bound(g.shape, steps, max(coefficients[0], 1.0))
    assert err <= bound, (g.shape, steps, err, bound, float(np.linalg.norm(want)))
    return err


# one entry; vectors; below, at and beyond a tile of 64, 128, 256; odd; long
SHAPES = [(1, 1), (1, 7), (9, 1), (2, 3), (10, 256), (256, 10), (31, 33), (63, 64), (64, 64), (65, 64), (64, 1000), (128, 784), (129, 257), (200, 200),
          (333, 1000), (1000, 333), (256, 256), (257, 300), (70, 5001), (1, 70000), (20000, 3), (1030, 1040)]


@pytest.mark.parametrize("steps", [0, 1, 2, 5])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%d" % s)
def test_against_64_bits(shape, steps):
    import gpu_support as G
    g = _gradient(*shape, seed=shape[0] + 3 * shape[1])
    _check(_ns(G, G.dev(g), steps), g, steps)


@pytest.mark.parametrize("shape", [(2048, 2048), (4096, 2050), (3000, 4100)], ids=lambda s: "%dx%d" % s)
def test_large_matrices(shape):
    """The 64-bit iteration by torch on the device (products in double)."""
    import gpu_support as G
    import torch
    gen = torch.Generator(device=G.DEV)
    gen.manual_seed(5)
    g = torch.randn(*shape, device=G.DEV, generator=gen)
    got = _ns(G, g).double()
    x = g.double()
    x = x / (x.norm() + 1e-7)
    if shape[0] > shape[1]:
        x = x.T.contiguous()
    a, b, c = (float(np.float32(v)) for v in O.COEFFICIENTS)
    for _ in range(5):
        gram = x @ x.T.contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    want = x.T if shape[0] > shape[1] else x
    assert float((got - want).norm()) <= O.newton_schulz_bound(shape, 5)
    # 5 steps make the singular values of such a matrix 0.68 ... 1.21
    assert 0.6 * np.sqrt(min(shape)) < float(got.norm()) < 1.25 * np.sqrt(min(shape))


# the sums of X X^T in parts, joined by the block that is last: few rows, long columns, ragged ends
LONG = [(128, 20000), (100, 9001), (20001, 130), (256, 16390), (66, 70001), (512, 8200), (64, 9001), (64, 60001), (30, 60000)]


@pytest.mark.parametrize("shape", LONG, ids=lambda s: "%dx%d" % s)
def test_few_long_rows(shape):
    import gpu_support as G
    import torch
    g = _gradient(*shape, seed=7)
    got = _ns(G, G.dev(g))
    _check(got, g)
    assert torch.equal(_ns(G, G.dev(g)), got)                                          # parts are added in their order


def test_few_long_rows_in_a_batch_on_two_streams_and_replayed():
    """A workspace's counters are back at zero after every product: a second call, a recorded one replayed, and a
    call at the same time in a workspace of its own give the first one's bits."""
    import gpu_support as G
    import torch
    lib = G.lib()
    g = _gradient(130, 9000, seed=3, batch=3)
    x = G.dev(g)
    size = C.c_size_t()
    assert lib.ctamd_newton_schulz_workspace(130, 9000, 3, C.byref(size)) == 0
    work = [_workspace(G, size.value) for _ in range(2)]
    want = _ns(G, x, work=work[0])
    for i in range(3):
        _check(want[i], g[i])
    streams = [C.c_void_p(), C.c_void_p()]
    for s in streams:
        assert lib.ctamd_stream_create(C.byref(s)) == 0
    out = [torch.empty_like(x) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for o, w, s in zip(out, work, streams):
            _ns(G, x, out=o, work=w, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(out[0], want) and torch.equal(out[1], want)
    graph = C.c_void_p()
    replayed = torch.empty_like(x)
    torch.cuda.synchronize()
    assert lib.ctamd_graph_begin(streams[0]) == 0
    _ns(G, x, out=replayed, work=work[0], stream=streams[0])
    assert lib.ctamd_graph_end(streams[0], C.byref(graph)) == 0
    for _ in range(3):
        replayed.zero_()
        torch.cuda.synchronize()
        assert lib.ctamd_graph_launch(graph, streams[0]) == 0
        _ns(G, x, out=out[1], work=work[1])                                            # the program's own, at the same time
        torch.cuda.synchronize()
        assert torch.equal(replayed, want) and torch.equal(out[1], want)
    assert lib.ctamd_graph_destroy(graph) == 0
    for s in streams:
        assert lib.ctamd_stream_destroy(s) == 0


def test_a_step_over_few_long_rows():
    import gpu_support as G
    import torch
    r = np.random.default_rng(2)
    shapes = [(96, 12000), (12001, 100), (128, 64)]
    host = [((r.standard_normal(s) / 10).astype(np.float32), _gradient(*s, 20 + k), 5 * _gradient(*s, 40 + k), float(0.2 * np.sqrt(max(s))))
            for k, s in enumerate(shapes)]
    dev = [tuple(G.dev(v) for v in h[:3]) for h in host]
    out = [(torch.full_like(p, float("nan")), torch.full_like(p, float("nan"))) for p, _, _ in dev]
    _muon(G, [(*d, *o, h[3]) for d, o, h in zip(dev, out, host)], _options())
    for (p, g, m, scale), (new, new_m) in zip(host, out):
        want, wm, err, merr = O.muon(p, g, m, scale, 0.02, 0.95, 0.01, True, 5)
        assert np.all(np.abs(new_m.cpu().numpy() - wm) <= merr)
        assert np.all(np.abs(new.cpu().numpy() - want) <= err), p.shape
    _muon(G, [(d[0], d[1], d[2], d[0], d[2], h[3]) for d, h in zip(dev, host)], _options())
    for (p, _, m), (new, new_m) in zip(dev, out):
        assert torch.equal(p, new) and torch.equal(m, new_m)


def test_singular_values_are_driven_towards_one():
    import gpu_support as G
    r = np.random.default_rng(1)
    u, v = np.linalg.qr(r.standard_normal((96, 96)))[0], np.linalg.qr(r.standard_normal((150, 96)))[0]
    g = ((u * np.geomspace(1, 0.05, 96)) @ v.T).astype(np.float32)
    s = np.linalg.svd(_ns(G, G.dev(g)).cpu().numpy().astype(np.float64), compute_uv=False)
    assert 0.65 < s.min() and s.max() < 1.25


@pytest.mark.parametrize("scale", [1e-30, 1e-18, 1e18, 1e36])
def test_scales_whose_squares_leave_the_range_of_a_float(scale):
    import gpu_support as G
    g = (_gradient(40, 90, 3) * 1e3 * scale).astype(np.float32)
    _check(_ns(G, G.dev(g), eps=0.0), g, eps=0.0)


def test_zero_infinite_and_undefined_updates():
    import gpu_support as G
    import torch
    assert float(_ns(G, torch.zeros(70, 30, device=G.DEV)).abs().max()) == 0
    for bad in (float("nan"), float("inf")):
        g = torch.randn(2, 70, 130, device=G.DEV)
        g[0, 3, 5] = bad
        out = _ns(G, g)
        # the norm is no number (or infinite): neither is the whole matrix - but not its neighbour in the batch
        assert bool(torch.isnan(out[0]).all()) and bool(torch.isfinite(out[1]).all())


def test_other_coefficients_and_steps():
    import gpu_support as G
    g = _gradient(80, 120, 8)
    cubic = (1.5, -0.5, 0.0)
    _check(_ns(G, G.dev(g), 12, cubic), g, 12, cubic)
    _check(_ns(G, G.dev(g), 1, (8.0, -23.0, 17.0)), g, 1, (8.0, -23.0, 17.0))
    _check(_ns(G, G.dev(g), 3, (1.0, 0.0, 0.0)), g, 3, (1.0, 0.0, 0.0))      # X itself, three times rounded


@pytest.mark.parametrize("batch,shape", [(7, (33, 65)), (3, (300, 130)), (40, (10, 12)), (2, (513, 512))], ids=str)
def test_a_batch_is_its_matrices(batch, shape):
    """Every matrix of a batch against 64 bits; the same bits again, and in place."""
    import gpu_support as G
    import torch
    g = _gradient(*shape, seed=4, batch=batch)
    got = _ns(G, G.dev(g))
    for i in range(batch):
        _check(got[i], g[i])
    assert torch.equal(_ns(G, G.dev(g)), got)
    inplace = G.dev(g)
    assert torch.equal(_ns(G, inplace, out=inplace), got)


@pytest.mark.parametrize("shift", [1, 2, 3])
def test_tensors_off_a_16_byte_boundary(shift):
    import gpu_support as G
    import torch
    g = _gradient(77, 140, 2)
    t = torch.full((77 * 140 + 24,), 7.5, device=G.DEV)
    src = torch.empty(77 * 140 + 8, device=G.DEV)[shift:shift + 77 * 140].view(77, 140)
    src.copy_(G.dev(g))
    out = t[8 + shift:8 + shift + 77 * 140].view(77, 140)
    _check(_ns(G, src, out=out), g)
    assert bool((t[:8 + shift] == 7.5).all()) and bool((t[8 + shift + 77 * 140:] == 7.5).all())


def _muon(G, mats, options, work=None, stream=None):
    """mats: (param, grad, momentum, new_param, new_momentum, scale) of tensors"""
    from ctorch_amd import capi
    lib = G.lib()
    table = (capi.MuonMatrix * max(1, len(mats)))(*[capi.MuonMatrix(*(t.data_ptr() for t in m[:5]), m[0].shape[0], m[0].shape[1], m[5]) for m in mats])
    size = C.c_size_t()
    assert lib.ctamd_muon_workspace(table, len(mats), C.byref(size)) == 0
    work = _workspace(G, size.value) if work is None else work
    rc = lib.ctamd_muon_step_f32(table, len(mats), C.byref(options), G.ptr(work), size.value, stream or G.stream())
    assert rc == 0, lib.ctamd_last_error()


def _options(lr=0.02, mu=0.95, decay=0.01, nesterov=True, steps=5, eps=1e-7):
    from ctorch_amd import capi
    return capi.MuonOptions(lr, mu, decay, eps, int(nesterov), steps, O.COEFFICIENTS)


@pytest.mark.parametrize("nesterov", [False, True])
@pytest.mark.parametrize("steps", [0, 1, 5])
@pytest.mark.parametrize("shapes", [[(784, 256), (256, 10)], [(128, 64)], [(5, 5), (64, 0), (300, 1000), (1000, 300), (1, 9)],
                                    [(8 + 7 * i, 300 - 11 * i) for i in range(21)]], ids=["mlp", "one", "mixed", "21"])
def test_steps_against_64_bits(shapes, steps, nesterov):
    import gpu_support as G
    import torch
    r = np.random.default_rng(9)
    host = []
    for k, (rows, cols) in enumerate(shapes):
        p = (r.standard_normal((rows, cols)) / np.sqrt(max(rows, 1))).astype(np.float32)
        g = _gradient(rows, cols, k) if rows and cols else np.zeros((rows, cols), np.float32)
        host.append((p, g, (5 * _gradient(rows, cols, 100 + k)) if rows and cols else g, float(0.2 * np.sqrt(max(rows, cols)))))
    dev = [tuple(G.dev(v) for v in h[:3]) for h in host]
    out = [(torch.full_like(p, float("nan")), torch.full_like(p, float("nan"))) for p, _, _ in dev]
    _muon(G, [(*d, *o, h[3]) for d, o, h in zip(dev, out, host)], _options(nesterov=nesterov, steps=steps))
    for (p, g, m, scale), (np_, nm) in zip(host, out):
        if p.size == 0:
            continue
        want, wm, err, merr = O.muon(p, g, m, scale, 0.02, 0.95, 0.01, nesterov, steps)
        got, gm = np_.cpu().numpy().astype(np.float64), nm.cpu().numpy().astype(np.float64)
        assert np.all(np.abs(gm - wm) <= merr), p.shape
        assert np.all(np.abs(got - want) <= err), (p.shape, float(np.max(np.abs(got - want) / err)))
    # in place: the same bits
    _muon(G, [(d[0], d[1], d[2], d[0], d[2], h[3]) for d, h in zip(dev, host)], _options(nesterov=nesterov, steps=steps))
    for (p, _, m), (np_, nm) in zip(dev, out):
        assert torch.equal(p, np_) and torch.equal(m, nm)


@pytest.mark.parametrize("shapes", [[(1500, 1533)], [(2048, 2100), (4100, 1001), (784, 2048)], [(4096, 4160)], [(3500, 2050), (1000, 3490)]], ids=str)
def test_large_steps(shapes):
    """Every size of tile with a parameter to update, ragged at its edges; the 64-bit iteration by torch on the
    device.  Bounds as tests/update_oracle.py's, of the Frobenius norm."""
    import gpu_support as G
    import torch
    gen = torch.Generator(device=G.DEV)
    gen.manual_seed(11)
    lr, mu, decay, band = 0.02, 0.95, 0.01, 64
    host = []
    for rows, cols in shapes:
        p, g, m = (torch.randn(rows, cols, device=G.DEV, generator=gen) * s for s in (1 / np.sqrt(rows), 1e-3, 5e-3))
        guarded = [torch.full((rows * cols + 2 * band,), 7.5, device=G.DEV) for _ in range(2)]
        out = [t[band:band + rows * cols].view(rows, cols) for t in guarded]
        host.append((p, g, m, out, guarded, float(0.2 * np.sqrt(max(rows, cols)))))
    _muon(G, [(p, g, m, *out, scale) for p, g, m, out, _, scale in host], _options(lr, mu, decay))
    f = lambda v: float(np.float32(v))  # noqa: E731
    a, b, c = (f(v) for v in O.COEFFICIENTS)
    for p, g, m, (new, new_m), guarded, scale in host:
        want_m = f(mu) * m.double() + g.double()
        assert bool(((new_m.double() - want_m).abs() <= 2.0 ** -23 * ((f(mu) * m.double()).abs() + want_m.abs())).all())
        x = g.double() + f(mu) * want_m
        x = x / (x.norm() + f(1e-7))
        tall = x.shape[0] > x.shape[1]
        x = x.T.contiguous() if tall else x
        for _ in range(5):
            gram = x @ x.T.contiguous()
            x = a * x + (b * gram + c * (gram @ gram)) @ x
        o = x.T if tall else x
        step = f(lr) * f(scale)
        want = p.double() * (1 - f(lr) * f(decay)) - step * o
        bound = step * (O.newton_schulz_bound(p.shape, 5) + a ** 5 * 2.0 ** -21) + 2.0 ** -22 * float((p.double().abs() + step * o.abs()).norm())
        assert float((new.double() - want).norm()) <= bound, (tuple(p.shape), float((new.double() - want).norm()), bound)
        assert all(bool((t[:band] == 7.5).all()) and bool((t[-band:] == 7.5).all()) for t in guarded)
    # in place: the same bits
    _muon(G, [(p, g, m, p, m, scale) for p, g, m, _, _, scale in host], _options(lr, mu, decay))
    for p, _, m, (new, new_m), _, _ in host:
        assert torch.equal(p, new) and torch.equal(m, new_m)


def test_streams_replays_and_two_graphs():
    import gpu_support as G
    import torch
    lib = G.lib()
    shapes = [(784, 256), (256, 10), (130, 70)]
    def fresh():
        return [tuple(G.dev(_gradient(r, c, s + k)) for s in (1, 50, 90)) for k, (r, c) in enumerate(shapes)]
    opt = _options()
    want = fresh()
    for _ in range(3):
        _muon(G, [(p, g, m, p, m, 1.0) for p, g, m in want], opt)
    side = torch.cuda.Stream()
    got = fresh()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            _muon(G, [(p, g, m, p, m, 1.0) for p, g, m in got], opt)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
    # a step recorded once and replayed three times, the program's own eager work in between; two graphs whose
    # replays follow each other on one stream may share a workspace
    from ctorch_amd import capi
    stream = C.c_void_p()
    assert lib.ctamd_stream_create(C.byref(stream)) == 0
    sets, graphs = [fresh(), fresh()], []
    size = C.c_size_t()
    table = (capi.MuonMatrix * 3)(*[capi.MuonMatrix(p.data_ptr(), g.data_ptr(), m.data_ptr(), p.data_ptr(), m.data_ptr(), *p.shape, 1.0)
                                    for p, g, m in sets[0]])
    assert lib.ctamd_muon_workspace(table, 3, C.byref(size)) == 0
    work = _workspace(G, size.value)
    torch.cuda.synchronize()
    for s in sets:
        graph = C.c_void_p()
        assert lib.ctamd_graph_begin(stream) == 0
        _muon(G, [(p, g, m, p, m, 1.0) for p, g, m in s], opt, work, stream)
        assert lib.ctamd_graph_end(stream, C.byref(graph)) == 0
        graphs.append(graph)
    eager = fresh()
    for _ in range(3):
        for graph in graphs:
            assert lib.ctamd_graph_launch(graph, stream) == 0
        _muon(G, [(p, g, m, p, m, 1.0) for p, g, m in eager], opt)
        torch.cuda.synchronize()
    for s in (*sets, eager):
        for a, b in zip(want, s):
            assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
    for graph in graphs:
        assert lib.ctamd_graph_destroy(graph) == 0
    assert lib.ctamd_stream_destroy(stream) == 0
