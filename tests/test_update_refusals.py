"""CPU side of the orthogonalised updates: the calls that the C ABI refuses before it launches anything."""
import ctypes as C


def _lib():
    from ctorch_amd import capi
    return capi, capi.load()


def test_refused_newton_schulz_calls():
    _, lib = _lib()
    size, p = C.c_size_t(77), C.c_void_p(4096)
    assert lib.ctamd_newton_schulz_workspace(10, 20, 1, None) == -1
    assert lib.ctamd_newton_schulz_workspace(-1, 20, 1, C.byref(size)) == -1 and size.value == 0
    assert lib.ctamd_newton_schulz_workspace(10, 20, -1, C.byref(size)) == -1
    assert lib.ctamd_newton_schulz_workspace((1 << 20) + 1, 1, 1, C.byref(size)) == -5
    assert lib.ctamd_newton_schulz_workspace(1 << 16, 1 << 16, 1, C.byref(size)) == -5
    for empty in ((0, 5, 1), (5, 0, 1), (5, 5, 0)):
        assert lib.ctamd_newton_schulz_workspace(*empty, C.byref(size)) == 0 and size.value == 0
    assert lib.ctamd_newton_schulz_workspace(100, 70, 3, C.byref(size)) == 0
    need = size.value
    assert need >= 3 * 4 * 100 * 70 * 4

    def call(g=p, out=p, rows=100, cols=70, batch=3, steps=5, c=None, eps=1e-7, work=p, nbytes=need):
        c = None if c is None else (C.c_float * 3)(*c)
        return lib.ctamd_newton_schulz_f32(g, out, rows, cols, batch, steps, c, C.c_float(eps), work, nbytes, None)
    assert call(g=None) == -1 and call(out=None) == -1 and call(work=None) == -1
    assert call(nbytes=need - 1) == -1 and b"workspace" in lib.ctamd_last_error()
    assert call(work=C.c_void_p(4096 + 8)) == -1
    assert call(steps=-1) == -1 and call(steps=65) == -1
    assert call(c=(33.0, 0, 0)) == -1 and call(c=(1.0, float("nan"), 0)) == -1 and call(c=(1.0, 0, float("inf"))) == -1
    assert call(eps=-1.0) == -1 and call(eps=float("nan")) == -1
    assert call(rows=-4) == -1 and call(batch=-1) == -1 and call(rows=1 << 21) == -5
    assert call(batch=0) == 0 and call(rows=0, g=None, out=None, work=None) == 0
    # a batch of any length needs a bounded workspace
    assert lib.ctamd_newton_schulz_workspace(10, 256, 1 << 40, C.byref(size)) == 0 and size.value <= (2 << 30)


def test_refused_muon_calls():
    capi, lib = _lib()
    p, size = 4096, C.c_size_t(5)
    def table(**kw):
        f = dict(param=p, grad=p, momentum=p, new_param=p, new_momentum=p, rows=8, cols=9, scale=1.0)
        f.update(kw)
        return (capi.MuonMatrix * 1)(capi.MuonMatrix(**f))
    def options(**kw):
        f = dict(learning_rate=0.1, momentum=0.9, weight_decay=0.0, eps=1e-7, nesterov=1, steps=5, coefficients=(3.0, -4.0, 2.0))
        f.update(kw)
        return capi.MuonOptions(*[(C.c_float * 3)(*v) if k == "coefficients" else v for k, v in f.items()])
    assert lib.ctamd_muon_workspace(table(), 1, None) == -1
    assert lib.ctamd_muon_workspace(table(), -1, C.byref(size)) == -1 and size.value == 0
    assert lib.ctamd_muon_workspace(None, 1, C.byref(size)) == -1
    assert lib.ctamd_muon_workspace(None, 0, C.byref(size)) == 0 and size.value == 0
    assert lib.ctamd_muon_workspace(table(rows=1 << 22), 1, C.byref(size)) == -5
    assert lib.ctamd_muon_workspace(table(), 1, C.byref(size)) == 0
    need = size.value

    def call(t=None, count=1, o=None, work=C.c_void_p(4096), nbytes=need):
        return lib.ctamd_muon_step_f32(t if t is not None else table(), count, C.byref(o if o is not None else options()), work, nbytes, None)
    for name in ("param", "grad", "momentum", "new_param", "new_momentum"):
        assert call(table(**{name: None})) == -1
    assert call(table(rows=-1)) == -1 and call(table(cols=1 << 21)) == -5
    assert call(work=None) == -1 and call(nbytes=need - 1) == -1 and call(work=C.c_void_p(4104)) == -1
    assert call(o=options(steps=65)) == -1 and call(o=options(eps=-1.0)) == -1 and call(o=options(coefficients=(40.0, 0.0, 0.0))) == -1
    assert lib.ctamd_muon_step_f32(table(), 1, None, None, 0, None) == -1
    assert call(count=0, work=None, nbytes=0) == 0 and call(table(rows=0, param=None), work=None, nbytes=0) == 0


def test_a_written_tensor_may_not_overlap_another():
    """The matrices of a call run side by side: a matrix given twice, or tensors that share memory, are refused."""
    capi, lib = _lib()
    opt = capi.MuonOptions(0.1, 0.9, 0.0, 1e-7, 1, 5, (C.c_float * 3)(3.0, -4.0, 2.0))
    nbytes = 8 * 9 * 4
    work = 1 << 20

    def call(*mats):
        table = (capi.MuonMatrix * len(mats))(*[capi.MuonMatrix(*m, 8, 9, 1.0) for m in mats])
        size = C.c_size_t()
        assert lib.ctamd_muon_workspace(table, len(mats), C.byref(size)) == 0
        rc = lib.ctamd_muon_step_f32(table, len(mats), C.byref(opt), C.c_void_p(work), size.value, None)
        return rc == -1 and b"overlaps" in lib.ctamd_last_error()
    at = [4096 + 1024 * k for k in range(12)]
    one = (at[0], at[1], at[2], at[0], at[2])
    assert call(one, one)                                                             # twice the same
    assert call(one, (at[3], at[4], at[5], at[0], at[6]))                             # two results in one place
    assert call(one, (at[3], at[4], at[5], at[6], at[2]))
    assert call(one, (at[3], at[0], at[5], at[6], at[7]))                             # another's gradient is written
    assert call((at[0], at[1], at[2], at[1], at[3]))                                  # its own gradient
    assert call((at[0], at[1], at[2], at[3], at[3]))
    assert call((at[0], at[1], at[2], at[0] + 4, at[3]))                              # in place, but for one element
    assert call((at[0], at[1], at[2], at[0] + nbytes - 4, at[3]))
