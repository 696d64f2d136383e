"""CPU side of the group normalisation: the 64-bit formulas against differences, and the calls that the C ABI
refuses before it launches anything."""
import ctypes as C

import numpy as np
import pytest

import norm_oracle as O


@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("shape", [(3, 1, 8, 2), (2, 5, 9, 3), (1, 7, 4, 1)], ids=str)
def test_oracle_gradient_is_the_derivative_of_the_oracle(shape, act):
    n, p, c, groups = shape
    r = np.random.default_rng(3)
    x, w, b, g = r.standard_normal((n, p, c)), r.uniform(0.5, 1.5, c), r.standard_normal(c), r.standard_normal((n, p, c))
    _, st, _, _ = O.forward(x, w, b, groups, act, 1e-5)
    grads, _ = O.backward(x, w, b, st, groups, act, g)
    for k in range(3):
        args = [x, w, b]
        flat = grads[k].reshape(-1)
        for i in r.choice(flat.size, min(flat.size, 12), replace=False):
            loss = []
            for h in (1e-6, -1e-6):
                v = args[k].copy()
                v.reshape(-1)[i] += h
                a = list(args)
                a[k] = v
                loss.append(float((O.forward(*a, groups, act, 1e-5)[0] * g).sum()))
            assert abs((loss[0] - loss[1]) / 2e-6 - flat[i]) <= 1e-6 * max(1.0, abs(flat[i])) + 2e-7


def _lib():
    from ctorch_amd import capi
    return capi.load()


def test_refused_forward_calls():
    lib, p = _lib(), C.c_void_p(64)
    def call(x=p, eps=1e-5, act=0, y=p, n=2, s=3, c=8, g=2):
        return lib.ctamd_group_norm_f32(x, None, None, C.c_float(eps), act, y, None, n, s, c, g, None)
    assert call(g=0) == -1 and call(g=3) == -1 and call(g=16) == -1
    assert b"divide" in lib.ctamd_last_error()
    assert call(act=3) == -1 and call(act=-1) == -1
    assert call(x=None) == -1 and call(y=None) == -1
    assert call(eps=-1.0) == -1 and call(eps=float("nan")) == -1
    assert call(c=(1 << 20) + 2) == -5 and call(s=1 << 60) == -5 and call(n=1 << 60) == -5 and call(n=(1 << 64) - 1, s=(1 << 64) - 1) == -5
    for empty in ({"n": 0}, {"s": 0}, {"c": 0}):
        assert call(**empty) == 0 and call(x=None, y=None, **empty) == 0


def test_refused_backward_calls():
    lib, p = _lib(), C.c_void_p(64)
    def call(x=p, st=p, act=0, go=p, dx=p, n=2, s=3, c=8, g=2):
        return lib.ctamd_group_norm_backward_f32(x, None, None, st, act, go, dx, None, None, n, s, c, g, None)
    assert call(g=0) == -1 and call(g=3) == -1 and call(act=7) == -1
    assert call(x=None) == -1 and call(st=None) == -1 and call(go=None) == -1
    assert call(c=(1 << 20) + 2) == -5 and call(n=1 << 60) == -5
    assert call(dx=None) == 0                     # nothing wanted
    assert call(n=0) == 0 and call(s=0) == 0 and call(c=0) == 0
