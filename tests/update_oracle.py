"""Newton-Schulz products and the optimiser step around them in 64 bits, and how far from them a kernel may be
that multiplies pairs of 11-bit numbers with fp32 sums.

Let a be the first coefficient (the slope of the step's polynomial at zero, its largest), X_k the iterate after
k steps, |X_0|_F = 1.  An error E of X_k grows to at most a^(s - k) E in X_s.  One step adds to X_k, in the Frobenius
norm and relative to |X_(k-1)|_F, at most: 2^-22 for every number kept as a pair (X, A, B, each met in a
product twice over) and for the product of the two low halves that is left out, times the sums of the
step's factors (a, b, 2c, ... about 16 in all), and for sums of K terms in fp32 about sqrt(K) 2^-24, twice over;
|X_k|_F is at most a^k and at most 1.3 sqrt(m)."""
import numpy as np

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def newton_schulz(g, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    a, b, c = (float(np.float32(v)) for v in coefficients)
    x = g.astype(np.float64)
    tall = x.shape[0] > x.shape[1]
    x = x / (np.sqrt(np.square(x).sum()) + float(np.float32(eps)))
    if tall:
        x = x.T
    for _ in range(steps):
        gram = x @ x.T
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.T if tall else x


def newton_schulz_bound(shape, steps, a=COEFFICIENTS[0]):
    """of the Frobenius norm of the error"""
    m, n = min(shape), max(shape)
    bound = a ** steps * 2.0 ** -22
    for k in range(1, steps + 1):
        bound += a ** (steps - k) * (16 + 0.5 * np.sqrt(n)) * 2.0 ** -22 * min(a ** (k - 1), 1.3 * np.sqrt(m))
    return bound


def muon(param, grad, momentum, scale, lr, mu, decay, nesterov, steps, eps=1e-7, coefficients=COEFFICIENTS):
    """new parameter, new momentum and the bounds of both, element by element"""
    f = lambda v: float(np.float32(v))  # noqa: E731
    p, g, mo = (v.astype(np.float64) for v in (param, grad, momentum))
    lr, mu, decay, scale = f(lr), f(mu), f(decay), f(scale)
    m = mu * mo + g
    u = g + mu * m if nesterov else m
    o = newton_schulz(u, steps, coefficients, eps)
    new = p * (1 - lr * decay) - lr * scale * o
    m_err = 2.0 ** -23 * (np.abs(mu * mo) + np.abs(m))
    # the update's own roundings (3 of 2^-24 an element, relative) reach X_0 and grow as any error of it
    o_err = newton_schulz_bound(param.shape, steps, coefficients[0]) + coefficients[0] ** steps * 2.0 ** -21
    new_err = lr * scale * o_err + 2.0 ** -22 * (np.abs(p) + np.abs(lr * scale * o))
    return new, m, new_err, m_err
