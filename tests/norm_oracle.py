"""Group normalisation with an activation and its gradient in 64 bits, from the formulas, and how far a
kernel that works in 32 bits may be from them.

The bounds count roundings of u = 2^-24.  A sum of the kernels is a tree whose longest path has at most
DEPTH additions (a thread's own values, then lanes, waves and parts), so its error is at most
DEPTH * u * sum |terms|."""
import numpy as np

U = 2.0 ** -24
DEPTH = 256
ACTS = {"none": 0, "relu": 1, "silu": 2}


def _per_group(v, groups):
    n, p, c = v.shape
    return v.reshape(n, p, groups, c // groups)


def _act(z, act):
    if act == "relu":
        return np.where(z > 0, z, 0.0)
    return z / (1 + np.exp(-z)) if act == "silu" else z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).astype(np.float64)
    if act == "silu":
        s = 1 / (1 + np.exp(-z))
        return s * (1 + z * (1 - s))
    return np.ones_like(z)


def forward(x, weight, bias, groups, act, eps):
    """y, stats [n, groups, 2] and the bounds of both, all 64-bit"""
    x, weight, bias = x.astype(np.float64), weight.astype(np.float64), bias.astype(np.float64)
    n, p, c = x.shape
    xg = _per_group(x, groups)
    mean = xg.mean((1, 3), keepdims=True)
    var = np.square(xg - mean).mean((1, 3), keepdims=True)
    rstd = 1 / np.sqrt(var + eps)
    xhat = ((xg - mean) * rstd).reshape(n, p, c)
    z = xhat * weight + bias
    # the mean is a tree sum; the deviations are taken from means inside that error, and the M2 of the
    # parts are sums of squares: relative DEPTH + 8 roundings, plus the square of the mean's own error
    mean_err = DEPTH * U * np.abs(xg).mean((1, 3), keepdims=True)
    var_err = (DEPTH + 8) * U * var + mean_err ** 2
    rstd_rel = 0.5 * var_err / (var + eps) + 4 * U
    over = lambda v: np.broadcast_to(v, xg.shape).reshape(n, p, c)  # noqa: E731
    xhat_err = over(rstd * (mean_err + U * np.abs(mean))) + np.abs(xhat) * (over(rstd_rel) + 3 * U)
    z_err = np.abs(weight) * xhat_err + 3 * U * (np.abs(xhat * weight) + np.abs(bias))
    y = _act(z, act)
    y_err = (1.1 if act == "silu" else 1.0) * z_err + (8 * U * np.abs(y) if act == "silu" else 0.0)   # |silu'| <= 1.1
    stats = np.concatenate((mean.reshape(n, groups, 1), rstd.reshape(n, groups, 1)), -1)
    stats_err = np.concatenate((mean_err.reshape(n, groups, 1), (rstd * rstd_rel).reshape(n, groups, 1)), -1)
    return y, stats, y_err + 1e-37, stats_err + 1e-37


def backward(x, weight, bias, stats, groups, act, g):
    """dx, dweight, dbias from 32-bit inputs (stats among them), and their bounds"""
    n, p, c = x.shape
    w = weight.astype(np.float64)
    mean32, rstd32 = (np.broadcast_to(stats[:, None, :, None, k], (n, p, groups, c // groups)).reshape(n, p, c) for k in (0, 1))
    xhat = (x.astype(np.float64) - mean32) * rstd32
    z = xhat * w + bias
    # ReLU's mask goes by z as 32 bits round it, step by step
    z32 = ((x - mean32) * rstd32).astype(np.float32) * weight + bias
    slope = (z32 > 0).astype(np.float64) if act == "relu" else _act_slope(z, act)
    dz = g.astype(np.float64) * slope
    xhat_err = 2 * U * np.abs(xhat) + U * np.abs(rstd32 * mean32.astype(np.float64))
    z_err = np.abs(w) * xhat_err + 2 * U * (np.abs(xhat * w) + np.abs(z))
    # |silu''| <= 0.5; the slope itself takes some ten roundings
    dz_err = np.abs(g) * ((0.5 * z_err + 10 * U) if act == "silu" else U * 0)
    dbias, dbias_err = dz.sum((0, 1)), (dz_err + DEPTH * U * np.abs(dz)).sum((0, 1))
    t = dz * xhat
    t_err = dz_err * np.abs(xhat) + np.abs(dz) * xhat_err + U * np.abs(t)
    dweight, dweight_err = t.sum((0, 1)), (t_err + DEPTH * U * np.abs(t)).sum((0, 1))
    grouped = lambda v: np.broadcast_to(_per_group(v, groups).mean((1, 3), keepdims=True), (n, p, groups, c // groups)).reshape(n, p, c)  # noqa: E731
    dh, dh_err = dz * w, np.abs(w) * dz_err + U * np.abs(dz * w)
    s1, s1_err = grouped(dh), grouped(dh_err + DEPTH * U * np.abs(dh))
    s2, s2_err = grouped(dh * xhat), grouped(np.abs(w) * t_err + (DEPTH + 2) * U * np.abs(dh * xhat))
    dx = (dh - s1 - xhat * s2) * rstd32
    dx_err = rstd32 * (dh_err + s1_err + np.abs(xhat) * s2_err + np.abs(s2) * xhat_err
                       + 4 * U * (np.abs(dh) + np.abs(s1) + np.abs(xhat * s2)))
    return (dx, dweight, dbias), (dx_err + 1e-37, dweight_err + 1e-37, dbias_err + 1e-37)
