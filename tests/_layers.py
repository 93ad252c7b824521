"""Group normalisation, cross attention and gated projections in float64 (numpy), each with the bound of its kernel's
error.  Views and device buffers are those of _blocks."""
import math

import numpy as np
from scipy.special import erfc

from simdyolo_amd import _native as N

UNIT = 2.0 ** -24  # half a step of float32, relative
TINY = 2.0 ** -149
ACTS = {"none": N.ACT_NONE, "silu": N.ACT_SILU, "gelu": N.ACT_GELU, "gelu_tanh": N.ACT_GELU_TANH, "relu": N.ACT_RELU,
        "sigmoid": N.ACT_SIGMOID}


def activate(act, x):
    with np.errstate(over="ignore", invalid="ignore"):
        if act == N.ACT_SILU:
            return x / (1 + np.exp(-x))
        if act == N.ACT_GELU:
            return 0.5 * x * erfc(-x / math.sqrt(2))
        if act == N.ACT_GELU_TANH:
            return x / (1 + np.exp(-2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))
        if act == N.ACT_RELU:
            return np.where(x < 0, 0.0, x)
        if act == N.ACT_SIGMOID:
            return 1 / (1 + np.exp(-x))
    return x


def activated(act, x, off):
    """(activation, bound) of a value known to within `off`: no slope is above 1.13; the exponential, its sum with 1, the
    reciprocal and the products are off by 10 halves of a step together.  The argument of GELU's exponentials is off by
    4 halves of a step of itself, which they take over as a factor: x^2 at most for erfc (|x| <= 14, where it ends), twice
    |x| + 0.09 |x|^3 for tanh's."""
    y = activate(act, x)
    with np.errstate(invalid="ignore", over="ignore"):
        if act == N.ACT_NONE or act == N.ACT_RELU:
            return y, off
        more = 10.0
        if act == N.ACT_GELU:
            more = 20 + 4 * np.minimum(x * x, 200)
        elif act == N.ACT_GELU_TANH:
            more = 10 + 4 * np.minimum(2 * np.abs(x) + 0.09 * np.abs(x) ** 3, 150) * (x < 0)
        return y, 1.13 * off + np.abs(y) * more * UNIT + TINY


def group_norm(x, groups, gamma, beta, eps, act):
    """x [n, t, c].  The moments are exact to 2^-40 and better; the mean comes off in two subtractions (of its leading and
    of its following 24 bits), 1 / std, its product with gamma and the sum round once each: 6 halves of a step of
    the product, one of the sum."""
    n, t, c = x.shape
    g = x.astype(np.float64).reshape(n, t, groups, c // groups)
    d = g - g.mean((1, 3), keepdims=True)
    var = (d * d).mean((1, 3), keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore"):
        z = (d / np.sqrt(var + float(np.float32(eps)))).reshape(n, t, c)
    gamma = np.ones(c) if gamma is None else gamma.astype(np.float64)
    beta = np.zeros(c) if beta is None else beta.astype(np.float64)
    z = z * gamma
    return activated(act, z + beta, 6 * UNIT * np.abs(z) + UNIT * np.abs(z + beta) + TINY)


def cross(q, k, v, scale, lengths=None, mask=None):
    """q [n, tq, heads, kd], k, v [n, tk, kv, ..]; mask [n, heads, tq, tk] or what broadcasts to it.

    A score: products of three-part operands within 2^-24 of each, sums of kd of them and the parts' (kd + 8 in
    all), twice (itself and the maximum).  A weight 2^t: its exponent's product, difference and moves with the running
    maximum, 3 halves of a step of |t| + 8, times ln 2, and the exponential; sums over the states and the parts of
    weights and values."""
    n, tq, heads, kd = q.shape
    tk, kv, hd = v.shape[1:]
    scale = float(np.float32(scale))
    out, bound = np.zeros((n, tq, heads, hd)), np.zeros((n, tq, heads, hd))
    if mask is not None:
        mask = np.broadcast_to(mask, (n, heads, tq, tk)) != 0
    for b in range(n):
        end = tk if lengths is None else min(max(int(lengths[b]), 0), tk)
        for h in range(heads):
            kg, vg = (a[b, :end, h // (heads // kv)].astype(np.float64) for a in (k, v))
            qh = q[b, :, h].astype(np.float64)
            for i in range(tq):
                at = slice(None) if mask is None else np.nonzero(mask[b, h, i, :end])[0]
                ki, vi = kg[at], vg[at]
                if not len(ki):
                    continue
                with np.errstate(invalid="ignore", over="ignore"):
                    s = ki @ qh[i] * scale
                    off = UNIT * (kd + 8) * (np.abs(ki) @ np.abs(qh[i])).max() * scale
                    t = s - s.max()
                    p = np.exp(t)
                    p /= p.sum()
                    w = p * (2.1 * (np.abs(t) * 1.4427 + 8) + 8) * UNIT
                    w = np.where(p > 0, w, 0) if np.isfinite(t).all() else w
                    out[b, i, h] = p @ vi
                    bound[b, i, h] = (np.abs(vi) * w[:, None]).sum(0) + \
                        (p @ np.abs(vi)) * (w.sum() + 2 * off + (len(ki) + 12) * UNIT) + TINY * len(ki)
    return out, bound


def gated(x, gate, up, gate_bias, up_bias, act):
    """x [rows, ic].  A product of pairs is off by 3 x 2^-22 of itself, 2^-50 of both rows' largest at most; ic of them (in
    plain float32, ic partial sums)."""
    x, out = x.astype(np.float64), []
    with np.errstate(invalid="ignore", over="ignore"):
        for w, b in ((gate, gate_bias), (up, up_bias)):
            w = w.astype(np.float64)
            near = np.abs(x) @ np.abs(w).T
            s = x @ w.T
            off = near * (x.shape[1] + 16) * UNIT + np.abs(x).sum(1)[:, None] * np.abs(w).max(1) * 2.0 ** -49 + \
                np.abs(x).max(1)[:, None] * np.abs(w).sum(1) * 2.0 ** -49
            if b is not None:
                s = s + b
            out.append((s, off + np.abs(s) * 2 * UNIT + TINY * x.shape[1]))
        (a, a_off), (u, u_off) = out
        y, y_off = activated(act, a, a_off)
        return y * u, y_off * (np.abs(u) + u_off) + np.abs(y) * u_off + np.abs(y * u) * UNIT + TINY
