"""Attention over chosen key blocks and rotary positions in float64 (numpy), and device buffers for their tests.

Arrays are [n, h * w, heads, dim]; `cfg` is a dict of sy_block_config's fields without strides and scale."""
import math

import numpy as np

from simdyolo_amd import Tensor
from simdyolo_amd import _native as N


UNIT = 2.0 ** -24  # half a step of float32, relative


def rng(seed):
    return np.random.Generator(np.random.PCG64(seed))


# ---------------------------------------------------------------- formulas

def frequencies(part, base, scaling, factor, low, high, original):
    i = np.arange(part // 2)
    f = float(np.float32(base)) ** (-2.0 * i / part)
    if scaling == N.ROTARY_LINEAR:
        return f / factor, 1.0
    if scaling == N.ROTARY_BASE:
        return (float(np.float32(base)) * factor ** (part / (part - 2))) ** (-2.0 * i / part), 1.0
    if scaling == N.ROTARY_PARTS:
        keep = np.clip((original * f / (2 * math.pi) - low) / (high - low), 0, 1)
        return f * keep + f / factor * (1 - keep), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def rotate(x, at, dim, interleaved, f, amplitude):
    """x [n, t, heads, d], at [n, t, axes]; also the bound's weight |a| + |b| of each value and the largest angle."""
    y, near = x.astype(np.float64), np.zeros(x.shape)
    axes, part = at.shape[-1], dim // at.shape[-1]
    for axis in range(axes):
        for i in range(part // 2):
            a = axis * part + (2 * i if interleaved else i)
            b = a + 1 if interleaved else a + part // 2
            angle = (at[..., axis].astype(np.float64) * f[i])[..., None]
            c, s = np.cos(angle) * amplitude, np.sin(angle) * amplitude
            u, v = x[..., a].astype(np.float64), x[..., b].astype(np.float64)
            y[..., a], y[..., b] = u * c - v * s, v * c + u * s
            near[..., a] = near[..., b] = (np.abs(u) + np.abs(v)) * amplitude * (1 + np.abs(angle) * 2.0 ** -30)
    return y, near


def block_tokens(cfg, h, w, j):
    """Token indices of block j."""
    across = -(-w // cfg["block_w"])
    y = np.arange(j // across * cfg["block_h"], min(h, (j // across + 1) * cfg["block_h"]))
    x = np.arange(j % across * cfg["block_w"], min(w, (j % across + 1) * cfg["block_w"]))
    return (y[:, None] * w + x[None]).reshape(-1)


def count_blocks(cfg, h, w):
    return -(-h // cfg["block_h"]) * -(-w // cfg["block_w"])


def means(cfg, k, h, w, lengths=None):
    n, _, kv, kd = k.shape
    out = np.zeros((n, count_blocks(cfg, h, w), kv, kd))
    for b in range(n):
        for j in range(out.shape[1]):
            at = block_tokens(cfg, h, w, j)
            if lengths is not None:
                at = at[at < lengths[b]]
            if at.size:
                out[b, j] = k[b, at].astype(np.float64).mean(0)
    return out


def select(cfg, q, m, starts=None, lengths=None):
    n, tq, heads, kd = q.shape
    blocks, kv, sel = m.shape[1], cfg["kv_heads"], cfg["selected"]
    out = np.full((n, tq, kv, sel), -1, np.int32)
    with np.errstate(invalid="ignore", over="ignore"):
        s = np.einsum("btgd,bjgd->btgj", q.astype(np.float64).reshape(n, tq, kv, heads // kv, kd).sum(3),
                      m.astype(np.float64))
    for b in range(n):
        for i in range(tq):
            seen, own = blocks, -1
            if lengths is not None:
                seen = min(seen, -(-max(int(lengths[b]), 0) // cfg["block_w"]))
            if cfg["causal"]:
                at = (int(starts[b]) if starts is not None else 0) + i
                seen = 0 if at < 0 else min(seen, at // cfg["block_w"] + 1)
                own = at // cfg["block_w"] if at >= 0 and at // cfg["block_w"] < seen else -1
            for g in range(kv):
                score = s[b, i, g, :seen]
                rank = sorted(range(seen), key=lambda j: (j != own, bool(np.isnan(score[j])),
                                                          0.0 if np.isnan(score[j]) else -score[j], j))
                got = sorted(rank[:sel])
                out[b, i, g, :len(got)] = got
    return out


def attend(cfg, q, k, v, blocks, h, w, scale, starts=None, lengths=None):
    """(output, bound) in float64.

    A score is a sum of kd products, each off by at most 3 x 2^-22 = 12 x 2^-24 (pairs of f16 values; in plain float32
    by 2^-24), its partial sums by 2^-24 each, and is multiplied by the scale: within (kd + 24) 2^-24 of sum |q||k|
    scale, which the exponential takes over twice (score and maximum).  The exponential itself, its argument's
    rounding (relative to the argument, below 128), the pairs of weights and values (3 x 2^-22 of each product) and the
    joins of partial sums add 2^-17 at most, and sums over the keys 2^-24 for each key."""
    n, tq, heads, kd = q.shape
    kv, hd, t = cfg["kv_heads"], v.shape[-1], h * w
    out, bound = np.zeros((n, tq, heads, hd)), np.zeros((n, tq, heads, hd))
    count = count_blocks(cfg, h, w)
    for b in range(n):
        for i in range(tq):
            end = t if lengths is None else min(max(int(lengths[b]), 0), t)
            if cfg["causal"]:
                end = min(end, max((int(starts[b]) if starts is not None else 0) + i + 1, 0))
            for g in range(kv):
                at = [block_tokens(cfg, h, w, j) for j in blocks[b, i, g] if 0 <= j < count]
                at = np.concatenate(at) if at else np.zeros(0, int)
                at = at[at < end]
                if not at.size:
                    continue
                kg, vg = k[b, at, g].astype(np.float64), v[b, at, g].astype(np.float64)
                mine = slice(g * (heads // kv), (g + 1) * (heads // kv))
                qg = q[b, i, mine].astype(np.float64)
                with np.errstate(invalid="ignore", over="ignore"):
                    s = qg @ kg.T * scale
                    off = UNIT * (kd + 24) * (np.abs(qg) @ np.abs(kg).T).max(-1, keepdims=True) * scale
                    p = np.exp(s - s.max(-1, keepdims=True))
                    p /= p.sum(-1, keepdims=True)
                    out[b, i, mine] = p @ vg
                    bound[b, i, mine] = (p @ np.abs(vg)) * (2 * off + 2.0 ** -17 + at.size * UNIT)
    return out, bound


# ------------------------------------------------------------------ device

class Device:
    """Device copies of numpy arrays, freed together."""

    def __init__(self, hip):
        self.hip, self.ptrs = hip, []

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.hip.flush()
        for p in self.ptrs:
            self.hip.free(p)

    def put(self, a):
        a = np.ascontiguousarray(a)
        p = self.hip.malloc(max(a.nbytes, 4))
        self.ptrs.append(p)
        if a.nbytes:
            self.hip.h2d(p, a)
        return p

    def view(self, a, h, w, pad=0, gap=0, before=0):
        """The view of [n, h * w, heads, dim] with `gap` channels between heads, `before` in front of the first and
        `pad` more behind the last; what does not belong to a head is NaN.  The view, its head stride and a
        function that reads the heads (and checks that the rest is as it was)."""
        n, t, heads, dim = a.shape
        stride = dim + gap
        full = np.full((n, t, before + heads * stride + pad), np.nan, np.float32)
        body = full[..., before:before + heads * stride].reshape(n, t, heads, stride)
        body[..., :dim] = a
        full[..., before:before + heads * stride] = body.reshape(n, t, heads * stride)
        p = self.put(full)

        def read():
            self.hip.flush()
            got = self.hip.d2h(p, full.shape)
            heads_ = got[..., before:before + heads * stride].reshape(n, t, heads, stride)
            assert np.isnan(heads_[..., dim:]).all() and np.isnan(got[..., :before]).all()
            assert np.isnan(got[..., before + heads * stride:]).all()
            return np.ascontiguousarray(heads_[..., :dim])
        return Tensor(p + 4 * before, n, (heads - 1) * stride + dim, h, w, full.shape[2], 0), stride, read

    def ints(self, a):
        return None if a is None else self.put(np.asarray(a, np.int32))


def config(cfg, kd, hd, strides=(0, 0, 0), scale=None):
    return N.BlockConfig(heads=cfg["heads"], kv_heads=cfg["kv_heads"], key_dim=kd, head_dim=hd, q_stride=strides[0],
                         k_stride=strides[1], v_stride=strides[2], block_h=cfg["block_h"], block_w=cfg["block_w"],
                         selected=cfg["selected"], causal=cfg["causal"], scale=kd ** -0.5 if scale is None else scale)


def shape(heads, kv_heads, block_h, block_w, selected, causal=0):
    return dict(heads=heads, kv_heads=kv_heads, block_h=block_h, block_w=block_w, selected=selected, causal=causal)
