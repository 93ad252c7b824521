"""Normalisation, cross attention, gated projections and the closing 1x1 convolution in a row, as a decoder's layer runs
them: object queries that look at a map (with a mask and ragged lengths), and a map that looks at a text, against
float64, eagerly and captured."""
import numpy as np
import pytest

import _blocks as R
import _layers as L
from simdyolo_amd import Tensor
from simdyolo_amd import _native as N
from simdyolo_amd.device import HipContext

pytestmark = pytest.mark.gpu


class Layer:
    """x + o(cross(q(norm x), states)), then + down(gated(norm .)); all of it on one context, in buffers of its own."""

    def __init__(self, ctx, d, n, h, w, c, heads, tk, cs, hidden, groups, masked, seed):
        g = R.rng(seed)
        self.ctx, self.d, self.shape = ctx, d, (n, h, w, c, heads, tk, cs, hidden, groups)
        r = lambda *s: (g.standard_normal(s) * s[-1] ** -0.5).astype(np.float32)
        self.wq, self.wkv, self.wo = r(c, c), r(2 * c, cs), r(c, c)
        self.wg, self.wu, self.wd = r(hidden, c), r(hidden, c), r(c, hidden)
        self.bg, self.bu = (0.1 * g.standard_normal(hidden)).astype(np.float32), np.zeros(hidden, np.float32)
        self.gamma, self.beta = (1 + 0.2 * g.standard_normal(c)).astype(np.float32), np.zeros(c, np.float32)
        conv = lambda a: ctx.conv_create(a[:, :, None, None])
        self.q, self.kv, self.o, self.down = conv(self.wq), conv(self.wkv), conv(self.wo), conv(self.wd)
        self.gated = ctx.gated_create(self.wg, self.wu, self.bg, self.bu, act=N.ACT_GELU)
        self.pg, self.pb = d.put(self.gamma), d.put(self.beta)
        t = h * w
        view = lambda t_, ch, hh, ww: Tensor(d.put(np.full((n, t_, ch), np.nan, np.float32)), n, ch, hh, ww, ch, 0)
        self.x, self.y, self.z = (view(t, c, h, w) for _ in range(3))
        self.a, self.b = view(t, c, h, w), view(t, c, h, w)
        self.states, self.kvs, self.hid = view(tk, cs, 1, tk), view(tk, 2 * c, 1, tk), view(t, hidden, h, w)
        self.lengths = d.ints([0] * n)
        self.mask = d.put(np.zeros((n, t, tk), np.uint8)) if masked else None
        self.cfg = N.CrossConfig(heads, heads, c // heads, c // heads, 0, 0, 0, (c // heads) ** -0.5)
        self.new(seed + 1)

    def new(self, seed):
        n, h, w, c, _, tk, cs, _, _ = self.shape
        g = R.rng(seed)
        self.hx = g.standard_normal((n, h * w, c)).astype(np.float32)
        self.hs = g.standard_normal((n, tk, cs)).astype(np.float32)
        self.hl = g.integers(0, tk + 1, n).astype(np.int32)
        self.ctx.h2d(self.x.data, self.hx)
        self.ctx.h2d(self.states.data, self.hs)
        self.ctx.h2d(self.lengths, self.hl)
        self.hm = None
        if self.mask:
            self.hm = (g.random((n, h * w, tk)) < 0.4).astype(np.uint8)
            self.hm[:, 1] = 0
            self.ctx.h2d(self.mask, self.hm)

    def __call__(self):
        n, h, w, c, heads, tk, cs, hidden, groups = self.shape
        ctx = self.ctx
        ctx.group_norm(self.x, self.a, groups, self.pg, self.pb)
        ctx.conv(self.q, self.a, self.b)
        ctx.conv(self.kv, self.states, self.kvs)
        m = N.KeyMask(self.mask, h * w * tk, 0, tk) if self.mask else None
        ctx.cross_attention(self.cfg, self.b, self.kvs.slice(0, c), self.kvs.slice(c, c), self.a, self.lengths, m)
        ctx.conv(self.o, self.a, self.y, self.x)
        ctx.group_norm(self.y, self.y, groups, self.pg, self.pb, act=N.ACT_SILU)
        ctx.gated(self.gated, self.y, self.hid)
        if hidden % 4 == 0:
            ctx.conv(self.down, self.hid, self.z, self.y)
        else:  # such convolutions take no residual
            ctx.conv(self.down, self.hid, self.a)
            ctx.add(self.a, self.y, self.z)

    def check(self):
        """The error of a step travels through the others: float32 in numpy, step by step, has one like it, and a few
        times that is allowed."""
        n, h, w, c, heads, tk, cs, hidden, groups = self.shape

        def forward(t):
            f = lambda a: a.astype(t)
            norm = lambda x, act: f(L.group_norm(x.astype(np.float32) if t == np.float32 else x, groups, self.gamma,
                                                 self.beta, 1e-5, act)[0])
            a = norm(f(self.hx), N.ACT_NONE)
            q, kv = a @ f(self.wq).T, f(self.hs) @ f(self.wkv).T
            kd = c // heads
            k, v = kv[..., :c].reshape(n, tk, heads, kd), kv[..., c:].reshape(n, tk, heads, kd)
            s = np.einsum("bihd,bjhd->bhij", q.reshape(n, h * w, heads, kd), k) * t(kd ** -0.5)
            see = (np.arange(tk) < self.hl[:, None])[:, None, None]
            if self.hm is not None:
                see = see & (self.hm != 0)[:, None]
            s = np.where(see, s, t(-np.inf))
            top = s.max(-1, keepdims=True)
            e = np.exp(s - np.where(np.isfinite(top), top, 0))
            p = e / np.maximum(e.sum(-1, keepdims=True), t(1e-30))
            o = np.einsum("bhij,bjhd->bihd", p, v).reshape(n, h * w, c)
            y = norm(f(self.hx) + o @ f(self.wo).T, N.ACT_SILU)
            g = f(L.activate(N.ACT_GELU, (y @ f(self.wg).T + f(self.bg)).astype(np.float64)))
            return y + (g * (y @ f(self.wu).T + f(self.bu))) @ f(self.wd).T

        exp = forward(np.float64)
        off = np.abs(forward(np.float32) - exp)
        self.ctx.flush()
        got = self.ctx.d2h(self.z.data, exp.shape)
        assert (np.abs(got - exp) <= 16 * off.max()).all(), (np.abs(got - exp).max(), off.max())


SHAPES = [(2, 1, 100, 64, 4, 420, 48, 170, 8, True), (1, 20, 20, 128, 4, 77, 64, 344, 32, False),
          (3, 1, 1, 32, 2, 300, 20, 90, 1, False)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_layer(hip, shape):
    with R.Device(hip) as d:
        layer = Layer(hip, d, *shape, seed=1)
        for seed in (2, 3):
            layer.new(seed)
            layer()
            layer.check()


def test_layers_captured():
    """Three layers' graphs that share the context's scratch, on new inputs, with eager work of another between."""
    with HipContext(0) as ctx, R.Device(ctx) as d:
        layers = [Layer(ctx, d, *s, seed=10 + i) for i, s in enumerate(SHAPES)]
        for l in layers:
            l()
        graphs = []
        for l in layers:
            ctx.graph_begin()
            l()
            graphs.append(ctx.graph_end())
        for turn in range(3):
            for i, (l, g) in enumerate(zip(layers, graphs)):
                l.new(100 * turn + i)
                ctx.h2d(l.z.data, np.full(l.z.n * l.z.h * l.z.w * l.z.c, np.nan, np.float32))
                if turn != 1:
                    layers[i - 1]()
                ctx.graph_launch(g)
                l.check()
