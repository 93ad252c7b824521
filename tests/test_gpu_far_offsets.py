"""Normalisation, cross attention and gated projections on views whose pixels lie so far apart that offsets pass 32 bits."""
import numpy as np
import pytest

import _blocks as R
import _layers as L
from simdyolo_amd import Tensor
from simdyolo_amd import _native as N

pytestmark = pytest.mark.gpu

FLOATS = 4_750_000_000  # 19 GB
PITCH = (1 << 23) + 32  # 560 pixels: 4.70e9 floats


class Far:
    def __init__(self, hip):
        self.hip, self.at = hip, hip.malloc(4 * FLOATS)

    def view(self, channel, rows, c, pitch=PITCH):
        assert channel + (rows - 1) * pitch + c <= FLOATS
        return Tensor(self.at + 4 * channel, 1, c, 1, rows, pitch, 0)

    def put(self, view, a):
        for i, row in enumerate(a.reshape(view.w, view.c)):
            self.hip.h2d(view.data + 4 * i * view.ldc, np.ascontiguousarray(row))
        return view

    def get(self, view):
        return np.stack([self.hip.d2h(view.data + 4 * i * view.ldc, (view.c,)) for i in range(view.w)])


@pytest.fixture
def far(hip):
    f = Far(hip)
    yield f
    hip.flush()
    hip.free(f.at)


@pytest.mark.parametrize("groups", [1, 8])
def test_norm(hip, far, groups):
    x = R.rng(1).standard_normal((1, 560, 64)).astype(np.float32)
    view = far.put(far.view(0, 560, 64), x)
    hip.group_norm(view, view, groups, act=N.ACT_SILU)
    exp, bound = L.group_norm(x, groups, None, None, 1e-5, N.ACT_SILU)
    assert (np.abs(far.get(view)[None] - exp) <= bound).all()


@pytest.mark.parametrize("rows,ic,oc,pitch", [(17, 64, 96, (1 << 28) + 4), (560, 64, 256, PITCH), (560, 320, 256, PITCH),
                                              (560, 600, 256, PITCH), (560, 600, 1900, PITCH)])
def test_gated(hip, far, rows, ic, oc, pitch):
    g = R.rng(2)
    x = g.standard_normal((rows, ic)).astype(np.float32)
    w = [(g.standard_normal((oc, ic)) * ic ** -0.5).astype(np.float32) for _ in range(2)]
    vx, vy = far.put(far.view(8, rows, ic, pitch), x), far.view(4096, rows, oc, pitch)
    hip.gated(hip.gated_create(*w), vx, vy)
    exp, bound = L.gated(x, *w, None, None, N.ACT_SILU)
    assert (np.abs(far.get(vy) - exp) <= bound).all()


@pytest.mark.parametrize("tq,heads", [(1, 2), (40, 4), (1200, 8)])
def test_states(hip, far, tq, heads):
    g = R.rng(3)
    q, k, v = (g.standard_normal(s).astype(np.float32) for s in ((1, tq, heads, 32), (1, 560, 2, 32), (1, 560, 2, 64)))
    vk, vv = far.put(far.view(0, 560, 64), k), far.put(far.view(1024, 560, 128), v)
    with R.Device(hip) as d:
        vq, _, _ = d.view(q, 1, tq)
        vo, _, read = d.view(np.zeros((1, tq, heads, 64), np.float32), 1, tq)
        hip.cross_attention(N.CrossConfig(heads, 2, 32, 64, 0, 0, 0, 32 ** -0.5), vq, vk, vv, vo)
        exp, bound = L.cross(q, k, v, 32 ** -0.5)
        assert (np.abs(read() - exp) <= bound).all()


@pytest.mark.parametrize("tk", [40, 900])
def test_queries(hip, far, tk):
    g = R.rng(4)
    q, k, v = (g.standard_normal(s).astype(np.float32) for s in ((1, 560, 4, 32), (1, tk, 2, 32), (1, tk, 2, 64)))
    vq, vo = far.put(far.view(0, 560, 128), q), far.view(2048, 560, 256)
    with R.Device(hip) as d:
        vk, _, _ = d.view(k, 1, tk)
        vv, _, _ = d.view(v, 1, tk)
        hip.cross_attention(N.CrossConfig(4, 2, 32, 64, 0, 0, 0, 32 ** -0.5), vq, vk, vv, vo)
        exp, bound = L.cross(q, k, v, 32 ** -0.5)
        assert (np.abs(far.get(vo).reshape(exp.shape) - exp) <= bound).all()
