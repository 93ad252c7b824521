"""What sy_group_norm, sy_cross_attention and sy_gated_create refuse, before the context is looked at: every call here
has none, and no pointer is followed."""
import ctypes

import numpy as np
import pytest

from simdyolo_amd import Tensor
from simdyolo_amd import _native as N

AT = 0x10000000


def view(c=64, h=4, w=8, n=2, ldc=None, data=AT):
    return Tensor(data, n, c, h, w, c if ldc is None else ldc, 0)


def far(i):
    return AT + (i << 24)


def why():
    return N.lib().sy_last_error().decode()


def norm(x=None, groups=8, gamma=far(7), beta=far(8), eps=1e-5, act=0, y=None):
    return N.lib().sy_group_norm(None, x or view(data=far(1)), groups, gamma, beta, eps, act, y or view(data=far(2)))


def cfg(**kw):
    base = dict(heads=4, kv_heads=2, key_dim=16, head_dim=32, scale=0.25)
    return N.CrossConfig(**{**base, **kw})


def cross(c=None, q=None, k=None, v=None, o=None, lengths=far(6), mask=None):
    return N.lib().sy_cross_attention(None, c or cfg(), q or view(64, data=far(1)), k or view(32, h=3, data=far(2)),
                                      v or view(64, h=3, data=far(3)), lengths, mask, o or view(128, data=far(4)))


def test_ordinary_calls_reach_the_context():
    mask = N.KeyMask(far(9), 24, 0, 0)
    for call in (norm, cross, lambda: cross(lengths=None), lambda: cross(mask=mask), lambda: norm(gamma=None, beta=None),
                 lambda: norm(y=view(data=far(1))), lambda: N.lib().sy_gated_run(None, 1, view(), view(data=far(1)))):
        assert call() == N.SY_EINVAL and why() == "null context"


@pytest.mark.parametrize("change,code", [
    (dict(groups=0), N.SY_EINVAL), (dict(groups=-1), N.SY_EINVAL), (dict(groups=5), N.SY_EINVAL),
    (dict(groups=128), N.SY_EINVAL), (dict(act=-1), N.SY_EINVAL), (dict(act=6), N.SY_EINVAL), (dict(eps=-1e-9), N.SY_EINVAL),
    (dict(eps=float("nan")), N.SY_EINVAL), (dict(eps=float("inf")), N.SY_EINVAL), (dict(gamma=far(7) + 2), N.SY_EINVAL),
    (dict(beta=far(8) + 1), N.SY_EINVAL), (dict(gamma=far(2) + 64), N.SY_EINVAL), (dict(beta=far(2)), N.SY_EINVAL),
    (dict(x=view(data=0)), N.SY_EINVAL), (dict(x=view(data=far(1) + 2)), N.SY_EINVAL), (dict(x=view(n=0)), N.SY_EINVAL),
    (dict(x=view(n=3, data=far(1))), N.SY_EINVAL), (dict(x=view(w=7, data=far(1))), N.SY_EINVAL),
    (dict(x=view(ldc=60, data=far(1))), N.SY_EINVAL), (dict(y=view(32, data=far(2))), N.SY_EINVAL),
    (dict(y=view(data=far(1) + 4)), N.SY_EINVAL), (dict(y=view(ldc=68, data=far(1))), N.SY_EINVAL),
    (dict(x=view(8, h=2 ** 15, w=2 ** 15, n=1), y=view(8, h=2 ** 15, w=2 ** 15, n=1)), N.SY_EUNSUPPORTED),
    (dict(x=Tensor(far(1), 2, 64, 4, 8, 64, 1)), N.SY_EUNSUPPORTED),
], ids=str)
def test_norm(change, code):
    assert norm(**change) == code
    assert why() != "null context"


@pytest.mark.parametrize("change,code", [
    (dict(heads=3), N.SY_EINVAL), (dict(heads=0), N.SY_EINVAL), (dict(kv_heads=0), N.SY_EINVAL),
    (dict(kv_heads=-2), N.SY_EINVAL), (dict(key_dim=0), N.SY_EINVAL), (dict(key_dim=18), N.SY_EUNSUPPORTED),
    (dict(head_dim=-4), N.SY_EINVAL), (dict(key_dim=132), N.SY_EUNSUPPORTED), (dict(head_dim=132), N.SY_EUNSUPPORTED),
    (dict(scale=0.0), N.SY_EINVAL), (dict(scale=-1.0), N.SY_EINVAL), (dict(scale=float("nan")), N.SY_EINVAL),
    (dict(scale=float("inf")), N.SY_EINVAL), (dict(q_stride=12), N.SY_EINVAL), (dict(k_stride=18), N.SY_EINVAL),
    (dict(v_stride=-32), N.SY_EINVAL), (dict(k_stride=20), N.SY_EINVAL),
    (dict(heads=2 ** 26, kv_heads=2 ** 26), N.SY_EUNSUPPORTED),
], ids=str)
def test_cross_config(change, code):
    assert cross(cfg(**change)) == code
    assert why() != "null context"


@pytest.mark.parametrize("name,good", [("q", dict(c=64)), ("k", dict(c=32, h=3)), ("v", dict(c=64, h=3)), ("o", dict(c=128))])
@pytest.mark.parametrize("bad", [dict(data=0), dict(data=far(8) + 4), dict(ldc=-4), dict(ldc=202), dict(n=0), dict(c=8),
                                 dict(n=3), dict(w=7), dict(h=2 ** 15, w=2 ** 15, n=1)], ids=str)
def test_cross_views(name, good, bad):
    code = cross(**{name: view(**{"data": far(8), **good, **bad})})
    assert code in (N.SY_EINVAL, N.SY_EUNSUPPORTED) and why() != "null context"


def test_cross_others():
    for mask in (N.KeyMask(0, 0, 0, 0), N.KeyMask(far(9), -1, 0, 0), N.KeyMask(far(9), 0, -1, 0), N.KeyMask(far(9), 0, 0, -1)):
        assert cross(mask=mask) == N.SY_EINVAL and why() != "null context"
    for at in (far(4), far(4) - 20, far(4) + 2 * 128 * 4 * 32 - 1):
        assert cross(mask=N.KeyMask(at, 24, 0, 0)) == N.SY_EINVAL and "mask" in why()
    assert cross(mask=N.KeyMask(far(3) + 8, 0, 0, 1 << 40)) == N.SY_EINVAL and "mask" in why()
    assert cross(lengths=far(4) + 64) == N.SY_EINVAL and "lengths" in why()
    for at in (1, 2, 3):
        assert cross(o=view(128, data=far(at))) == N.SY_EINVAL and "overlaps" in why()
    assert cross(k=view(32, h=3, ldc=1 << 24, data=far(100)), v=view(64, h=3, data=far(40))) == N.SY_EUNSUPPORTED
    assert N.lib().sy_cross_attention(None, None, view(), view(), view(), None, None, view()) == N.SY_EINVAL


def gated(gate=True, up=True, oc=4, ic=6, act=1, out=True):
    w = np.zeros((4, 6), np.float32)
    p = w.ctypes.data_as(ctypes.POINTER(ctypes.c_float))
    h = ctypes.c_uint64()
    return N.lib().sy_gated_create(None, p if gate else None, p if up else None, None, None, oc, ic, act,
                                   ctypes.byref(h) if out else None)


@pytest.mark.parametrize("change,code", [
    (dict(gate=False), N.SY_EINVAL), (dict(up=False), N.SY_EINVAL), (dict(out=False), N.SY_EINVAL), (dict(oc=0), N.SY_EINVAL),
    (dict(ic=-1), N.SY_EINVAL), (dict(act=-1), N.SY_EINVAL), (dict(act=6), N.SY_EINVAL),
    (dict(oc=1 << 16, ic=1 << 15), N.SY_EUNSUPPORTED), (dict(oc=1 << 24, ic=1), N.SY_EUNSUPPORTED),
    (dict(oc=1, ic=1 << 24), N.SY_EUNSUPPORTED)], ids=str)
def test_gated_create(change, code):
    assert gated() == N.SY_EINVAL and why() == "null context"
    assert gated(**change) == code and why() != "null context"
