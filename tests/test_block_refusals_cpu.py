"""What sy_rotary_create, sy_block_means, sy_block_select and sy_block_attention refuse, before the context is looked
at: every call here has none, and no pointer is followed."""
import ctypes

import pytest

from simdyolo_amd import Tensor
from simdyolo_amd import _native as N

AT = 0x10000000


def view(c=64, h=4, w=8, n=2, ldc=None, data=AT):
    return Tensor(data, n, c, h, w, c if ldc is None else ldc, 0)


def cfg(**kw):
    base = dict(heads=4, kv_heads=2, key_dim=16, head_dim=32, block_h=2, block_w=4, selected=2, causal=0, scale=0.25)
    return N.BlockConfig(**{**base, **kw})


def far(i):
    return AT + (i << 24)


def attention(c=None, q=None, k=None, v=None, o=None, blocks=far(9), starts=None, lengths=None):
    q = q or view(64, data=far(1))
    k = k or view(32, data=far(2))
    v = v or view(64, data=far(3))
    o = o or view(128, data=far(4))
    return N.lib().sy_block_attention(None, c or cfg(), q, k, v, blocks, starts, lengths, o)


def select(c=None, q=None, m=None, blocks=far(9), starts=None, lengths=None):
    return N.lib().sy_block_select(None, c or cfg(), q or view(64, data=far(1)),
                                   m or view(32, h=2, w=2, data=far(2)), starts, lengths, blocks)


def means(c=None, k=None, m=None, starts=None, tokens=0, lengths=None):
    return N.lib().sy_block_means(None, c or cfg(), k or view(32, data=far(2)), starts, tokens, lengths,
                                  m or view(32, h=2, w=2, data=far(5)))


def why():
    return N.lib().sy_last_error().decode()


@pytest.mark.parametrize("call", [attention, select, means])
def test_ordinary_call_reaches_the_context(call):
    assert call() == N.SY_EINVAL and why() == "null context"


@pytest.mark.parametrize("call", [attention, select, means])
@pytest.mark.parametrize("change,code", [
    (dict(heads=3), N.SY_EINVAL), (dict(heads=0), N.SY_EINVAL), (dict(kv_heads=0), N.SY_EINVAL),
    (dict(key_dim=0), N.SY_EINVAL), (dict(key_dim=18), N.SY_EUNSUPPORTED), (dict(head_dim=-4), N.SY_EINVAL),
    (dict(key_dim=132), N.SY_EUNSUPPORTED), (dict(head_dim=132), N.SY_EUNSUPPORTED),
    (dict(block_h=0), N.SY_EINVAL), (dict(block_w=-1), N.SY_EINVAL),
    (dict(block_h=32, block_w=33), N.SY_EUNSUPPORTED), (dict(block_h=2 ** 30, block_w=2 ** 30), N.SY_EUNSUPPORTED),
    (dict(selected=0), N.SY_EINVAL), (dict(selected=65), N.SY_EUNSUPPORTED), (dict(causal=2), N.SY_EINVAL),
    (dict(causal=1), N.SY_EINVAL), (dict(scale=0.0), N.SY_EINVAL), (dict(scale=-1.0), N.SY_EINVAL),
    (dict(scale=float("nan")), N.SY_EINVAL), (dict(scale=float("inf")), N.SY_EINVAL),
], ids=str)
def test_config(call, change, code):
    assert call(cfg(**change)) == code
    assert why() != "null context"


@pytest.mark.parametrize("call,name,good", [(attention, "q", dict(c=64)), (attention, "k", dict(c=32)),
                                            (attention, "v", dict(c=64)), (attention, "o", dict(c=128)),
                                            (select, "q", dict(c=64)), (select, "m", dict(c=32, h=2, w=2)),
                                            (means, "k", dict(c=32)), (means, "m", dict(c=32, h=2, w=2))])
@pytest.mark.parametrize("bad", [dict(data=0), dict(data=far(8) + 4), dict(ldc=-4), dict(ldc=200 + 2), dict(n=0),
                                 dict(c=8), dict(n=3)], ids=str)
def test_views(call, name, good, bad):
    if bad == dict(n=3) and name == "q" and call is select:
        assert call(q=view(**{**good, "data": far(8), **bad})) == N.SY_EINVAL
        return
    assert call(**{name: view(**{"data": far(8), **good, **bad})}) == N.SY_EINVAL
    assert why() != "null context"


def test_nchw_views():
    t = view(64, data=far(8))
    t.layout = 1
    assert attention(q=t) == N.SY_EUNSUPPORTED and select(q=t) == N.SY_EUNSUPPORTED
    t = view(32, data=far(8))
    t.layout = 1
    assert means(k=t) == N.SY_EUNSUPPORTED


@pytest.mark.parametrize("strides", [dict(q_stride=8), dict(k_stride=18), dict(v_stride=28), dict(q_stride=20)], ids=str)
def test_strides(strides):
    assert attention(cfg(**strides)) == N.SY_EINVAL
    assert why() != "null context"


def test_shapes_differ():
    assert attention(k=view(32, w=9, data=far(2))) == N.SY_EINVAL
    assert attention(o=view(128, w=9, data=far(4))) == N.SY_EINVAL
    assert attention(o=view(132, data=far(4))) == N.SY_EINVAL
    assert means(m=view(32, h=2, w=3, data=far(5))) == N.SY_EINVAL
    assert attention(blocks=None) == N.SY_EINVAL and select(blocks=None) == N.SY_EINVAL
    assert means(tokens=-1) == N.SY_EINVAL
    assert why() != "null context"


@pytest.mark.parametrize("extra", [dict(lengths=far(10))], ids=str)
def test_lengths_are_of_rows(extra):
    assert attention(**extra) == N.SY_EINVAL and select(**extra) == N.SY_EINVAL and means(**extra) == N.SY_EINVAL
    assert why() != "null context"
    assert means(starts=far(10), tokens=1) == N.SY_EINVAL


def test_causal_needs_rows():
    c = cfg(causal=1, block_h=1)
    assert attention(c) == N.SY_EINVAL and select(c) == N.SY_EINVAL and means(c, m=view(32, h=4, w=2)) == N.SY_EINVAL
    assert why() != "null context"


def test_outputs_overlap():
    assert attention(o=view(128, data=far(1))) == N.SY_EINVAL
    assert attention(o=view(128, data=far(3) + 64)) == N.SY_EINVAL
    assert means(m=view(32, h=2, w=2, data=far(2) + 128)) == N.SY_EINVAL
    assert "overlap" in why()


def test_more_heads_and_queries_than_lists():
    one = dict(h=1, w=1, data=far(1))
    many = cfg(heads=4096, kv_heads=4096, key_dim=4, head_dim=4, block_h=1, block_w=1, selected=1)
    n = 1 << 13  # 2^25 key heads
    q, k, v = (view(4 * 4096, n=n, **{**one, "data": AT + (i << 40)}) for i in (1, 2, 3))
    assert select(many, q=q, m=k) == N.SY_EUNSUPPORTED
    assert attention(many, q=q, k=k, v=v, o=view(4 * 4096, n=n, h=1, w=1, data=AT + (4 << 40))) == N.SY_EUNSUPPORTED
    q, o = (view(c, h=1 << 14, w=1 << 15, n=1, data=AT + (i << 44)) for c, i in ((64, 1), (128, 2)))
    assert attention(cfg(selected=4), q=q, o=o, k=view(32, n=1, data=far(2)), v=view(64, n=1, data=far(3))) == \
        N.SY_EUNSUPPORTED
    assert why() != "null context"


ROTARY = dict(head_dim=32, dim=16, axes=1, interleaved=0, base=10000.0, scaling=0, factor=1.0, low=1.0, high=32.0,
              original=4096)


def rotary(**kw):
    h = ctypes.c_uint64()
    c = N.RotaryConfig(**{**ROTARY, **kw})
    return N.lib().sy_rotary_create(None, ctypes.byref(c), ctypes.byref(h))


def test_rotary_create_reaches_the_context():
    for s in range(4):
        assert rotary(scaling=s, factor=4.0) == N.SY_EINVAL and why() == "null context"


@pytest.mark.parametrize("change,code", [
    (dict(axes=0), N.SY_EINVAL), (dict(axes=3), N.SY_EINVAL), (dict(dim=0), N.SY_EINVAL), (dict(dim=36), N.SY_EINVAL),
    (dict(dim=15), N.SY_EINVAL), (dict(dim=6, axes=2), N.SY_EINVAL), (dict(head_dim=30), N.SY_EUNSUPPORTED),
    (dict(head_dim=516), N.SY_EUNSUPPORTED), (dict(interleaved=2), N.SY_EINVAL), (dict(base=0.0), N.SY_EINVAL),
    (dict(base=float("nan")), N.SY_EINVAL), (dict(scaling=4), N.SY_EINVAL), (dict(scaling=-1), N.SY_EINVAL),
    (dict(scaling=1, factor=0.5), N.SY_EINVAL), (dict(scaling=2, factor=2.0, dim=2), N.SY_EINVAL),
    (dict(scaling=3, factor=2.0, original=0), N.SY_EINVAL), (dict(scaling=3, factor=2.0, low=40.0), N.SY_EINVAL),
], ids=str)
def test_rotary_config(change, code):
    assert rotary(**change) == code
    assert why() != "null context"


def test_rotary_run_without_context():
    assert N.lib().sy_rotary_run(None, 1, None, 0, None) == N.SY_EINVAL
