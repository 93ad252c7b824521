"""sy_rotary_run against the formula in float64.

Bound of a value a c - b s: the reduced angle is a float of at most half a quarter turn (off by 2^-26 of one, 2^-25 in
radians), cosine and sine are within 2 ulp (2^-23), their amplitude, the products and the sum round once each (2^-24):
together below 2^-21 of |a| + |b|.  The angle itself is a product in 64 bits of a 64-bit frequency: 2^-51 of it."""
import numpy as np
import pytest

import _blocks as R
from simdyolo_amd import SyError
from simdyolo_amd import _native as N

pytestmark = pytest.mark.gpu

# head_dim, dim, axes, interleaved: whole and partial heads, halves of 4 n, 4 n + 1 .. 4 n + 3 channels, one pair.
LAYOUTS = [(32, 32, 1, 0), (32, 32, 2, 0), (64, 24, 1, 0), (64, 48, 2, 1), (128, 64, 1, 1), (20, 20, 2, 0),
           (12, 6, 1, 1), (12, 6, 1, 0), (8, 2, 1, 0), (8, 4, 2, 1), (40, 28, 2, 0), (512, 512, 1, 0)]


def run(hip, layout, n, h, w, heads, positions, scaling=N.ROTARY_PLAIN, factor=1.0, base=10000.0, place="apart",
        seed=1):
    hd, dim, axes, inter = layout
    x = [R.rng(seed + i).standard_normal((n, h * w, c, hd)).astype(np.float32) for i, c in enumerate(heads)]
    handle = hip.rotary_create(hd, dim, axes, bool(inter), base, scaling, factor, 1.0, 32.0, 512)
    f, amplitude = R.frequencies(dim // axes, base, scaling, factor, 1.0, 32.0, 512)
    if positions is None:
        i = np.arange(h * w)
        at = np.broadcast_to((i[:, None] if axes == 1 else np.stack([i // w, i % w], -1)), (n, h * w, axes))
    else:
        at = positions
    with R.Device(hip) as d:
        parts, reads = [], []
        for a in x:
            vx, sx, read = d.view(a, h, w, pad=4, gap=8, before=4)
            vy, sy = vx, sx
            if place == "apart":
                vy, sy, read = d.view(np.full_like(a, np.nan), h, w, gap=4)
            parts.append(N.RotaryHeads(vx, vy, a.shape[2], sx, sy))
            reads.append(read)
        hip.rotary(handle, parts, d.ints(positions))
        got = [r() for r in reads]
    for a, y in zip(x, got):
        exp, near = R.rotate(a, at, dim, bool(inter), f, amplitude)
        np.testing.assert_array_equal(y[..., dim:], a[..., dim:])
        off, most = np.abs(y - exp), near * 2.0 ** -21
        assert (off <= most).all(), (off / np.maximum(most, 1e-30)).max()


@pytest.mark.parametrize("place", ["apart", "in place"])
@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
def test_layouts(hip, layout, place):
    run(hip, layout, 2, 3, 5, (3, 1), None, place=place)


@pytest.mark.parametrize("scaling,factor", [(N.ROTARY_LINEAR, 4.0), (N.ROTARY_BASE, 8.0), (N.ROTARY_PARTS, 16.0),
                                            (N.ROTARY_PARTS, 1.0)])
@pytest.mark.parametrize("layout", [(64, 64, 1, 0), (64, 32, 2, 1)], ids=str)
def test_scalings(hip, layout, scaling, factor):
    at = R.rng(3).integers(0, 100000, (1, 33, layout[2]))
    run(hip, layout, 1, 1, 33, (2,), at, scaling, factor, base=500000.0)


@pytest.mark.parametrize("tokens", [1, 7, 4097])
@pytest.mark.parametrize("far", [10, 1000000, 2 ** 31 - 1])
def test_positions(hip, tokens, far):
    """From one token on, positions of both signs up to the largest."""
    at = R.rng(tokens).integers(-far, far, (2, tokens, 1), endpoint=True)
    run(hip, (32, 32, 1, 0), 2, 1, tokens, (2, 2), at)


def test_many_tokens(hip):
    """Enough workgroups for the widest tile, and a last one that is not full."""
    run(hip, (32, 32, 2, 0), 3, 77, 101, (2, 2), None)


def test_queries_and_keys_of_one_tensor(hip):
    """q and k of a qkv tensor, both in place and each beside the other's heads."""
    n, h, w, heads, kd, hd = 2, 4, 6, 3, 16, 24
    per = 2 * kd + hd
    x = R.rng(5).standard_normal((n, h * w, heads, per)).astype(np.float32)
    handle = hip.rotary_create(kd, kd, 2)
    f, _ = R.frequencies(kd // 2, 10000.0, 0, 1, 1, 32, 0)
    i = np.arange(h * w)
    at = np.broadcast_to(np.stack([i // w, i % w], -1), (n, h * w, 2))
    with R.Device(hip) as d:
        v, _, read = d.view(x, h, w)
        c = (heads - 1) * per + kd
        q, k = (N.Tensor(v.data + 4 * s, n, c, h, w, v.ldc, 0) for s in (0, kd))
        hip.rotary(handle, [N.RotaryHeads(q, q, heads, per, per), N.RotaryHeads(k, k, heads, per, per)])
        got = read()
        # Outputs that meet another set's heads are refused.
        for bad in ([N.RotaryHeads(q, q, heads, per, per), N.RotaryHeads(q, k, heads, per, per)],
                    [N.RotaryHeads(q, k, heads, per, per), N.RotaryHeads(k, k, heads, per, per)],
                    [N.RotaryHeads(q, N.Tensor(v.data + 16, n, c, h, w, v.ldc, 0), heads, per, per)]):
            with pytest.raises(SyError, match="overlaps"):
                hip.rotary(handle, bad)
    np.testing.assert_array_equal(got[..., 2 * kd:], x[..., 2 * kd:])
    for s in (0, kd):
        exp, near = R.rotate(x[..., s:s + kd], at, kd, False, f, 1.0)
        assert (np.abs(got[..., s:s + kd] - exp) <= near * 2.0 ** -21).all()


def test_refusals(hip):
    handle = hip.rotary_create(32, 32)
    with R.Device(hip) as d:
        v, s, _ = d.view(np.zeros((1, 6, 2, 32), np.float32), 2, 3)
        o, _, _ = d.view(np.zeros((1, 6, 2, 32), np.float32), 2, 3)
        good = N.RotaryHeads(v, o, 2, s, s)
        for parts, match in [([], "one or two"), ([good] * 3, "one or two"),
                             ([N.RotaryHeads(v, o, 0, s, s)], "needs a head"),
                             ([N.RotaryHeads(v, o, 3, s, s)], "channels"),
                             ([N.RotaryHeads(v, o, 2, 16, s)], "stride"),
                             ([N.RotaryHeads(v, o, 2, s, 34)], "stride"),
                             ([N.RotaryHeads(v, N.Tensor(o.data, 1, 64, 3, 2, 64, 0), 2, s, s)], "differ"),
                             ([N.RotaryHeads(v, N.Tensor(o.data + 4, 1, 64, 2, 3, 64, 0), 2, s, s)], "aligned")]:
            with pytest.raises(SyError, match=match):
                hip.rotary(handle, parts)
        with pytest.raises(SyError, match="unknown rotary"):
            hip.rotary(handle + 1000, [good])
        with pytest.raises(SyError, match="unknown rotary"):
            hip.rotary(0, [good])


def test_non_finite(hip):
    """A pair with an infinity or a NaN spoils itself alone."""
    x = R.rng(2).standard_normal((1, 5, 2, 32)).astype(np.float32)
    x[0, 2, 1, 3], x[0, 4, 0, 20] = np.inf, np.nan
    handle = hip.rotary_create(32, 32)
    with R.Device(hip) as d:
        v, s, read = d.view(x, 1, 5)
        hip.rotary(handle, [N.RotaryHeads(v, v, 2, s, s)])
        got = read()
    bad = np.zeros_like(got, bool)
    bad[0, 2, 1, [3, 19]] = bad[0, 4, 0, [4, 20]] = True
    np.testing.assert_array_equal(~np.isfinite(got), bad)
