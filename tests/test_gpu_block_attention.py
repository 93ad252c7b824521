"""sy_block_attention, and rotation, means, selection and attention in a row, against float64 (bounds: _blocks.attend)."""
import numpy as np
import pytest

import _blocks as R
from simdyolo_amd import SyError
from simdyolo_amd import _native as N
from simdyolo_amd.device import HipContext

pytestmark = pytest.mark.gpu


def tensors(n, tq, t, cfg, kd, hd, seed):
    g = R.rng(seed)
    return (g.standard_normal((n, tq, cfg["heads"], kd)).astype(np.float32),
            g.standard_normal((n, t, cfg["kv_heads"], kd)).astype(np.float32),
            g.standard_normal((n, t, cfg["kv_heads"], hd)).astype(np.float32))


def choice(n, tq, cfg, h, w, seed, skew=1.0):
    """Distinct blocks in ascending order for every query, -1 behind them; blocks at the front more often."""
    g, count = R.rng(seed), R.count_blocks(cfg, h, w)
    out = np.full((n, tq, cfg["kv_heads"], cfg["selected"]), -1, np.int32)
    weight = (np.arange(count) + 1.0) ** -skew
    for i in np.ndindex(out.shape[:3]):
        k = min(cfg["selected"], count, np.count_nonzero(weight))
        out[i][:k] = np.sort(g.choice(count, k, replace=False, p=weight / weight.sum()))
    return out


def run(hip, cfg, q, k, v, blocks, h, w, qh=1, starts=None, lengths=None, scale=None, pads=True, sort=None):
    """sort: whether the pairs have to be taken as tiles of a block's queries (many queries), or one by one."""
    n, tq, heads, kd = q.shape
    hd = v.shape[-1]
    gap, before = (4, 8) if pads else (0, 0)
    with R.Device(hip) as d:
        vq, sq, _ = d.view(q, qh, tq // qh, gap=gap, before=before)
        vk, sk, _ = d.view(k, h, w, gap=2 * gap, pad=before)
        vv, sv, _ = d.view(v, h, w, gap=gap, before=gap)
        vo, _, read = d.view(np.full((n, tq, heads, hd), np.nan, np.float32), qh, tq // qh, pad=gap, before=before)
        cf = R.config(cfg, kd, hd, (sq, sk, sv), scale)
        hip.profile_enable(True)
        try:
            hip.block_attention(cf, vq, vk, vv, d.put(blocks.astype(np.int32)), vo, d.ints(starts), d.ints(lengths))
            hip.flush()
            names = set(hip.profile_read())
        finally:
            hip.profile_enable(False)
        assert names - {"block_sort"} in ({"block_attention", "block_join"}, {"block_few", "block_join"})
        assert sort is None or ("block_attention" in names) == sort
        return read()


def check(got, exp, bound):
    np.testing.assert_array_equal(np.isnan(got), np.isnan(exp))
    fine = ~np.isnan(exp)
    assert (np.abs(got - exp)[fine] <= bound[fine]).all(), (np.abs(got - exp)[fine] / np.maximum(bound[fine], 1e-30)).max()


# n, query map, key map, config, key dim, head dim, whether the pairs of query and block are sorted
CASES = [
    (1, (1, 1), (1, 1), R.shape(1, 1, 1, 1, 1), 4, 4, False),
    (1, (6, 9), (30, 22), R.shape(2, 1, 5, 3, 9), 36, 20, False),      # queries of another map
    (1, (1, 70), (1, 500), R.shape(3, 1, 1, 33, 7), 64, 128, False),   # blocks one key past a tile
    (2, (1, 5), (1, 300), R.shape(8, 2, 1, 64, 3), 128, 128, False),
    (1, (1, 2), (1, 40), R.shape(7, 1, 1, 31, 2), 80, 80, False),
    (1, (1, 3), (2, 1500), R.shape(2, 2, 2, 512, 3), 16, 8, False),    # the largest block
    (1, (1, 1), (1, 4096), R.shape(16, 2, 1, 16, 64), 64, 64, False),  # one query, the longest list
    (1, (1, 33), (1, 65), R.shape(5, 5, 1, 1, 64), 128, 4, True),      # blocks of one key
    (2, (20, 20), (20, 20), R.shape(2, 2, 4, 4, 4), 32, 64, True),
    (4, (20, 20), (20, 20), R.shape(4, 4, 4, 4, 4), 32, 64, True),     # sorted, one workgroup to a list
    (1, (15, 25), (15, 25), R.shape(4, 4, 7, 7, 6), 32, 64, True),     # windows cut on both sides
    (1, (12, 40), (12, 40), R.shape(2, 2, 8, 8, 10), 128, 128, True),  # every block of the map
    (1, (1, 900), (1, 500), R.shape(3, 1, 1, 33, 7), 64, 128, True),   # tiles that start within a query's heads
    (2, (1, 700), (1, 300), R.shape(8, 2, 1, 64, 3), 36, 20, True),
    (1, (1, 300), (2, 1500), R.shape(2, 2, 2, 512, 3), 16, 8, True),
    (1, (1, 560), (1, 30), R.shape(300, 1, 1, 4, 2), 8, 12, True),     # more heads to a key head than a tile's rows
    (1, (1, 600), (1, 90), R.shape(20, 2, 1, 8, 5), 128, 64, True),
    (1, (30, 30), (30, 30), R.shape(1, 1, 30, 30, 1), 32, 32, True),   # one block for all
    (1, (1, 800), (1, 200), R.shape(2, 2, 1, 50, 2), 100, 100, True),
]


@pytest.mark.parametrize("pads", [False, True], ids=["dense", "strided"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_shapes(hip, case, pads):
    n, (qh, qw), (h, w), cfg, kd, hd, sort = case
    q, k, v = tensors(n, qh * qw, h * w, cfg, kd, hd, h + 13 * w)
    blocks = choice(n, qh * qw, cfg, h, w, 3)
    exp, bound = R.attend(cfg, q, k, v, blocks, h, w, kd ** -0.5)
    check(run(hip, cfg, q, k, v, blocks, h, w, qh, pads=pads, sort=sort), exp, bound)


@pytest.mark.parametrize("skew", [0.0, 6.0])
def test_long_and_short_lists(hip, skew):
    """Blocks that every query chooses, and blocks that none does."""
    cfg, kd, hd, h, w = R.shape(2, 2, 4, 4, 3), 16, 16, 24, 24
    q, k, v = tensors(1, h * w, h * w, cfg, kd, hd, 4)
    blocks = choice(1, h * w, cfg, h, w, 5, skew)
    if skew == 0.0:
        blocks[:] = [0, 7, 35]
    exp, bound = R.attend(cfg, q, k, v, blocks, h, w, kd ** -0.5)
    check(run(hip, cfg, q, k, v, blocks, h, w, h, sort=True), exp, bound)


@pytest.mark.parametrize("tq", [1, 3, 150])
@pytest.mark.parametrize("starts", [None, (0, 100, -2, 130)], ids=str)
@pytest.mark.parametrize("lengths", [None, (0, 1, 150, 77)], ids=str)
def test_causal(hip, tq, starts, lengths):
    cfg, kd, hd, w = R.shape(4, 2, 1, 16, 4, causal=1), 32, 64, 150
    q, k, v = tensors(4, tq, w, cfg, kd, hd, 21)
    blocks = choice(4, tq, cfg, 1, w, 6, 0.5)
    blocks[:, :, :, 3] = (np.maximum(np.asarray(starts or [0] * 4), 0)[:, None, None] + np.arange(tq)[:, None]) // 16
    exp, bound = R.attend(cfg, q, k, v, blocks, 1, w, kd ** -0.5, starts, lengths)
    got = run(hip, cfg, q, k, v, blocks, 1, w, 1, starts, lengths, sort=tq == 150)
    check(got, exp, bound)
    assert lengths is None or not got[0].any()


@pytest.mark.parametrize("tq", [1, 80])
def test_lists(hip, tq):
    """No block, blocks out of range, gaps and repeats (which count again)."""
    cfg, kd, hd, w = R.shape(2, 2, 1, 10, 6), 16, 24, 95
    q, k, v = tensors(2, tq, w, cfg, kd, hd, 2)
    blocks = choice(2, tq, cfg, 1, w, 8)
    blocks[0, :, 0] = -1
    blocks[1, :, 0] = [10, -7, 2 ** 31 - 1, -2 ** 31, 11, 3]
    blocks[1, :, 1] = [4, 4, -1, 9, 4, 9]
    exp, bound = R.attend(cfg, q, k, v, blocks, 1, w, kd ** -0.5)
    got = run(hip, cfg, q, k, v, blocks, 1, w, sort=tq == 80)
    check(got, exp, bound)
    assert not got[0, :, 0].any() and got[1, :, 0].any()


@pytest.mark.parametrize("tq", [1, 300])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf, np.finfo(np.float32).max, 2.0 ** 60], ids=str)
def test_hidden_keys_are_not_read(hip, tq, value):
    """Whatever stands behind a sequence, behind a causal query, in blocks not chosen."""
    cfg, kd, hd, w = R.shape(4, 2, 1, 16, 3, causal=1), 32, 32, 90
    lengths, starts = (40, 70), (40 - tq if tq == 1 else 0, 70 - tq if tq == 1 else 0)
    q, k, v = tensors(2, tq, w, cfg, kd, hd, 2)
    blocks = choice(2, tq, cfg, 1, w, 8, 0.0)
    blocks[blocks == 1] = 0
    exp, bound = R.attend(cfg, q, k, v, blocks, 1, w, kd ** -0.5, starts, lengths)
    k[:, 16:32], v[:, 16:32] = value, value
    for b in range(2):
        k[b, lengths[b]:], v[b, lengths[b]:] = value, value
    got = run(hip, cfg, q, k, v, blocks, 1, w, 1, starts, lengths, sort=tq == 300)
    check(got, exp, bound)


@pytest.mark.parametrize("tq", [1, 700])
@pytest.mark.parametrize("part", ["q", "k", "v"])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf], ids=str)
def test_non_finite(hip, tq, part, value):
    """What one of them spoils is as in the formula, and no more."""
    cfg, kd, hd, w = R.shape(2, 1, 1, 20, 2), 32, 36, 100
    q, k, v = tensors(1, tq, w, cfg, kd, hd, 2)
    {"q": q, "k": k, "v": v}[part][0, 0 if part == "q" else 33, 0, 5] = value
    blocks = choice(1, tq, cfg, 1, w, 8, 0.0)
    blocks[0, 0, 0] = [1, 3]
    with np.errstate(invalid="ignore", over="ignore"):
        exp, bound = R.attend(cfg, q, k, v, blocks, 1, w, kd ** -0.5)
    got = run(hip, cfg, q, k, v, blocks, 1, w, sort=tq == 700)
    np.testing.assert_array_equal(np.isfinite(got), np.isfinite(exp))
    np.testing.assert_array_equal(np.isnan(got), np.isnan(exp))
    fine = np.isfinite(exp) & np.isfinite(bound)
    assert (np.abs(got[fine] - exp[fine]) <= bound[fine]).all()


@pytest.mark.parametrize("tq", [1, 400])
def test_scores_that_are_all_minus_infinite(hip, tq):
    """The formula's 0 / 0; where one score is finite, the others weigh nothing."""
    cfg, kd, hd, w = R.shape(2, 2, 1, 20, 3), 8, 8, 100
    q, k, v = tensors(1, tq, w, cfg, kd, hd, 2)
    q[..., 0] = 1.0
    k[:, :, 0, 0] = -np.inf
    k[:, :99, 1, 0] = -np.inf
    blocks = choice(1, tq, cfg, 1, w, 8, 0.0)
    blocks[..., 2] = 4
    exp, bound = R.attend(cfg, q, k, v, blocks, 1, w, kd ** -0.5)
    assert np.isnan(exp[:, :, 0]).all() and np.isfinite(exp[:, :, 1]).all()
    got = run(hip, cfg, q, k, v, blocks, 1, w, sort=tq == 400)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(exp))
    check(got[:, :, 1:], exp[:, :, 1:], np.abs(exp[:, :, 1:]) * 2.0 ** -16)


@pytest.mark.parametrize("tq", [1, 300])
@pytest.mark.parametrize("scales", [(1e-6, 1e6, 1e-20), (30.0, 1.0, 1e4), (0.0, 1.0, 1.0), (1e-30, 1e-30, 1e-30),
                                    (1.0, 1.0, 1e30), (1e-30, 1e30, 1.0), (1.0, 1.0, 1e-37), (1e35, 1e-36, 1e-44)], ids=str)
def test_operand_scales(hip, tq, scales):
    """Operands of far apart magnitudes, subnormal ones; values that grow by 2^14 from block to block."""
    cfg, kd, hd, w = R.shape(2, 2, 1, 16, 4), 32, 64, 96
    q, k, v = (a * np.float32(s) for a, s in zip(tensors(1, tq, w, cfg, kd, hd, 5), scales))
    v[:, 48:] *= np.float32(16384)
    blocks = choice(1, tq, cfg, 1, w, 8, 0.0)
    exp, bound = R.attend(cfg, q, k, v, blocks, 1, w, kd ** -0.5)
    check(run(hip, cfg, q, k, v, blocks, 1, w, sort=tq == 300), exp, bound + 2.0 ** -126)


@pytest.mark.parametrize("tq", [1, 300])
@pytest.mark.parametrize("part", ["k", "v"])
@pytest.mark.parametrize("step", [0.7, 3.0, 40.0])
def test_keys_of_many_sizes(hip, tq, part, step):
    """Keys, or values, that grow by e^step from one to the next within a block: beside, past and far past the range
    within which they share a power of two."""
    cfg, kd, hd, w = R.shape(2, 2, 1, 32, 3, causal=1), 32, 64, 96
    q, k, v = tensors(1, tq, w, cfg, kd, hd, 5)
    grow = np.exp(np.minimum(step * (np.arange(w) % 32), 80.0) - 40.0).astype(np.float32)[:, None, None]
    if part == "k":
        k, q = k * grow, q * np.float32(1e-17)
    else:
        v = v * grow
    blocks = choice(1, tq, cfg, 1, w, 8, 0.0)
    exp, bound = R.attend(cfg, q, k, v, blocks, 1, w, kd ** -0.5)
    check(run(hip, cfg, q, k, v, blocks, 1, w, sort=tq == 300), exp, bound)


@pytest.mark.parametrize("tq", [1, 700])
def test_heavy_key_in_a_light_block(hip, tq):
    """A key with values of 2^20 and no weight beside ordinary ones: their precision is their own."""
    cfg, kd, hd, w = R.shape(1, 1, 1, 32, 2), 32, 64, 96
    q, k, v = tensors(1, tq, w, cfg, kd, hd, 5)
    q[..., 0], k[..., 0] = 40.0, 0.0
    k[:, 40, 0, 0] = -40.0
    v[:, 40] *= np.float32(2.0 ** 20)
    blocks = choice(1, tq, cfg, 1, w, 8, 0.0)
    blocks[..., 1] = np.maximum(blocks[..., 1], 1)
    blocks[..., 0] = 0
    exp, bound = R.attend(cfg, q, k, v, blocks, 1, w, kd ** -0.5)
    check(run(hip, cfg, q, k, v, blocks, 1, w, sort=tq == 700), exp, bound)


@pytest.mark.parametrize("step", [0.5, 3.0, 60.0, -60.0])
def test_creeping_maximum(hip, step):
    """Scores that rise or fall from one tile of keys to the next."""
    cfg, kd, hd, w = R.shape(1, 1, 1, 200, 3), 32, 64, 600
    for tq in (1, 150):
        q, k, v = tensors(1, tq, w, cfg, kd, hd, 8)
        q[:] = 1.0
        k *= np.float32(0.25)
        k[..., 0] += (np.float32(step) * (np.arange(w) // 32)).astype(np.float32)[:, None]
        blocks = choice(1, tq, cfg, 1, w, 8, 0.0)
        exp, bound = R.attend(cfg, q, k, v, blocks, 1, w, 1.0)
        check(run(hip, cfg, q, k, v, blocks, 1, w, scale=1.0, sort=tq == 150), exp, bound)


def test_neighbours_do_not_change_a_row(hip):
    """The same query among others, at other places of a list and alone: the same bits."""
    cfg, kd, hd, h, w = R.shape(4, 2, 4, 4, 3), 32, 64, 16, 24
    q, k, v = tensors(1, h * w, h * w, cfg, kd, hd, 4)
    blocks = choice(1, h * w, cfg, h, w, 5)
    whole = run(hip, cfg, q, k, v, blocks, h, w, h, sort=True)
    np.testing.assert_array_equal(whole, run(hip, cfg, q, k, v, blocks, h, w, h))
    turn = R.rng(3).permutation(h * w)
    moved = run(hip, cfg, np.ascontiguousarray(q[:, turn]), k, v, np.ascontiguousarray(blocks[:, turn]), h, w, h)
    np.testing.assert_array_equal(moved, whole[:, turn])


@pytest.mark.parametrize("tq,cfg,w,dim,sort", [(40000, R.shape(2, 2, 1, 2, 64), 400, 128, True),
                                               (140000, R.shape(1, 1, 1, 1, 64), 13000, 4, False)], ids=["sorted", "few"])
def test_more_results_than_one_launch_holds(hip, tq, cfg, w, dim, sort):
    """1.34 GB of results for each head, in two launches; 9.0 million pairs of query and block, in two."""
    q, k, v = tensors(1, tq, w, cfg, 32, dim, 9)
    g, count = R.rng(10), R.count_blocks(cfg, 1, w)
    blocks = (g.integers(0, count, (1, tq, cfg["kv_heads"], 1)) + np.arange(64) * 3) % count
    got = run(hip, cfg, q, k, v, blocks, 1, w, pads=False, sort=sort)
    assert np.isfinite(got).all()
    keep = np.unique(np.concatenate([[0, tq - 1], g.integers(0, tq, 200), np.arange(tq // 2 - 20, tq // 2 + 20)]))
    exp, bound = R.attend(cfg, q[:, keep], k, v, blocks[:, keep], 1, w, 32 ** -0.5)
    check(got[:, keep], exp, bound)


@pytest.mark.parametrize("tq,sort", [(3, False), (4000, True)])
def test_offsets_past_32_bits(hip, tq, sort):
    """A cache whose last keys lie 17 GB behind its first: rotation in place, means of the last block, selection and
    attention there."""
    cfg, kd, hd, w, ldc, last = R.shape(4, 2, 1, 128, 4, causal=1), 32, 64, (1 << 20) + 6400, 4160, 6400
    _, k, v = tensors(1, 1, last, cfg, kd, hd, 21)
    q = R.rng(22).standard_normal((1, tq, 4, kd)).astype(np.float32)
    blocks, tail = w // 128, last // 128
    with R.Device(hip) as d:
        base = hip.malloc(4 * w * ldc)
        d.ptrs.append(base)
        slab = np.zeros((last, ldc), np.float32)
        slab[:, :64], slab[:, 64:192] = k[0].reshape(last, 64), v[0].reshape(last, 128)
        end = base + 4 * ldc * (w - last)
        hip.h2d(end, slab)
        vk, vv = N.Tensor(base, 1, 64, 1, w, ldc, 0), N.Tensor(base + 256, 1, 128, 1, w, ldc, 0)
        hip.rotary(hip.rotary_create(kd, kd), [N.RotaryHeads(vk, vk, 2, 0, 0)])
        hip.flush()
        rk = hip.d2h(end, (last, ldc))[:, :64].reshape(1, last, 2, kd)
        f, _ = R.frequencies(kd, 10000.0, 0, 1, 1, 32, 0)
        exp, near = R.rotate(k, np.arange(w - last, w).reshape(1, last, 1), kd, False, f, 1.0)
        assert (np.abs(rk - exp) <= near * 2.0 ** -21).all()
        m = np.zeros((1, blocks, 2, kd), np.float32)
        m[:, -tail:] = R.means(cfg, rk, 1, last)  # in front of them: zeros
        vm, _, read_m = d.view(m.reshape(1, blocks, 1, 64), 1, blocks)
        at = d.ints([w - tq])
        cf = R.config(cfg, kd, hd)
        hip.h2d(vm.data + 4 * 64 * (blocks - tail), np.full((tail, 64), np.nan, np.float32))
        hip.block_means(cf, vk, vm, d.ints([w - last]), last)
        got_m = read_m().reshape(1, blocks, 2, kd)
        assert (np.abs(got_m - m)[:, -tail:] <= np.abs(m)[:, -tail:] * 2.0 ** -23 + np.abs(rk).max() * 2.0 ** -45).all()
        vq, _, _ = d.view(q, 1, tq)
        lists = d.put(np.zeros((1, tq, 2, 4), np.int32))
        hip.block_select(cf, vq, vm, lists, at)
        chosen = hip.d2h(lists, (1, tq, 2, 4), np.int32)
        np.testing.assert_array_equal(chosen[:, ::37], np.concatenate(
            [R.select(cfg, q[:, i:i + 1], got_m, [w - tq + i]) for i in range(0, tq, 37)], 1))
        near_end = np.maximum(chosen, blocks - tail)  # blocks whose keys were written; named twice they count twice
        vo, _, read = d.view(np.full((1, tq, 4, hd), np.nan, np.float32), 1, tq)
        hip.profile_enable(True)
        try:
            hip.block_attention(cf, vq, vk, vv, d.put(near_end), vo, at)
            hip.flush()
            assert ("block_sort" in hip.profile_read()) == sort
        finally:
            hip.profile_enable(False)
        exp, bound = R.attend(cfg, q, rk, v, near_end - (blocks - tail), 1, last, kd ** -0.5, [last - tq])
        check(read(), exp, bound)


# ------------------------------------------------------------------ in a row

class Chain:
    """Rotation, means, selection and attention on one qkv tensor, as a block of a network runs them."""

    def __init__(self, hip, d, n, h, w, cfg, kd, hd, seed, x=None):
        self.hip, self.cfg, self.kd, self.hd, self.h, self.w, self.n = hip, cfg, kd, hd, h, w, n
        heads = cfg["heads"]
        per = 2 * kd + hd
        self.x = R.rng(seed).standard_normal((n, h * w, heads, per)).astype(np.float32) if x is None else x
        self.view, _, _ = d.view(self.x, h, w)
        c = (heads - 1) * per

        def part(at, dim):
            return N.Tensor(self.view.data + 4 * at, n, c + dim, h, w, self.view.ldc, 0)
        self.q, self.k, self.v = part(0, kd), part(kd, kd), part(2 * kd, hd)
        empty = np.full((n, h * w, heads, kd), np.nan, np.float32)
        self.rq, _, self.read_q = d.view(empty, h, w)
        self.rk, _, self.read_k = d.view(empty, h, w)
        self.o, _, self.read_o = d.view(np.full((n, h * w, heads, hd), np.nan, np.float32), h, w)
        by, bx = -(-h // cfg["block_h"]), -(-w // cfg["block_w"])
        self.m, _, self.read_m = d.view(np.zeros((n, by * bx, 1, heads * kd), np.float32), by, bx)
        self.list_shape = (n, h * w, heads, cfg["selected"])
        self.list = d.put(np.zeros(self.list_shape, np.int32))
        self.rotary = hip.rotary_create(kd, kd, 2)
        self.cfg_q = R.config(cfg, kd, hd, (0, 0, per))
        self.per = per

    def __call__(self):
        hip, heads = self.hip, self.cfg["heads"]
        hip.rotary(self.rotary, [N.RotaryHeads(self.q, self.rq, heads, self.per, 0),
                                 N.RotaryHeads(self.k, self.rk, heads, self.per, 0)])
        hip.block_means(self.cfg_q, self.rk, self.m)
        hip.block_select(self.cfg_q, self.rq, self.m, self.list)
        hip.block_attention(self.cfg_q, self.rq, self.rk, self.v, self.list, self.o)

    def check(self):
        got = self.read_o()
        q, k, m = self.read_q(), self.read_k(), self.read_m()
        blocks = self.hip.d2h(self.list, self.list_shape, np.int32)
        f, _ = R.frequencies(self.kd // 2, 10000.0, 0, 1, 1, 32, 0)
        i = np.arange(self.h * self.w)
        at = np.broadcast_to(np.stack([i // self.w, i % self.w], -1), (self.n, i.size, 2))
        for a, b in ((q, self.x[..., :self.kd]), (k, self.x[..., self.kd:2 * self.kd])):
            exp, near = R.rotate(b, at, self.kd, False, f, 1.0)
            assert (np.abs(a - exp) <= near * 2.0 ** -21).all()
        m = m.reshape(self.n, -1, self.cfg["heads"], self.kd)
        exp = R.means(self.cfg, k, self.h, self.w)
        assert (np.abs(m - exp) <= np.abs(exp) * 2.0 ** -24 + np.abs(k).max() * 2.0 ** -45).all()
        np.testing.assert_array_equal(blocks, R.select(self.cfg, q, m))
        exp, bound = R.attend(self.cfg, q, k, self.x[..., 2 * self.kd:], blocks, self.h, self.w, self.kd ** -0.5)
        check(got, exp, bound)
        return got


def test_chain(hip):
    with R.Device(hip) as d:
        c = Chain(hip, d, 2, 13, 22, R.shape(2, 2, 4, 4, 5), 32, 64, 3)
        c()
        c.check()


def test_chain_captured(hip):
    """Two graphs of one context, replayed in turn with eager calls between them, on inputs that change."""
    with HipContext(0) as ctx, R.Device(ctx) as d:
        chains = [Chain(ctx, d, n, h, w, cfg, 32, 64, 3 + h) for n, h, w, cfg in
                  ((1, 20, 20, R.shape(2, 2, 4, 4, 4)), (2, 9, 14, R.shape(2, 2, 3, 3, 6)))]
        for c in chains:
            c()
        expected = [c.check() for c in chains]
        graphs = []
        for c in chains:
            ctx.graph_begin()
            c()
            graphs.append(ctx.graph_end())
        for turn in range(4):
            for c, g, e in zip(chains, graphs, expected):
                ctx.h2d(c.list, np.full(c.list_shape, -1, np.int32))
                ctx.graph_launch(g)
                if turn % 2:
                    chains[1]()  # eager work in between
                np.testing.assert_array_equal(c.read_o(), e)
        with R.Device(ctx) as e:
            other = Chain(ctx, e, 1, 20, 20, chains[0].cfg, 32, 64, 77)
            other()
            other.check()
            ctx.h2d(chains[0].view.data, other.x)
            chains[0].x = other.x
            ctx.graph_launch(graphs[0])
            chains[0].check()


def test_two_contexts_in_turn():
    """Calls on two contexts' streams without a wait between them."""
    with HipContext(0) as a, HipContext(0) as b, R.Device(a) as da, R.Device(b) as db:
        chains = [Chain(x, d, 1, 17, 18, R.shape(2, 2, 4, 4, 4), 32, 64, s) for x, d, s in ((a, da, 1), (b, db, 2))]
        for _ in range(3):
            for c in chains:
                c()
        for c in chains:
            c.check()


def test_token_by_token(hip):
    """A sequence that grows: means renewed, blocks selected and attended to for one token at a time give what
    the whole sequence gives at once (up to the tolerance of either)."""
    cfg, kd, hd, w = R.shape(4, 2, 1, 8, 3, causal=1), 32, 32, 43
    q, k, v = tensors(2, w, w, cfg, kd, hd, 12)
    cf = R.config(cfg, kd, hd)
    with R.Device(hip) as d:
        vk, _, _ = d.view(k, 1, w)
        vv, _, _ = d.view(v, 1, w)
        bx = -(-w // 8)
        m, _, _ = d.view(np.full((2, bx, 1, 2 * kd), np.nan, np.float32), 1, bx)
        out = np.zeros((2, w, 4, hd), np.float32)
        lists = np.zeros((2, w, 2, 3), np.int32)
        for t in range(w):
            s, ln = d.ints([t, t]), d.ints([t + 1, t + 1])
            vq, _, _ = d.view(q[:, t:t + 1], 1, 1)
            vo, _, read = d.view(np.full((2, 1, 4, hd), np.nan, np.float32), 1, 1)
            p = d.put(np.zeros((2, 1, 2, 3), np.int32))
            hip.block_means(cf, vk, m, s, 1, ln)
            hip.block_select(cf, vq, m, p, s, ln)
            hip.block_attention(cf, vq, vk, vv, p, vo, s, ln)
            out[:, t:t + 1] = read()
            lists[:, t:t + 1] = hip.d2h(p, (2, 1, 2, 3), np.int32)
    exp, bound = R.attend(cfg, q, k, v, lists, 1, w, kd ** -0.5)
    check(out, exp, bound)
    whole = run(hip, cfg, q, k, v, lists, 1, w, pads=False)
    check(whole, exp, bound)


def test_lists_of_each_launch(hip):
    """Five sequences of 0.31 GB of results each: three and two to a launch, which sorts its own pairs."""
    cfg, n, tq, dim = R.shape(1, 1, 1, 16, 30, causal=1), 5, 20000, 128
    lengths, starts = (20000, 19000, 5, 20000, 12345), (0, -700, 10, 0, 60)
    q, k, v = tensors(n, tq, tq, cfg, dim, dim, 9)
    g = R.rng(10)
    last = np.clip((np.asarray(starts)[:, None, None, None] + np.arange(tq)[:, None, None]) // 16, 0, 1249)
    blocks = np.minimum(g.integers(0, 1250, (n, tq, 1, 30)), last).astype(np.int32)
    got = run(hip, cfg, q, k, v, blocks, 1, tq, 1, starts, lengths, pads=False, sort=True)
    assert np.isfinite(got).all()
    for b in range(n):
        for i in np.unique(np.r_[0, 1, tq - 1, g.integers(0, tq, 25)]):
            one = slice(b, b + 1)
            check(got[one, i:i + 1], *R.attend(cfg, q[one, i:i + 1], k[one], v[one], blocks[one, i:i + 1], 1, tq, dim ** -0.5,
                                               [starts[b] + i], [lengths[b]]))
