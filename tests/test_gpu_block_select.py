"""sy_block_means and sy_block_select against float64.

A mean is a sum in 64 bits rounded once to float32: within 2^-24 of itself and 2^-45 of the keys' magnitudes.  The
selection, on the means that the device holds, is exact."""
import numpy as np
import pytest

import _blocks as R
from simdyolo_amd import SyError, Tensor
from simdyolo_amd import _native as N

pytestmark = pytest.mark.gpu

# n, h, w, config, key dim
MAPS = [(1, 1, 1, R.shape(1, 1, 1, 1, 1), 4), (2, 20, 20, R.shape(2, 2, 4, 4, 4), 32),
        (1, 15, 25, R.shape(4, 2, 7, 7, 6), 36), (3, 9, 31, R.shape(6, 2, 3, 5, 64), 128),
        (1, 40, 70, R.shape(8, 8, 1, 1, 12), 16), (1, 2, 3000, R.shape(2, 1, 2, 1024 // 2, 3), 8),
        (2, 33, 40, R.shape(3, 3, 2, 3, 5), 80)]


def tensors(n, t, tq, cfg, kd, seed):
    g = R.rng(seed)
    return (g.standard_normal((n, tq, cfg["heads"], kd)).astype(np.float32),
            g.standard_normal((n, t, cfg["kv_heads"], kd)).astype(np.float32))


def means_view(d, cfg, n, h, w, kd, a=None):
    """A means view (kv_heads * key_dim channels side by side) and its reader."""
    by, bx = -(-h // cfg["block_h"]), -(-w // cfg["block_w"])
    if a is None:
        a = np.full((n, by * bx, cfg["kv_heads"] * kd), np.nan, np.float32)
    v, _, read = d.view(a.reshape(n, by * bx, 1, -1), by, bx, pad=4, before=4)
    return v, lambda: read().reshape(n, by * bx, cfg["kv_heads"], kd)


def close(got, exp, k):
    assert (np.abs(got - exp) <= np.abs(exp) * 2.0 ** -24 + np.abs(k).max() * 2.0 ** -45).all()


# Few queries are ranked as they are, many (2,048 and more pairs of query and key head, or 64 blocks and less) through
# the matrix cores; of many, some are compared.
FEW, MANY = 21, 2100


def some(q, *more):
    keep = np.unique(R.rng(1).permutation(q.shape[1])[:90])
    return [np.ascontiguousarray(a[:, keep]) for a in (q, *more)]


def run_select(hip, cfg, q, m, h, w, starts=None, lengths=None, qh=None, gap=0, many=None):
    """Selection on the means m [n, blocks, kv, kd]; many: whether through the matrix cores."""
    n, tq, _, kd = q.shape
    with R.Device(hip) as d:
        vq, sq, _ = d.view(q, qh or 1, tq // (qh or 1), pad=8, gap=gap, before=4)
        vm, _ = means_view(d, cfg, n, h, w, kd, m)
        out = np.full((n, tq, cfg["kv_heads"], cfg["selected"]), 77, np.int32)
        p = d.put(out)
        hip.profile_enable(True)
        try:
            hip.block_select(R.config(cfg, kd, 4, (sq, 0, 0)), vq, vm, p, d.ints(starts), d.ints(lengths))
            hip.flush()
            names = set(hip.profile_read())
        finally:
            hip.profile_enable(False)
        assert names in ({"block_score", "block_rank"}, {"block_parts", "block_select"}, {"block_select"})
        assert many is None or ("block_select" in names) == many
        return hip.d2h(p, out.shape, np.int32)


@pytest.mark.parametrize("case", MAPS, ids=str)
def test_maps(hip, case):
    n, h, w, cfg, kd = case
    q, k = tensors(n, h * w, h * w, cfg, kd, 7 * h + w)
    with R.Device(hip) as d:
        vk, sk, _ = d.view(k, h, w, gap=4, before=8)
        vm, read = means_view(d, cfg, n, h, w, kd)
        hip.block_means(R.config(cfg, kd, 4, (0, sk, 0)), vk, vm)
        m = read()
    close(m, R.means(cfg, k, h, w), k)
    keep = R.rng(1).permutation(h * w)[:100]  # a query's choice does not hang on the others
    got = run_select(hip, cfg, q, m, h, w, qh=h, gap=4)
    exp = R.select(cfg, np.ascontiguousarray(q[:, keep]), m)
    np.testing.assert_array_equal(got[:, keep], exp)


@pytest.mark.parametrize("kd", [32, 128])
@pytest.mark.parametrize("starts", [None, (0, 5, -3, 200, 2 ** 31 - 300)], ids=str)
@pytest.mark.parametrize("lengths", [None, (0, 1, 64, 250, 1000), (-5, 299, 300, 17, 128)], ids=str)
def test_causal(hip, kd, starts, lengths):
    """Rows with empty, partial and overlong sequences; queries before, in and far behind the keys."""
    n, w, tq, cfg = 5, 300, 261, R.shape(4, 2, 1, 16, 5, causal=1)
    q, k = tensors(n, w, tq, cfg, kd, 3)
    with R.Device(hip) as d:
        vk, _, _ = d.view(k, 1, w)
        vm, read = means_view(d, cfg, n, 1, w, kd)
        hip.block_means(R.config(cfg, kd, 4), vk, vm, lengths=d.ints(lengths))
        m = read()
    close(m, R.means(cfg, k, 1, w, lengths), k)
    got = run_select(hip, cfg, q, m, 1, w, starts, lengths)
    np.testing.assert_array_equal(got, R.select(cfg, q, m, starts, lengths))


def test_lengths_without_causal(hip):
    n, w, cfg, kd, lengths = 4, 100, R.shape(4, 4, 1, 8, 3), 16, (0, 8, 9, 100)
    q, k = tensors(n, w, 37, cfg, kd, 11)
    m = R.means(cfg, k, 1, w, lengths).astype(np.float32)
    got = run_select(hip, cfg, q, m, 1, w, None, lengths)
    np.testing.assert_array_equal(got, R.select(cfg, q, m, None, lengths))


def test_keys_behind_the_length_do_not_count(hip):
    n, w, cfg, kd, lengths = 2, 50, R.shape(2, 2, 1, 16, 2), 8, (20, 33)
    _, k = tensors(n, w, 1, cfg, kd, 2)
    exp = R.means(cfg, k, 1, w, lengths)
    for b in range(n):
        k[b, lengths[b]:] = np.nan
    with R.Device(hip) as d:
        vk, _, _ = d.view(k, 1, w)
        vm, read = means_view(d, cfg, n, 1, w, kd)
        hip.block_means(R.config(cfg, kd, 4), vk, vm, lengths=d.ints(lengths))
        got = read()
    close(got, exp, k[:, :20])


@pytest.mark.parametrize("starts,tokens", [((0, 15, 16, 60, 63), 1), ((-3, 15, 31, 47, 62), 2), ((-9, 0, 20, 49, 63), 40),
                                           (None, 17), ((1000, -2 ** 31, 2 ** 31 - 1, 64, 0), 5)], ids=str)
def test_renewed_means(hip, starts, tokens):
    """Only the blocks that hold new tokens are written, wherever those stand."""
    n, w, cfg, kd = 5, 64, R.shape(2, 2, 1, 16, 2), 20
    lengths = [64 if starts is None else min(64, max(1, s + tokens)) for s in (starts or [0] * 5)]
    _, k = tensors(n, w, 1, cfg, kd, 9)
    old = R.rng(4).standard_normal((n, 4, 2, kd)).astype(np.float32)
    with R.Device(hip) as d:
        vk, _, _ = d.view(k, 1, w)
        vm, read = means_view(d, cfg, n, 1, w, kd, old)
        hip.block_means(R.config(cfg, kd, 4), vk, vm, d.ints(starts), tokens, d.ints(lengths))
        got = read()
    exp = R.means(cfg, k, 1, w, lengths)
    for b in range(n):
        s = 0 if starts is None else starts[b]
        for j in range(4):
            if j * 16 < s + tokens and s < (j + 1) * 16:
                close(got[b, j], exp[b, j], k)
            else:
                np.testing.assert_array_equal(got[b, j], old[b, j])


@pytest.mark.parametrize("tq", [FEW, MANY])
@pytest.mark.parametrize("blocks", [3, 70, 1500])
@pytest.mark.parametrize("selected", [1, 8, 13, 30, 64])
def test_ties_and_non_finite_means(hip, tq, blocks, selected):
    """Equal means: the lower block.  NaN scores come last, infinities at the ends."""
    cfg, kd = R.shape(2, 2, 1, 1, selected), 12
    q, _ = tensors(2, 1, tq, cfg, kd, 5)
    m = np.round(R.rng(6).standard_normal((2, blocks, 2, kd)) * 2).astype(np.float32)
    m[:, 1::3] = m[:, :1]

    def compare():
        got = run_select(hip, cfg, q, m, 1, blocks, many=tq == MANY or blocks <= 64)
        few, got = some(q, got)
        np.testing.assert_array_equal(got, R.select(cfg, few, m))
    compare()
    m[0, blocks // 2, :, 3] = np.nan
    m[1, blocks // 3, 0, 2] = np.inf
    m[1, blocks // 4, 1, 2] = -np.inf
    compare()
    m[:] = np.nan
    compare()


@pytest.mark.parametrize("tq", [FEW, MANY])
@pytest.mark.parametrize("kd,selected", [(64, 6), (32, 16), (128, 40)])
def test_near_ties(hip, tq, kd, selected):
    """Scores that differ by less than float32 could tell: blocks that differ in the last bit of one channel, all of
    them (a query's candidates do not fit anywhere) or a few near the border."""
    cfg, blocks = R.shape(4, 1, 1, 1, selected), 200
    q, _ = tensors(1, 1, tq, cfg, kd, 8)
    near = np.repeat(R.rng(3).standard_normal((1, 1, 1, kd)), blocks, 1).astype(np.float32)
    at = R.rng(4).integers(0, kd, blocks)
    for j in range(blocks):
        near[0, j, 0, at[j]] = np.nextafter(near[0, j, 0, at[j]], np.float32(np.inf if j % 2 else -np.inf))
    apart = R.rng(9).standard_normal((1, blocks, 1, kd)).astype(np.float32)
    for m in (near, np.where((np.arange(blocks) % 9 < 3)[:, None, None], near, apart)):
        got = run_select(hip, cfg, q, m, 1, blocks, many=tq == MANY)
        few, got = some(q, got)
        np.testing.assert_array_equal(got, R.select(cfg, few, m))


@pytest.mark.parametrize("tq", [FEW, MANY])
def test_pairs_of_blocks_that_are_alike(hip, tq):
    """Every block has a neighbour 2^-20 away: many queries of one wave are in doubt between two."""
    cfg, kd, blocks = R.shape(2, 2, 1, 1, 7), 48, 300
    q, _ = tensors(1, 1, tq, cfg, kd, 8)
    m = R.rng(3).standard_normal((1, blocks, 2, kd)).astype(np.float32)
    m[:, 1::2] = m[:, ::2] * np.float32(1 + 2.0 ** -20)
    got = run_select(hip, cfg, q, m, 1, blocks, many=tq == MANY)
    few, got = some(q, got)
    np.testing.assert_array_equal(got, R.select(cfg, few, m))


@pytest.mark.parametrize("kd,selected", [(32, 7), (32, 16), (64, 5), (128, 12)])
def test_pairs_in_many_heads(hip, kd, selected):
    """The same with so many heads that their means are laid out first; one head's hold NaN."""
    cfg, tq, blocks = R.shape(40, 20, 1, 1, selected), 1900, 300
    q, _ = tensors(1, 1, tq, cfg, kd, 8)
    m = R.rng(3).standard_normal((1, blocks, 20, kd)).astype(np.float32)
    m[:, 1::2] = m[:, ::2] * np.float32(1 + 2.0 ** -20)
    m[0, 17, 3, 1] = np.nan
    got = run_select(hip, cfg, q, m, 1, blocks, many=True)
    few, got = some(q, got)
    np.testing.assert_array_equal(got, R.select(cfg, few, m))


@pytest.mark.parametrize("blocks", [4096, 4097])
@pytest.mark.parametrize("kd,selected", [(32, 5), (64, 16), (128, 8), (128, 16), (32, 33)])
def test_many_blocks(hip, blocks, kd, selected):
    """Up to and past the blocks whose numbers fit into their scores; pairs of them 2^-18 apart."""
    cfg = R.shape(2, 1, 1, 1, selected)
    q, _ = tensors(1, 1, MANY, cfg, kd, 8)
    m = R.rng(3).standard_normal((1, blocks, 1, kd)).astype(np.float32)
    m[:, 1::2] = m[:, :blocks // 2 * 2:2] * np.float32(1 + 2.0 ** -18)
    got = run_select(hip, cfg, q, m, 1, blocks, many=True)
    few, got = some(q, got)
    np.testing.assert_array_equal(got, R.select(cfg, few, m))


@pytest.mark.parametrize("tq", [FEW, MANY])
@pytest.mark.parametrize("selected", [1, 8, 16])
def test_negative_and_tiny_scores(hip, tq, selected):
    """No score above zero, and blocks with scores of zero or far below the others' among them."""
    cfg, kd, blocks = R.shape(2, 2, 1, 1, selected), 40, 333
    q, _ = tensors(1, 1, tq, cfg, kd, 8)
    q, m = np.abs(q), -np.abs(R.rng(3).standard_normal((1, blocks, 2, kd))).astype(np.float32)
    m[:, ::60] = 0
    m[:, 1::70] *= np.float32(2.0 ** -120)
    got = run_select(hip, cfg, q, m, 1, blocks, many=tq == MANY)
    few, got = some(q, got)
    np.testing.assert_array_equal(got, R.select(cfg, few, m))


@pytest.mark.parametrize("tq", [FEW, MANY])
@pytest.mark.parametrize("scales", [(1e-30, 1e-12), (1e25, 1e20), (1e-42, 1.0), (0.0, 1.0), (1.0, 0.0), (1e12, 1e-12)], ids=str)
def test_far_scaled(hip, tq, scales):
    """Products below float32's range, above it, of subnormal queries, of zeros."""
    cfg, kd, blocks = R.shape(2, 2, 1, 1, 5), 32, 90
    q, _ = tensors(2, 1, tq, cfg, kd, 8)
    m = R.rng(3).standard_normal((2, blocks, 2, kd)).astype(np.float32)
    q, m = (q * np.float32(scales[0])).astype(np.float32), (m * np.float32(scales[1])).astype(np.float32)
    got = run_select(hip, cfg, q, m, 1, blocks, many=tq == MANY)
    few, got = some(q, got)
    np.testing.assert_array_equal(got, R.select(cfg, few, m))


@pytest.mark.parametrize("tq", [FEW, MANY])
def test_uneven_channels(hip, tq):
    """One channel far above the others, and cancelled: what decides lies 2^-30 below the largest product."""
    cfg, kd, blocks = R.shape(1, 1, 1, 1, 4), 16, 150
    q, _ = tensors(1, 1, tq, cfg, kd, 1)
    m = R.rng(2).standard_normal((1, blocks, 1, kd)).astype(np.float32)
    q[..., 1] = -q[..., 0]
    m[..., 0] = m[..., 1] = np.float32(2.0 ** 30)
    got = run_select(hip, cfg, q, m, 1, blocks, many=tq == MANY)
    few, got = some(q, got)
    np.testing.assert_array_equal(got, R.select(cfg, few, m))


@pytest.mark.parametrize("kv,kd,selected", [(2, 32, 8), (2, 64, 20), (2, 128, 64), (2, 64, 1), (20, 32, 1), (20, 32, 9), (20, 64, 16)])
def test_long_causal_rows(hip, kv, kd, selected):
    """More blocks than a wave's tile, a few of them seen by the first queries and all by the last."""
    cfg = R.shape(3 * kv, kv, 1, 4, selected, causal=1)
    tq, w, starts, lengths = 1500, 1600, (0, 100), (1490, 1600)
    q, k = tensors(2, w, tq, cfg, kd, 3)
    m = R.means(cfg, k, 1, w, lengths).astype(np.float32)
    got = run_select(hip, cfg, q, m, 1, w, starts, lengths, many=True)
    keep = np.unique(np.concatenate([np.arange(0, 120, 7), np.arange(1380, 1500, 9), R.rng(2).integers(0, tq, 40)]))
    for i in keep:
        exp = R.select(cfg, q[:, i:i + 1], m, [s + i for s in starts], lengths)
        np.testing.assert_array_equal(got[:, i:i + 1], exp)


def test_means_behind_the_sequence_are_not_read(hip):
    """Whatever a cache's means hold behind the last query or the length: nothing of it in the choice."""
    cfg, kd, w, tq = R.shape(4, 2, 1, 4, 5, causal=1), 32, 1600, 1030
    q, k = tensors(2, w, tq, cfg, kd, 5)
    m = R.means(cfg, k, 1, w).astype(np.float32)
    starts, lengths = (100, 400), (1130, 1300)
    whole = run_select(hip, cfg, q, m, 1, w, starts, lengths, many=True)
    for value in (np.nan, np.inf, 1e30):
        far = m.copy()
        far[0, -(-1130 // 4):] = value
        far[1, -(-1300 // 4):] = value
        np.testing.assert_array_equal(run_select(hip, cfg, q, far, 1, w, starts, lengths, many=True), whole)
        far[1, -(-1300 // 4):] = m[1, -(-1300 // 4):]
        far[1, -(-1430 // 4):] = value  # no lengths: behind the last query
        np.testing.assert_array_equal(run_select(hip, cfg, q, far, 1, w, starts, None, many=True),
                                      run_select(hip, cfg, q, m, 1, w, starts, None, many=True))
    keep = np.arange(0, tq, 41)
    for i in keep:
        np.testing.assert_array_equal(whole[:, i:i + 1], R.select(cfg, q[:, i:i + 1], m, [x + i for x in starts], lengths))


def test_one_image_too_many(hip):
    cfg, kd = R.shape(2, 2, 1, 4, 2), 8
    with R.Device(hip) as d:
        vq, _, _ = d.view(np.zeros((2, 3, 2, kd), np.float32), 1, 3)
        vm, _ = means_view(d, cfg, 1, 1, 8, kd)
        with pytest.raises(SyError, match="images"):
            hip.block_select(R.config(cfg, kd, 4), vq, vm, d.put(np.zeros(12, np.int32)))
