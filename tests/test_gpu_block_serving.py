"""Means, selection and attention as a program that serves runs them: a cache that grows by tokens and by pieces, and
captured calls replayed on new inputs."""
import numpy as np
import pytest

import _blocks as R
from test_gpu_block_attention import Chain, check, run, tensors
from simdyolo_amd.device import HipContext

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("piece", [1, 5, 8, 19])
@pytest.mark.parametrize("kd,selected", [(32, 3), (64, 5)])
def test_a_cache_that_grows(hip, piece, kd, selected):
    """Each step's means are those of the keys that are there, its lists those of these means, and both end as the whole
    sequence gives them; what is behind the last key, in the cache and in its means, is NaN all the time."""
    cfg, hd, w, n = R.shape(4, 2, 1, 8, selected, causal=1), 32, 91, 2
    q, k, v = tensors(n, w, w, cfg, kd, hd, 12)
    cf = R.config(cfg, kd, hd)
    bx = -(-w // 8)
    with R.Device(hip) as d:
        empty = np.full((n, w, 2, kd), np.nan, np.float32), np.full((n, w, 2, hd), np.nan, np.float32)
        vk, _, _ = d.view(empty[0], 1, w)
        vv, _, _ = d.view(empty[1], 1, w)
        vm, _, _ = d.view(np.full((n, bx, 1, 2 * kd), np.nan, np.float32), 1, bx)
        out = np.zeros((n, w, 4, hd), np.float32)
        lists = np.zeros((n, w, 2, selected), np.int32)
        for t in range(0, w, piece):
            m = min(piece, w - t)
            for b in range(n):  # the new tokens' keys and values join the cache
                hip.h2d(vk.data + 4 * (b * w + t) * 2 * kd, k[b, t:t + m])
                hip.h2d(vv.data + 4 * (b * w + t) * 2 * hd, v[b, t:t + m])
            s, ln = d.ints([t] * n), d.ints([t + m] * n)
            vq, _, _ = d.view(q[:, t:t + m], 1, m)
            vo, _, read = d.view(np.full((n, m, 4, hd), np.nan, np.float32), 1, m)
            p = d.put(np.full((n, m, 2, selected), 77, np.int32))
            hip.block_means(cf, vk, vm, s, m, ln)
            hip.block_select(cf, vq, vm, p, s, ln)
            hip.block_attention(cf, vq, vk, vv, p, vo, s, ln)
            out[:, t:t + m] = read()
            lists[:, t:t + m] = hip.d2h(p, (n, m, 2, selected), np.int32)
            means = hip.d2h(vm.data, (n, bx, 2, kd))
            there = -(-(t + m) // 8)
            exp = R.means(cfg, k, 1, w, [t + m] * n)
            assert np.isnan(means[:, there:]).all()
            assert (np.abs(means - exp)[:, :there] <= np.abs(exp)[:, :there] * 2.0 ** -24 + np.abs(k).max() * 2.0 ** -45).all()
            np.testing.assert_array_equal(lists[:, t:t + m], R.select(cfg, q[:, t:t + m], means, [t] * n, [t + m] * n))
        # The whole sequence at once: the block of a query's own token, whose mean has other keys in it then, is taken anyway.
        hip.h2d(vm.data, np.full((n, bx, 2, kd), np.nan, np.float32))
        hip.block_means(cf, vk, vm)
        np.testing.assert_array_equal(hip.d2h(vm.data, (n, bx, 2, kd)), means)
        vq, _, _ = d.view(q, 1, w)
        p = d.put(np.full(lists.shape, 77, np.int32))
        hip.block_select(cf, vq, vm, p)
        whole = hip.d2h(p, lists.shape, np.int32)
    own = np.arange(w) // 8
    if piece == 1:
        np.testing.assert_array_equal(lists, whole)
    np.testing.assert_array_equal(whole, R.select(cfg, q, means))
    assert (whole == own[:, None, None]).any(-1).all() and (lists == own[:, None, None]).any(-1).all()
    exp, bound = R.attend(cfg, q, k, v, lists, 1, w, kd ** -0.5)
    check(out, exp, bound)
    check(run(hip, cfg, q, k, v, whole, 1, w, pads=False), *R.attend(cfg, q, k, v, whole, 1, w, kd ** -0.5))


def test_two_graphs_on_new_inputs():
    """Two graphs that share the context's scratch, each replayed on inputs that neither was captured with, their lists
    and outputs wiped before, with eager work of the other between them."""
    with HipContext(0) as ctx, R.Device(ctx) as d:
        chains = [Chain(ctx, d, n, h, w, cfg, kd, hd, 3 + h) for n, h, w, cfg, kd, hd in
                  ((1, 20, 20, R.shape(2, 2, 4, 4, 4), 32, 64), (2, 26, 31, R.shape(2, 2, 3, 3, 6), 64, 32))]
        for c in chains:
            c()
        graphs = []
        for c in chains:
            ctx.graph_begin()
            c()
            graphs.append(ctx.graph_end())
        for turn in range(4):
            for i, (c, g) in enumerate(zip(chains, graphs)):
                c.x = R.rng(100 * turn + i).standard_normal(c.x.shape).astype(np.float32)
                ctx.h2d(c.view.data, c.x)
                for t in (c.rq, c.rk, c.m, c.o):
                    ctx.h2d(t.data, np.full(t.n * t.h * t.w * t.ldc, np.nan, np.float32))
                ctx.h2d(c.list, np.full(c.list_shape, -1, np.int32))
                if turn % 2:
                    chains[1 - i]()
                ctx.graph_launch(g)
                c.check()


def test_garbage_behind_the_last_token_costs_nothing(hip):
    """A causal call on a cache without lengths whose rest holds NaN: the rows of the last tokens are not computed twice (7
    times the call's time when they were)."""
    cfg, tq, w, dim = R.shape(16, 4, 1, 64, 8, causal=1), 4036, 4096, 64
    q, k, v = tensors(1, tq, w, cfg, dim, dim, 7)
    g = R.rng(8)
    blocks = np.sort(g.integers(0, np.arange(tq)[None, :, None, None] // 64 + 1, (1, tq, 4, 8)), -1).astype(np.int32)
    blocks[..., -1] = np.arange(tq)[:, None] // 64
    took = []
    for rest in (0.0, np.nan):
        k[:, tq:], v[:, tq:] = rest, rest
        with R.Device(hip) as d:
            vq, vk, vv = (d.view(a, 1, a.shape[1])[0] for a in (q, k, v))
            vo, _, read = d.view(np.full((1, tq, 16, dim), np.nan, np.float32), 1, tq)
            p, cf, least = d.put(blocks), R.config(cfg, dim, dim), np.inf
            for _ in range(5):
                hip.timer_start()
                hip.block_attention(cf, vq, vk, vv, p, vo)
                least = min(least, hip.timer_stop())
            got = read()
        took.append(least)
        keep = np.r_[g.integers(0, tq, 60), 3968:tq:5]
        for i in keep:
            check(got[:, i:i + 1], *R.attend(cfg, q[:, i:i + 1], k, v, blocks[:, i:i + 1], 1, w, dim ** -0.5, [i]))
    assert took[1] < 2 * took[0]
