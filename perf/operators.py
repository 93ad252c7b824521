"""Attention over chosen key blocks, and the rotary positions before it, as cases
that can be timed: rotation of queries and keys, the means of key blocks and the
selection of blocks for each query, and attention over the selected blocks.

Maps are feature maps of YOLO networks at inputs between 320 and 1280 pixels
(strides 8 to 32), whose blocks are windows of pixels; sequences are tokens in
one row, whose blocks are runs of tokens, whole (every token a query) or a token
at a time against a cache.
"""
import math

import torch

own = False

# Rotary scalings, as the framework numbers them.
NONE, LINEAR, BASE, PARTS = 0, 1, 2, 3


def listed():
    return [
        # One new token for each of 32 sequences at far positions: latency.
        dict(name="rotary token b32", kind="rotary", n=32, h=1, w=1, heads=8, kv=2, kd=64, dim=64, axes=1,
             inter=False, scaling=NONE, factor=1.0, packed=False, far=1000000),
        # Queries and keys of a stride-8 map, rotated by row and column on their way out of the qkv tensor.
        dict(name="rotary map 80x80 b8", kind="rotary", n=8, h=80, w=80, heads=4, kv=4, kd=32, dim=32, axes=2,
             inter=False, scaling=NONE, factor=1.0, packed=True, far=0),
        # A long sequence: half of each head, interleaved pairs, frequencies scaled by parts.
        dict(name="rotary 32768 partial", kind="rotary", n=1, h=1, w=32768, heads=32, kv=8, kd=128, dim=64, axes=1,
             inter=True, scaling=PARTS, factor=8.0, packed=False, far=32768),
        # Selection on the C2PSA map of one 640x640 frame: latency.
        dict(name="select 20x20 b1", kind="select", n=1, h=20, w=20, heads=2, kv=2, kd=32, bh=4, bw=4, sel=4,
             causal=False, new=0, ragged=False),
        # The stride-8 map of 1280x1280 frames.
        dict(name="select 160x160 b4", kind="select", n=4, h=160, w=160, heads=4, kv=4, kd=32, bh=8, bw=8, sel=8,
             causal=False, new=0, ragged=False),
        # Whole sequences of unequal lengths, four query heads to a key head.
        dict(name="select causal 16001 b2", kind="select", n=2, h=1, w=16001, heads=16, kv=4, kd=128, bh=1, bw=64,
             sel=16, causal=True, new=0, ragged=True),
        # One token against long caches whose older means are kept.
        dict(name="select token 65536 b16", kind="select", n=16, h=1, w=65536, heads=16, kv=4, kd=128, bh=1, bw=64,
             sel=16, causal=True, new=1, ragged=True),
        # Attention on the map of one 640x640 frame: latency.
        dict(name="attend 20x20 b1", kind="attend", n=1, h=20, w=20, heads=2, kv=2, kd=32, hd=64, bh=4, bw=4, sel=4,
             causal=False, new=0, ragged=False),
        # The stride-8 map of 1280x1280 frames.
        dict(name="attend 160x160 b2", kind="attend", n=2, h=160, w=160, heads=4, kv=4, kd=32, hd=64, bh=8, bw=8,
             sel=8, causal=False, new=0, ragged=False),
        # A whole sequence, four query heads to a key head.
        dict(name="attend causal 8192", kind="attend", n=1, h=1, w=8192, heads=16, kv=4, kd=128, hd=128, bh=1, bw=64,
             sel=16, causal=True, new=0, ragged=False),
        # One token against long caches.
        dict(name="attend token 65536 b16", kind="attend", n=16, h=1, w=65536, heads=16, kv=4, kd=128, hd=128, bh=1,
             bw=64, sel=16, causal=True, new=1, ragged=True),
        # Means, selection and attention in a row on ragged maps: windows that end outside the map.
        dict(name="chain 45x75 b4", kind="chain", n=4, h=45, w=75, heads=4, kv=4, kd=32, hd=64, bh=7, bw=7, sel=6,
             causal=False, new=0, ragged=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["rotary", "select", "attend", "chain"])
        form = rng.choice(["map", "sequence", "token"])
        kv = rng.choice([1, 2, 4, 8])
        group = 1 if form == "map" else rng.choice([1, 2, 3, 4, 8])
        kd = rng.choice([32, 64, 128, 36, 80])
        n = _log(rng, 1, 32)
        h, w = (_log(rng, 10, 160), _log(rng, 10, 160)) if form == "map" else (1, _log(rng, 2, 65536))
        case = dict(kind=kind, n=n, h=h, w=w, heads=kv * group, kv=kv, kd=kd)
        if kind == "rotary":
            axes = 2 if form == "map" else 1
            if form == "token":
                case["w"] = 1
            case.update(dim=rng.choice([kd, kd // 2 // 4 * 4]), axes=axes, inter=rng.random() < 0.5,
                        scaling=rng.choice([NONE, LINEAR, BASE, PARTS]), factor=rng.choice([2.0, 4.0, 32.0]),
                        packed=form == "map", far=0 if form == "map" else _log(rng, 1000, 1000000))
            if case["scaling"] == NONE:
                case["factor"] = 1.0
        else:
            bh, bw = (rng.randint(3, 8), rng.randint(3, 8)) if form == "map" else (1, rng.choice([16, 32, 48, 64, 128]))
            case.update(bh=bh, bw=bw, sel=rng.randint(1, 24), causal=form != "map", new=1 if form == "token" else 0,
                        ragged=form != "map" and rng.random() < 0.7)
            if kind != "select":
                case["hd"] = rng.choice([kd, 64, 128])
        cost = work(case)
        gathered = 0
        if kind in ("attend", "chain"):
            gathered = n * _queries(case) * kv * min(case["sel"], _blocks(case)) * bh * bw * (kd + case["hd"])
        sorted_ = 0 if kind == "rotary" else n * _queries(case) * kv * _blocks(case)
        if cost["bytes"] < 1.2e9 and cost["flops"] < 60e9 and gathered < 8e9 and sorted_ < 50e6 and \
                n * h * w * kv * kd < 1.2e9:
            return case


def _blocks(case):
    return -(-case["h"] // case["bh"]) * -(-case["w"] // case["bw"])


def _queries(case):
    return case["new"] or case["h"] * case["w"]


# ------------------------------------------------------------------ inputs

class _State:
    def __init__(self, **kw):
        self.__dict__.update(kw)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(seed, *shape):
    return torch.randn(shape, generator=_gen(seed), device="cuda")


def _window(case):
    """The block of every key token, and the blocks across."""
    y = torch.arange(case["h"], device="cuda") // case["bh"]
    x = torch.arange(case["w"], device="cuda") // case["bw"]
    across = -(-case["w"] // case["bw"])
    return (y[:, None] * across + x[None, :]).reshape(-1)


def _lengths(case, seed):
    """Valid keys of each sequence: the whole row, or from three quarters of it up."""
    t = case["h"] * case["w"]
    low = t * 3 // 4 + 1 if case["ragged"] else t
    return torch.randint(low, t + 1, (case["n"],), generator=_gen(seed), device="cuda", dtype=torch.int32)


def prepare(case, seed):
    s = _State(case=case, plan=None, lengths=None, starts=None)
    n, h, w, heads, kv, kd, kind = (case[k] for k in ("n", "h", "w", "heads", "kv", "kd", "kind"))
    t = h * w
    if kind == "rotary":
        if case["packed"]:
            # The output of a qkv convolution: per head q | k | v.
            s.x = _normal(seed, n, t, heads, 4 * kd)
            s.q, s.k = s.x[..., :kd], s.x[..., kd:2 * kd]
        else:
            s.q, s.k = _normal(seed, n, t, heads, kd), _normal(seed + 1, n, t, kv, kd)
        s.positions = None
        if case["far"]:
            first = torch.randint(0, case["far"], (n, 1), generator=_gen(seed + 2), device="cuda", dtype=torch.int32)
            s.positions = first + torch.arange(t, device="cuda", dtype=torch.int32)
        s.yq, s.yk = torch.zeros_like(s.q).contiguous(), torch.zeros_like(s.k).contiguous()
        return s
    blocks, window = _blocks(case), _window(case)
    tq = _queries(case)
    # Keys gather around one centre for each block and head, queries around the centre of a block that they
    # look for; blocks at the front are looked for more often.
    centre = _normal(seed + 3, n, blocks, kv, kd)
    s.k = _normal(seed, n, t, kv, kd)
    s.k += 0.6 * centre[:, window]
    sought = (blocks * torch.rand((n, tq), generator=_gen(seed + 4), device="cuda") ** 2).long()
    s.q = _normal(seed + 1, n, tq, kv, heads // kv, kd)
    s.q += 0.6 * centre[torch.arange(n, device="cuda")[:, None], sought][:, :, :, None]
    s.q = s.q.reshape(n, tq, heads, kd)
    if case["causal"]:
        s.lengths = _lengths(case, seed + 5)
        s.starts = s.lengths - case["new"] if case["new"] else torch.zeros_like(s.lengths)
    if kind != "select":
        s.v = _normal(seed + 2, n, t, kv, case["hd"])
        s.o = torch.zeros((n, tq, heads, case["hd"]), device="cuda")
    s.blocks = torch.zeros((n, tq, kv, case["sel"]), dtype=torch.int32, device="cuda")
    s.means = torch.zeros((n, blocks, kv, kd), device="cuda")
    if kind == "attend" or case["new"]:
        s.means.copy_(_means(case, s.k, s.lengths))
    if kind == "attend":
        s.blocks.copy_(_select(case, s.q, s.means, s.starts, s.lengths))
    return s


# --------------------------------------------------------------- plain forms

def _frequencies(case):
    """Radians for each position, and what cosines and sines are multiplied by."""
    part = case["dim"] // case["axes"]
    i = torch.arange(part // 2, dtype=torch.float64, device="cuda")
    base, factor = 10000.0, case["factor"]
    if case["scaling"] == BASE:
        base = base * factor ** (part / (part - 2))
    f = base ** (-2.0 * i / part)
    if case["scaling"] == LINEAR:
        return f / factor, 1.0
    if case["scaling"] != PARTS:
        return f, 1.0
    # Turns that a pair makes over the 4096 positions of the unscaled range: slow pairs (up to 1 turn) are
    # stretched, fast ones (32 and more) kept.
    keep = ((4096.0 * f / (2 * math.pi) - 1.0) / 31.0).clamp(0, 1)
    return f * (keep + (1 - keep) / factor), 0.1 * math.log(factor) + 1.0


def _rotate(case, x, positions):
    n, t, heads, kd = x.shape
    if positions is None:
        at = torch.arange(t, device="cuda")
        at = torch.stack([at // case["w"], at % case["w"]], -1) if case["axes"] == 2 else at[:, None]
        at = at[None]
    else:
        at = positions[..., None]
    f, m = _frequencies(case)
    angle = at.double()[..., None] * f  # [n or 1, t, axes, pairs]
    c, sn = ((g(angle) * m).float()[:, :, None] for g in (torch.cos, torch.sin))
    r = x[..., :case["dim"]].reshape(n, t, heads, case["axes"], -1)
    if case["inter"]:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack([a * c - b * sn, b * c + a * sn], -1)
    else:
        a, b = r.chunk(2, -1)
        y = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    return torch.cat([y.reshape(n, t, heads, case["dim"]), x[..., case["dim"]:]], -1)


def _means(case, k, lengths):
    """Mean key of every block; sums in 64 bits, as selections hang on them."""
    n, t, kv, kd = k.shape
    h, w, bh, bw = case["h"], case["w"], case["bh"], case["bw"]
    down, across = -(-h // bh), -(-w // bw)
    valid = torch.ones((n, t), dtype=torch.bool, device=k.device)
    if lengths is not None:
        valid = torch.arange(t, device=k.device)[None] < lengths[:, None]

    def windows(x):  # sums over windows
        x = torch.nn.functional.pad(x.reshape(n, h, w, -1), (0, 0, 0, across * bw - w, 0, down * bh - h))
        return x.reshape(n, down, bh, across, bw, -1).sum((2, 4)).reshape(n, down * across, -1)

    total = windows(k.double().reshape(n, t, -1) * valid[..., None])
    count = windows(valid[..., None].double()).clamp(min=1)
    return (total / count).reshape(n, -1, kv, kd).float()


def _last_means(case, k, starts, lengths, means):
    """Renews the mean of the block that holds the new token."""
    n, t, kv, kd = k.shape
    j = (starts // case["bw"]).long()
    at = j[:, None] * case["bw"] + torch.arange(case["bw"], device=k.device)
    valid = at < lengths[:, None]
    got = k[torch.arange(n, device=k.device)[:, None], at.clamp(max=t - 1)].double() * valid[..., None, None]
    means[torch.arange(n, device=k.device), j] = (got.sum(1) / valid.sum(1)[:, None, None]).float()
    return means


def _select(case, q, means, starts, lengths):
    """Indices of each query's blocks in ascending order, then -1.  Scores in 64 bits: their order decides."""
    n, tq, heads, kd = q.shape
    blocks, kv, sel = means.shape[1], case["kv"], case["sel"]
    qs = q.double().reshape(n, tq, kv, heads // kv, kd).sum(3)
    score = torch.matmul(qs.permute(0, 2, 1, 3).contiguous(), means.double().permute(0, 2, 3, 1).contiguous())
    j = torch.arange(blocks, device=q.device)
    sees = torch.ones((n, 1, tq, blocks), dtype=torch.bool, device=q.device)
    if case["causal"]:
        at = (starts[:, None] + torch.arange(tq, device=q.device))[:, None, :, None]
        sees = (j * case["bw"] <= at) & (j * case["bw"] < lengths[:, None, None, None])
        score = score.masked_fill(j == at // case["bw"], math.inf)
    score = score.masked_fill(~sees, -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True)[1][..., :sel]
    seen = torch.gather(sees.expand(score.shape), 3, order)
    order = order.masked_fill(~seen, blocks).sort(-1)[0]
    order = order.masked_fill(order == blocks, -1)
    got = torch.full((n, tq, kv, sel), -1, dtype=torch.int32, device=q.device)
    got[..., :order.shape[-1]] = order.permute(0, 2, 1, 3)
    return got


def _block_keys(case, blocks):
    """Token index of every key of the given blocks, and whether the map holds it."""
    u = torch.arange(case["bh"] * case["bw"], device=blocks.device)
    across = -(-case["w"] // case["bw"])
    j = blocks.long().clamp(min=0)[..., None]
    y = j // across * case["bh"] + u // case["bw"]
    x = j % across * case["bw"] + u % case["bw"]
    inside = (blocks[..., None] >= 0) & (y < case["h"]) & (x < case["w"])
    return torch.where(inside, y * case["w"] + x, 0), inside


def _attend(case, q, k, v, blocks, starts, lengths):
    n, tq, heads, kd = q.shape
    kv, hd, t = case["kv"], v.shape[-1], k.shape[1]
    at, sees = _block_keys(case, blocks)
    if case["causal"]:
        sees = sees & (at < lengths[:, None, None, None, None])
        sees = sees & (at <= (starts[:, None] + torch.arange(tq, device=q.device))[:, :, None, None, None])
    at, sees = at.flatten(3), sees.flatten(3)  # [n, tq, kv, keys]
    row = (torch.arange(n, device=q.device)[:, None, None, None] * t + at) * kv + \
        torch.arange(kv, device=q.device)[:, None]
    keys = k.reshape(-1, kd)[row]
    qt = q.reshape(n, tq, kv, heads // kv, kd).transpose(3, 4).contiguous()
    s = torch.matmul(keys, qt) * kd ** -0.5  # [n, tq, kv, keys, group]
    del keys
    s = s.masked_fill(~sees[..., None], -math.inf)
    top = s.amax(3, keepdim=True)
    e = torch.exp(s - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    p = (e / e.sum(3, keepdim=True).clamp(min=1e-37)).transpose(3, 4).contiguous()
    return torch.matmul(p, v.reshape(-1, hd)[row]).reshape(n, tq, heads, hd)


# ------------------------------------------------------- the framework's calls

_context = None


def _ctx():
    """One context for the process, as a program has."""
    global _context
    if _context is None:
        from simdyolo_amd.device import HipContext
        _context = HipContext(0)
    return _context


def _view(t, h, w):
    """The NHWC view of a [n, h * w, heads, dim] tensor whose channels are contiguous."""
    from simdyolo_amd import Tensor
    n, _, heads, dim = t.shape
    return Tensor(t.data_ptr(), n, (heads - 1) * t.stride(2) + dim, h, w, t.stride(1), 0)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _make_plan(s):
    """The handle and views that a program makes once for its buffers."""
    from simdyolo_amd import _native as N
    case, ctx = s.case, _ctx()
    h, w = case["h"], case["w"]
    if case["kind"] == "rotary":
        handle = ctx.rotary_create(case["kd"], case["dim"], axes=case["axes"], interleaved=case["inter"],
                                   base=10000.0, scaling=case["scaling"], factor=case["factor"], original=4096,
                                   low=1.0, high=32.0)
        parts = [N.RotaryHeads(_view(x, h, w), _view(y, h, w), x.shape[2], x.stride(2), y.stride(2))
                 for x, y in ((s.q, s.yq), (s.k, s.yk))]
        return handle, parts, _ptr(s.positions)
    cfg = N.BlockConfig(heads=case["heads"], kv_heads=case["kv"], key_dim=case["kd"], head_dim=case.get("hd", 4),
                        block_h=case["bh"], block_w=case["bw"], selected=case["sel"], causal=int(case["causal"]),
                        scale=case["kd"] ** -0.5)
    qh, qw = (1, case["new"]) if case["new"] else (h, w)
    p = _State(cfg=cfg, q=_view(s.q, qh, qw), k=_view(s.k, h, w), starts=_ptr(s.starts), lengths=_ptr(s.lengths),
               means=_view(s.means, -(-h // case["bh"]), -(-w // case["bw"])), blocks=_ptr(s.blocks))
    p.means.c, p.means.ldc = case["kv"] * case["kd"], case["kv"] * case["kd"]
    if case["kind"] != "select":
        p.v, p.o = _view(s.v, h, w), _view(s.o, qh, qw)
    return p


def _run_own(s):
    case, ctx = s.case, _ctx()
    if s.plan is None:
        s.plan = _make_plan(s)
    p, kind = s.plan, case["kind"]
    if kind == "rotary":
        ctx.rotary(*p)
        return s.yq, s.yk
    if kind != "attend":
        if case["new"]:
            ctx.block_means(p.cfg, p.k, p.means, starts=p.starts, tokens=case["new"], lengths=p.lengths)
        else:
            ctx.block_means(p.cfg, p.k, p.means, lengths=p.lengths)
        ctx.block_select(p.cfg, p.q, p.means, p.blocks, starts=p.starts, lengths=p.lengths)
        if kind == "select":
            return s.means, s.blocks
    ctx.block_attention(p.cfg, p.q, p.k, p.v, p.blocks, p.o, starts=p.starts, lengths=p.lengths)
    return s.o if kind == "attend" else (s.means, s.blocks, s.o)


# -------------------------------------------------------------------- pass

def run(s):
    if own:
        return _run_own(s)
    case, kind = s.case, s.case["kind"]
    if kind == "rotary":
        return _rotate(case, s.q, s.positions), _rotate(case, s.k, s.positions)
    if kind == "attend":
        return _attend(case, s.q, s.k, s.v, s.blocks, s.starts, s.lengths)
    if case["new"]:
        means = _last_means(case, s.k, s.starts, s.lengths, s.means)
    else:
        means = _means(case, s.k, s.lengths)
    blocks = _select(case, s.q, means, s.starts, s.lengths)
    if kind == "select":
        return means, blocks
    return means, blocks, _attend(case, s.q, s.k, s.v, blocks, s.starts, s.lengths)


def work(case):
    n, heads, kv, kd = case["n"], case["heads"], case["kv"], case["kd"]
    t = case["h"] * case["w"]
    if case["kind"] == "rotary":
        values = n * t * (heads + kv) * kd
        return {"bytes": 8 * values + (4 * n * t if case["far"] else 0), "flops": 3 * values * case["dim"] // kd}
    tq, blocks, sel = _queries(case), _blocks(case), case["sel"]
    size = case["bh"] * case["bw"]
    near = 4 * n * tq * (heads * kd + kv * sel)  # queries and indices
    whole = case["causal"] and not case["new"]
    moved, flops = near, 0
    if case["kind"] != "attend":
        read = size if case["new"] else t
        moved += 4 * n * kv * kd * (read + blocks)
        flops += n * tq * kv * kd * blocks * (1 if whole else 2)
    if case["kind"] != "select":
        hd, used = case["hd"], min(sel, blocks)
        # Keys that a query meets: all blocks' up to `sel`; in a whole causal sequence fewer at the front, and
        # half of its own block.
        met = size * used
        if whole:
            met = size * (used - 0.5 - used * (used - 1) / 2 / blocks)
        met = min(met, t)
        seen = met * kv * min(tq, t / met) if case["new"] else t * kv
        moved += 4 * n * (seen * (kd + hd) + tq * heads * hd)
        flops += 2 * n * tq * heads * met * (kd + hd)
    return {"bytes": int(moved), "flops": int(flops)}


# ------------------------------------------------------------ in 64 bits

def _exact_rotary(case, x, positions):
    n, t, heads, kd = x.shape
    y = x.double().clone()
    part, factor, m = case["dim"] // case["axes"], case["factor"], 1.0
    base = 10000.0
    for axis in range(case["axes"]):
        if positions is not None:
            at = positions.double()
        else:
            i = torch.arange(t, device="cuda")
            at = (i if case["axes"] == 1 else i // case["w"] if axis == 0 else i % case["w"]).double()[None]
        for i in range(part // 2):
            f = base ** (-2.0 * i / part)
            if case["scaling"] == BASE:
                f = (base * factor ** (part / (part - 2.0))) ** (-2.0 * i / part)
            elif case["scaling"] == LINEAR:
                f /= factor
            elif case["scaling"] == PARTS:
                keep = min(1.0, max(0.0, (4096.0 * f / (2 * math.pi) - 1.0) / 31.0))
                f = f * keep + f / factor * (1.0 - keep)
                m = 0.1 * math.log(factor) + 1.0
            c, sn = torch.cos(at * f)[..., None] * m, torch.sin(at * f)[..., None] * m
            first = axis * part + (2 * i if case["inter"] else i)
            second = first + (1 if case["inter"] else part // 2)
            a, b = x[..., first].double(), x[..., second].double()
            y[..., first], y[..., second] = a * c - b * sn, a * sn + b * c
    return y


def _exact_means(case, k, lengths):
    n, t, kv, kd = k.shape
    bh, bw, h, w = case["bh"], case["bw"], case["h"], case["w"]
    across, down = -(-w // bw), -(-h // bh)
    valid = torch.ones((n, t), dtype=torch.float64, device="cuda")
    if lengths is not None:
        valid = (torch.arange(t, device="cuda") < lengths[:, None]).double()
    x = (k.double() * valid[..., None, None]).reshape(n, h, w, kv * kd)
    valid = valid.reshape(n, h, w, 1)
    total = torch.zeros((n, down, across, kv * kd), dtype=torch.float64, device="cuda")
    count = torch.zeros((n, down, across, 1), dtype=torch.float64, device="cuda")
    for dy in range(min(bh, h)):
        for dx in range(min(bw, w)):
            part = x[:, dy::bh, dx::bw]
            total[:, :part.shape[1], :part.shape[2]] += part
            count[:, :part.shape[1], :part.shape[2]] += valid[:, dy::bh, dx::bw]
    return (total / count.clamp(min=1.0)).reshape(n, -1, kv, kd)


def _exact_select(case, q, means, starts, lengths):
    """One ranking for each sequence and key head."""
    n, tq, heads, kd = q.shape
    blocks, kv, sel = means.shape[1], case["kv"], case["sel"]
    got = torch.full((n, tq, kv, sel), -1, dtype=torch.int32, device="cuda")
    first = torch.arange(blocks, device="cuda") * case["bw"]
    for b in range(n):
        for g in range(kv):
            mine = q[b, :, g * (heads // kv):(g + 1) * (heads // kv)].double().sum(1)
            score = mine @ means[b, :, g].double().t().contiguous()
            hidden = torch.zeros_like(score, dtype=torch.bool)
            if case["causal"]:
                at = (int(starts[b]) + torch.arange(tq, device="cuda"))[:, None]
                hidden = (first > at) | (first >= int(lengths[b]))
                score[(first <= at) & (at < first + case["bw"])] = math.inf
                score[hidden] = -math.inf
            rank = torch.argsort(-score, dim=1, stable=True)[:, :sel]
            rank = torch.where(torch.gather(hidden, 1, rank), blocks, rank).sort(1)[0]
            got[b, :, g, :rank.shape[1]] = torch.where(rank == blocks, -1, rank).int()
    return got


def _exact_attend(case, q, k, v, blocks, starts, lengths):
    n, tq, heads, kd = q.shape
    kv, hd, group = case["kv"], v.shape[-1], heads // case["kv"]
    bh, bw, h, w = case["bh"], case["bw"], case["h"], case["w"]
    across = -(-w // bw)
    dy = torch.arange(bh, device="cuda").repeat_interleave(bw)
    dx = torch.arange(bw, device="cuda").repeat(bh)
    out = torch.zeros((n, tq, heads, hd), dtype=torch.float64, device="cuda")
    step = max(1, 20000000 // (blocks.shape[-1] * bh * bw * (kd + hd)))
    for b in range(n):
        for g in range(kv):
            kb, vb = k[b, :, g].double(), v[b, :, g].double()
            for i in range(0, tq, step):
                j = blocks[b, i:i + step, g].long()
                y = (torch.div(j, across, rounding_mode="floor") * bh)[..., None] + dy
                x = ((j % across) * bw)[..., None] + dx
                ok = (j[..., None] >= 0) & (y < h) & (x < w)
                at = (y * w + x)
                if case["causal"]:
                    pos = int(starts[b]) + torch.arange(i, i + j.shape[0], device="cuda")
                    ok &= (at < int(lengths[b])) & (at <= pos[:, None, None])
                at, ok = torch.where(ok, at, 0).flatten(1), ok.flatten(1)
                qh = q[b, i:i + step, g * group:(g + 1) * group].double()
                s = (qh @ kb[at].transpose(1, 2).contiguous()) / math.sqrt(kd)
                s = s.masked_fill(~ok[:, None], -math.inf)
                p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
                out[b, i:i + step, g * group:(g + 1) * group] = p @ vb[at]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        return _exact_rotary(case, s.q, s.positions), _exact_rotary(case, s.k, s.positions)
    if case["kind"] == "attend":
        return _exact_attend(case, s.q, s.k, s.v, s.blocks, s.starts, s.lengths)
    means = _exact_means(case, s.k, s.lengths)
    if case["kind"] == "select":
        return means, None
    blocks = _exact_select(case, s.q, means.float(), s.starts, s.lengths)
    return means, None, _exact_attend(case, s.q, s.k, s.v, blocks, s.starts, s.lengths)
