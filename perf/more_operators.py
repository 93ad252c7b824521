"""Group normalisation with an activation, cross attention and the gated
projections of a feed-forward block, as cases that can be timed: the parts of a
decoder or an open-vocabulary neck whose maps and queries look at states of
another length.

Maps are feature maps of YOLO networks at inputs between 320 and 1280 pixels
(strides 8 to 32), channels last; encoders' states are the tokens of a text, the
pixels of all map levels or a long sequence of frames.
"""
import math

import torch

own = False

# Activations, as the framework numbers them.
NONE, SILU, GELU, GELU_TANH, RELU = 0, 1, 2, 3, 4


def listed():
    return [
        # The stride-32 map of one 640x640 frame between two convolutions: latency.
        dict(name="norm 20x20x256 b1", kind="norm", n=1, h=20, w=20, c=256, groups=32, act=SILU, wide=False),
        # Tokens on their own, one group: what stands before a block's projections.
        dict(name="norm 8400 tokens x256", kind="norm", n=8400, h=1, w=1, c=256, groups=1, act=NONE, wide=False),
        # Odd maps, a channel slice of a wider tensor, groups of 9 channels.
        dict(name="norm 45x75x108 b5", kind="norm", n=5, h=45, w=75, c=108, groups=12, act=RELU, wide=True),
        # The stride-8 map of 1280x1280 frames.
        dict(name="norm 160x160x256 b8", kind="norm", n=8, h=160, w=160, c=256, groups=32, act=SILU, wide=False),
        # The stride-32 map of one frame looks at a text of up to 77 tokens: latency.
        dict(name="cross 20x20 to 77 b1", kind="cross", n=1, tq=400, tk=77, heads=8, kv=8, kd=32, hd=32, ragged=True,
             masked=False),
        # One new token of each of 32 sequences against an encoder's 1500 states.
        dict(name="cross token to 1500 b32", kind="cross", n=32, tq=1, tk=1500, heads=8, kv=8, kd=64, hd=64,
             ragged=True, masked=False),
        # The stride-8 map of 1280x1280 frames and a text.
        dict(name="cross 160x160 to 77 b4", kind="cross", n=4, tq=25600, tk=77, heads=8, kv=8, kd=64, hd=64,
             ragged=True, masked=False),
        # Object queries that look at their own region of all three levels of a 640x640 frame.
        dict(name="cross 300 to 8400 b8 masked", kind="cross", n=8, tq=300, tk=8400, heads=8, kv=8, kd=32, hd=32,
             ragged=False, masked=True),
        # A long sequence and all levels' pixels, four query heads to a key head.
        dict(name="cross 4096 to 8400 b2", kind="cross", n=2, tq=4096, tk=8400, heads=16, kv=4, kd=128, hd=128,
             ragged=False, masked=False),
        # One new token: the weights are what is read.
        dict(name="gated token 1024-2816", kind="gated", rows=1, ic=1024, oc=2816, act=SILU, bias=False),
        # Object queries of four frames, odd widths.
        dict(name="gated 1200 rows 255-690", kind="gated", rows=1200, ic=255, oc=690, act=GELU, bias=True),
        # A long batch of tokens.
        dict(name="gated 16384 rows 1024-2816", kind="gated", rows=16384, ic=1024, oc=2816, act=SILU, bias=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["norm", "cross", "gated"])
        if kind == "norm":
            groups, each = rng.choice([1, 2, 8, 16, 32, 12]), rng.choice([4, 8, 16, 9, 5, 24])
            case = dict(kind=kind, c=groups * each, groups=groups, act=rng.choice([NONE, SILU, GELU, RELU]),
                        wide=rng.random() < 0.4)
            if rng.random() < 0.3:
                case.update(n=_log(rng, 1, 30000), h=1, w=1, groups=1)
            else:
                case.update(n=_log(rng, 1, 32), h=_log(rng, 4, 160), w=_log(rng, 4, 160))
        elif kind == "cross":
            kv, kd = rng.choice([1, 2, 4, 8]), rng.choice([32, 64, 128, 36, 80])
            form = rng.choice(["text", "map", "token"])
            tq = 1 if form == "token" else _log(rng, 16, 26000 if form == "text" else 2000)
            tk = _log(rng, 1, 300) if form == "text" else _log(rng, 100, 20000)
            case = dict(kind=kind, n=_log(rng, 1, 32), tq=tq, tk=tk, heads=kv * rng.choice([1, 1, 2, 3, 8]), kv=kv,
                        kd=kd, hd=rng.choice([kd, 32, 64, 128]), ragged=rng.random() < 0.6,
                        masked=form == "map" and rng.random() < 0.5)
        else:
            ic = _log(rng, 32, 2048)
            rows = _log(rng, 1, 16) if rng.random() < 0.4 else _log(rng, 16, 20000)
            case = dict(kind=kind, rows=rows, ic=ic, oc=int(ic * rng.choice([1, 2, 2.75, 4])) + rng.choice([0, 0, 1, 3]),
                        act=rng.choice([SILU, GELU, GELU_TANH, RELU]), bias=rng.random() < 0.5)
        cost = work(case)
        scores = case["n"] * case["heads"] * case["tq"] * case["tk"] if kind == "cross" else 0
        if cost["bytes"] < 4.0e8 and cost["flops"] < 1.8e11 and scores < 6.0e8:
            return case


# ------------------------------------------------------------------ inputs

class _State:
    def __init__(self, **kw):
        self.__dict__.update(kw)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(seed, *shape):
    return torch.randn(shape, generator=_gen(seed), device="cuda")


def _regions(case, seed):
    """One byte for each query and key: whether the key, one of a row of runs, is in the query's region.  A run is
    what a box cuts out of a map row; one query in fifty sees nothing."""
    n, tq, tk = case["n"], case["tq"], case["tk"]
    u = torch.rand((n, tq, 4), generator=_gen(seed), device="cuda")
    row = max(4, int(tk ** 0.5))
    at = torch.arange(tk, device="cuda")
    y, x = at // row, at % row
    lo_y, lo_x = u[..., 0:1] * (row * 0.8), u[..., 1:2] * (row * 0.8)
    far_y, far_x = lo_y + 1 + u[..., 2:3] * row * 0.5, lo_x + 1 + u[..., 3:4] * row * 0.5
    m = (y >= lo_y) & (y < far_y) & (x >= lo_x) & (x < far_x)
    return (m & (u[..., 0:1] < 0.98)).to(torch.uint8)


def prepare(case, seed):
    s = _State(case=case, plan=None, lengths=None, mask=None)
    if case["kind"] == "norm":
        n, h, w, c = (case[k] for k in ("n", "h", "w", "c"))
        wide = c + 32 if case["wide"] else c
        s.x = _normal(seed, n, h * w, wide)[..., wide - c:]
        # Channels of unequal spread about means of their own, as a convolution leaves them.
        s.x *= 0.5 + torch.rand(c, generator=_gen(seed + 1), device="cuda") * 2
        s.x += 2 * _normal(seed + 2, c)
        s.gamma, s.beta = 1 + 0.2 * _normal(seed + 3, c), 0.2 * _normal(seed + 4, c)
        s.y = torch.zeros((n, h * w, c), device="cuda")
        return s
    if case["kind"] == "gated":
        rows, ic, oc = case["rows"], case["ic"], case["oc"]
        s.x = _normal(seed, rows, ic)
        s.gate, s.up = (_normal(seed + i, oc, ic) * ic ** -0.5 for i in (1, 2))
        s.gate_bias, s.up_bias = (0.1 * _normal(seed + i, oc) if case["bias"] else None for i in (3, 4))
        s.y = torch.zeros((rows, oc), device="cuda")
        s.layer = _layer(s) if own else None
        return s
    n, tq, tk, heads, kv, kd, hd = (case[k] for k in ("n", "tq", "tk", "heads", "kv", "kd", "hd"))
    s.q = 1.5 * _normal(seed, n, tq, heads, kd)
    # Keys and values are the two halves of one projection of the states.
    s.states = _normal(seed + 1, n, tk, kv * (kd + hd))
    s.k = s.states[..., :kv * kd].unflatten(-1, (kv, kd))
    s.v = s.states[..., kv * kd:].unflatten(-1, (kv, hd))
    if case["ragged"]:
        s.lengths = torch.randint(tk // 4 + 1, tk + 1, (n,), generator=_gen(seed + 2), device="cuda",
                                  dtype=torch.int32)
    if case["masked"]:
        s.mask = _regions(case, seed + 3)
    s.o = torch.zeros((n, tq, heads, hd), device="cuda")
    return s


# --------------------------------------------------------------- plain forms

def _act(kind, x):
    if kind == SILU:
        return x / (1 + torch.exp(-x))
    if kind == GELU:
        return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    if kind == GELU_TANH:
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))
    if kind == RELU:
        return torch.where(x > 0, x, torch.zeros_like(x))
    return x


def _norm(case, x, gamma, beta):
    n, t, c = x.shape
    g = x.reshape(n, t, case["groups"], -1)
    mean = g.mean((1, 3), keepdim=True)
    d = g - mean
    d = d * torch.rsqrt((d * d).mean((1, 3), keepdim=True) + 1e-5)
    return _act(case["act"], d.reshape(n, t, c) * gamma + beta)


def _cross(case, q, k, v, lengths, mask):
    n, tq, heads, kd = q.shape
    kv, tk, hd = k.shape[2], k.shape[1], v.shape[-1]
    group = heads // kv
    qt = q.reshape(n, tq, kv, group, kd).permute(0, 2, 3, 1, 4).reshape(n, kv, group * tq, kd)
    s = torch.matmul(qt, k.permute(0, 2, 3, 1).contiguous()) * kd ** -0.5
    s = s.reshape(n, kv, group, tq, tk)
    if lengths is not None:
        s.masked_fill_((torch.arange(tk, device=q.device) >= lengths[:, None])[:, None, None, None], -math.inf)
    if mask is not None:
        s.masked_fill_((mask == 0)[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    s = torch.exp(s - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    s = s / s.sum(-1, keepdim=True).clamp(min=1e-37)
    o = torch.matmul(s.reshape(n, kv, group * tq, tk), v.transpose(1, 2).contiguous())
    return o.reshape(n, kv, group, tq, hd).permute(0, 3, 1, 2, 4).reshape(n, tq, heads, hd)


def _gated(case, x, gate, up, gate_bias, up_bias):
    a, b = torch.matmul(x, gate.t()), torch.matmul(x, up.t())
    if gate_bias is not None:
        a, b = a + gate_bias, b + up_bias
    return _act(case["act"], a) * b


# ------------------------------------------------------- the framework's calls

_context = None


def _ctx():
    """One context for the process, as a program has."""
    global _context
    if _context is None:
        from simdyolo_amd.device import HipContext
        _context = HipContext(0)
    return _context


def _layer(s):
    """The layer that a program makes once of its weights."""
    host = [None if t is None else t.cpu().numpy() for t in (s.gate, s.up, s.gate_bias, s.up_bias)]
    return _ctx().gated_create(host[0], host[1], gate_bias=host[2], up_bias=host[3], act=s.case["act"])


def _view(t, n, h, w, c, ldc):
    from simdyolo_amd import Tensor
    return Tensor(t.data_ptr(), n, c, h, w, ldc, 0)


def _make_plan(s):
    """The views that a program makes once for its buffers."""
    from simdyolo_amd import _native as N
    case = s.case
    if case["kind"] == "norm":
        n, h, w, c = (case[k] for k in ("n", "h", "w", "c"))
        return _State(x=_view(s.x, n, h, w, c, s.x.stride(1)), y=_view(s.y, n, h, w, c, c))
    if case["kind"] == "gated":
        rows, ic, oc = case["rows"], case["ic"], case["oc"]
        if s.layer is None:
            s.layer = _layer(s)
        return _State(x=_view(s.x, 1, 1, rows, ic, ic), y=_view(s.y, 1, 1, rows, oc, oc))
    n, tq, tk, heads, kv, kd, hd = (case[k] for k in ("n", "tq", "tk", "heads", "kv", "kd", "hd"))
    ld = s.states.stride(1)
    cfg = N.CrossConfig(heads=heads, kv_heads=kv, key_dim=kd, head_dim=hd, scale=kd ** -0.5)
    mask = None if s.mask is None else N.KeyMask(s.mask.data_ptr(), tq * tk, 0, tk)
    return _State(cfg=cfg, q=_view(s.q, n, 1, tq, heads * kd, heads * kd), k=_view(s.k, n, 1, tk, kv * kd, ld),
                  v=_view(s.v, n, 1, tk, kv * hd, ld), o=_view(s.o, n, 1, tq, heads * hd, heads * hd),
                  lengths=None if s.lengths is None else s.lengths.data_ptr(), mask=mask)


def _run_own(s):
    case, ctx = s.case, _ctx()
    if s.plan is None:
        s.plan = _make_plan(s)
    p = s.plan
    if case["kind"] == "norm":
        ctx.group_norm(p.x, p.y, case["groups"], gamma=s.gamma.data_ptr(), beta=s.beta.data_ptr(), eps=1e-5,
                       act=case["act"])
        return s.y
    if case["kind"] == "gated":
        ctx.gated(s.layer, p.x, p.y)
        return s.y
    ctx.cross_attention(p.cfg, p.q, p.k, p.v, p.o, lengths=p.lengths, mask=p.mask)
    return s.o


# -------------------------------------------------------------------- pass

def run(s):
    if own:
        return _run_own(s)
    case = s.case
    if case["kind"] == "norm":
        return _norm(case, s.x, s.gamma, s.beta)
    if case["kind"] == "gated":
        return _gated(case, s.x, s.gate, s.up, s.gate_bias, s.up_bias)
    return _cross(case, s.q, s.k, s.v, s.lengths, s.mask)


def work(case):
    if case["kind"] == "norm":
        values = case["n"] * case["h"] * case["w"] * case["c"]
        return {"bytes": 8 * values + 8 * case["c"], "flops": 8 * values}
    if case["kind"] == "gated":
        rows, ic, oc = case["rows"], case["ic"], case["oc"]
        return {"bytes": 4 * (rows * ic + 2 * oc * ic + rows * oc), "flops": 4 * rows * ic * oc}
    n, tq, tk, heads, kv, kd, hd = (case[k] for k in ("n", "tq", "tk", "heads", "kv", "kd", "hd"))
    seen = tk * 0.625 if case["ragged"] else tk  # lengths lie between a quarter and the whole
    moved = 4 * n * (tq * heads * (kd + hd) + seen * kv * (kd + hd)) + (n * tq * tk if case["masked"] else 0)
    return {"bytes": int(moved), "flops": int(2 * n * heads * tq * seen * (kd + hd))}


# ------------------------------------------------------------ in 64 bits

def _exact_act(kind, x):
    if kind == SILU:
        return x * torch.sigmoid(x)
    if kind == GELU:
        return x * 0.5 * torch.erfc(-x / math.sqrt(2.0))
    if kind == GELU_TANH:
        return x * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3))
    if kind == RELU:
        return x.clamp(min=0)
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        y = torch.empty(s.y.shape, dtype=torch.float64, device="cuda")
        each = case["c"] // case["groups"]
        for g in range(case["groups"]):
            part = slice(g * each, (g + 1) * each)
            x = s.x[..., part].double()
            x = x - x.mean((1, 2), keepdim=True)
            std = (x.square().mean((1, 2), keepdim=True) + 1e-5).sqrt()
            y[..., part] = _exact_act(case["act"], x / std * s.gamma[part].double() + s.beta[part].double())
        return y
    if case["kind"] == "gated":
        y = torch.empty(s.y.shape, dtype=torch.float64, device="cuda")
        gate, up = s.gate.double().t().contiguous(), s.up.double().t().contiguous()
        for i in range(0, case["rows"], 4096):
            x = s.x[i:i + 4096].double()
            a, b = x @ gate, x @ up
            if case["bias"]:
                a, b = a + s.gate_bias.double(), b + s.up_bias.double()
            y[i:i + 4096] = _exact_act(case["act"], a) * b
        return y
    n, tq, heads, kd = s.q.shape
    group, tk = heads // case["kv"], case["tk"]
    o = torch.zeros(s.o.shape, dtype=torch.float64, device="cuda")
    for b in range(n):
        used = tk if s.lengths is None else int(s.lengths[b])
        hidden = None if s.mask is None else s.mask[b, :, :used] == 0
        for h in range(heads):
            k = s.k[b, :used, h // group].double().t().contiguous()
            w = (s.q[b, :, h].double() @ k) / math.sqrt(kd)
            if hidden is not None:
                w = w.masked_fill(hidden, -math.inf)
            w = torch.nan_to_num(torch.softmax(w, -1), nan=0.0)
            o[b, :, h] = w @ s.v[b, :used, h // group].double()
    return o
