"""The operators around a decoder's KV cache that a program on this framework calls beside the decode and prefill
attention, as timed cases: rows written into a cache of q8_0 blocks and read back, attention of a drafted tree of tokens
over a cache, and attention with a sliding window and a few first tokens that stay visible.

A cache is one layer's, [n_kv][n_ctx][128], in f16 or as q8_0 blocks of 32 values: int8 quants q and an f16 scale d, which
stand for f16(q·d). A block's scale is the smallest f16 number d with 127·d >= max |x|, its quants are x / d rounded to the
nearest integer, ties to even. Each operator is here in its plain form too (elementary torch operations), which says what
it computes; `own` picks the framework's kernels. Inputs are synthetic: normed keys and queries ~ N(0, 1), values ~
N(0, 4^2), norm weights 1 + N(0, 0.02^2), as perf/cases.py has them.
"""
from __future__ import annotations

import math
import os
import random
import sys

import numpy as np
import torch

own = False

HEAD, EPS, ROPE_BASE = 128, 1e-6, 1e6
F16, Q8_0 = 1, 8  # the ggml types of a cache's rows
MODEL = dict(n_head=16, n_kv=8)  # the LightOnOCR decoder's heads


def listed():
    return [
        # one token's q / k norm, RoPE and quantised store, and its row read back: a decode step's share, all latency
        dict(name="write_token", kind="write", n=1, pos0=700, **MODEL),
        # the same for a page's prompt
        dict(name="write_page", kind="write", n=1925, pos0=0, **MODEL),
        # a read that is put aside: its f16 cache into q8_0 and back, a page's and the longest
        dict(name="park_page", kind="park", rows=2437, n_kv=8),
        dict(name="park_long", kind="park", rows=60001, n_kv=8),
        # one layer's share of a drafted step: the nodes' rows made and stored, their attention over the f16 cache, the
        # accepted path's rows moved together; a narrow draft early in a page and the widest one late
        dict(name="draft_narrow", kind="draft", nodes=7, past=1300, **MODEL),
        dict(name="draft_wide", kind="draft", nodes=64, past=6001, **MODEL),
        # attention alone: one token (the decode step over a q8_0 cache), a middling tree over a long q8_0 cache, the
        # widest one over the f16 cache of a page with more queries to a KV head than the model has
        dict(name="token_q8", kind="tree", type=Q8_0, nodes=1, past=7999, **MODEL),
        dict(name="tree_q8_long", kind="tree", type=Q8_0, nodes=27, past=40013, **MODEL),
        dict(name="tree_f16_groups", kind="tree", type=F16, nodes=61, past=2437, n_head=32, n_kv=4),
        # a long read that keeps a window: one token, a page's prompt on f16 rows, a long prompt's second part on q8_0 rows
        dict(name="window_token", kind="window", type=Q8_0, n=1, pos0=9000, window=1024, sink=4, **MODEL),
        dict(name="window_page", kind="window", type=F16, n=1925, pos0=0, window=512, sink=4, **MODEL),
        dict(name="window_long", kind="window", type=Q8_0, n=6001, pos0=1925, window=1500, sink=16, **MODEL),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["write", "park", "draft", "draft", "tree", "tree", "tree", "window", "window", "window"])
    n_kv = rng.choice([1, 2, 4, 8, 8])
    heads = dict(n_head=n_kv * rng.choice([1, 2, 2, 3, 4]), n_kv=n_kv)
    if kind == "write":
        return dict(kind=kind, n=_log(rng, 1, 1925), pos0=rng.choice([0, rng.randint(1, 4000)]), **heads)
    if kind == "park":
        return dict(kind=kind, rows=_log(rng, 1, 60001), n_kv=n_kv)
    if kind == "draft":
        return dict(kind=kind, nodes=_log(rng, 1, 64), past=_log(rng, 1, 6001), **heads)
    if kind == "tree":
        return dict(kind=kind, type=rng.choice([F16, Q8_0]), nodes=_log(rng, 1, 64), past=_log(rng, 1, 16000), **heads)
    return dict(kind=kind, type=rng.choice([F16, Q8_0]), n=_log(rng, 1, 2500), pos0=rng.choice([0, rng.randint(1, 4000)]),
                window=_log(rng, 16, 1500), sink=rng.choice([0, 1, 4, 16, 64]), **heads)


# ---- inputs --------------------------------------------------------------------------------------------------------

class _State:
    """what a program holds for a case"""

    def __init__(self, case):
        self.case, self.held = case, None

    def __del__(self):
        if self.held is not None:
            _dev().sync()  # nothing in flight still uses the tensors


def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed(1_000_003 * int(seed) + salt)
    return g


def _normal(g, *shape, mean=0.0, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda").mul_(std).add_(mean)


def _rope(n):
    """(cos, sin) of the positions 0 ... n - 1 and the 64 pairs of a head: f32 [n, 64, 2]"""
    i = torch.arange(HEAD // 2, dtype=torch.float64, device="cuda")
    a = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * ROPE_BASE ** (-2.0 * i / HEAD)
    return torch.stack([a.cos(), a.sin()], dim=2).float()


def _quantise(x):
    """q8_0 blocks of rows x [..., 128]: int8 quants of the same shape and f16 scales [..., 4]"""
    b = x.double().unflatten(-1, (4, 32))
    top = b.abs().amax(-1, keepdim=True)
    d = (top / 127).half()
    d = torch.where(127 * d.double() < top, (d.view(torch.int16) + 1).view(torch.float16), d)
    q = torch.where(d > 0, (b / d.double()).round(), 0.0)
    return q.to(torch.int8).flatten(-2), d.squeeze(-1)


def _values(q, d):
    """the f16 values that q8_0 blocks stand for"""
    return (q.float().unflatten(-1, (4, 32)) * d.float().unsqueeze(-1)).flatten(-2).half()


def _cache(case, g, rows, std):
    x = _normal(g, case["n_kv"], rows, HEAD, std=std).half()
    return _quantise(x) if case.get("type") == Q8_0 else (x, None)


def _tree(case, seed):
    """a drafted tree: each node's parent is an earlier one (near it, mostly) or the last committed token (-1); the nodes
    of an accepted path, from the root down"""
    rng = random.Random(int(seed) * 7919 + case["nodes"])
    parent = [-1 if i == 0 or rng.random() < 0.1 else max(0, i - 1 - int(rng.expovariate(0.4))) for i in range(case["nodes"])]
    path, i = [], case["nodes"] - 1
    while i >= 0:
        path.append(i)
        i = parent[i]
    return parent, path[::-1]


def prepare(case, seed):
    s, kind = _State(case), case["kind"]
    g = _gen(seed, 21)
    n_kv = case["n_kv"]
    if kind == "park":
        s.k, s.v = _normal(g, n_kv, case["rows"], HEAD).half(), _normal(g, n_kv, case["rows"], HEAD, std=4.0).half()
        s.qk, s.qv = (torch.zeros_like(x, dtype=torch.int8) for x in (s.k, s.v))
        s.dk, s.dv = (torch.zeros(*x.shape[:2], 4, dtype=torch.float16, device="cuda") for x in (s.k, s.v))
        s.back_k, s.back_v = torch.zeros_like(s.k), torch.zeros_like(s.v)
        return s
    n_head = case["n_head"]
    if kind in ("write", "draft"):
        n = case["n"] if kind == "write" else case["nodes"]
        # the rows of the fused projections, [q | k | v]
        s.qkv = _normal(g, n, (n_head + 2 * n_kv) * HEAD)
        s.qkv[:, (n_head + n_kv) * HEAD:] *= 4.0
        s.q_norm, s.k_norm = _normal(g, HEAD, mean=1.0, std=0.02), _normal(g, HEAD, mean=1.0, std=0.02)
        s.q = torch.zeros(n, n_head * HEAD, device="cuda")
    if kind == "write":
        ctx = case["pos0"] + n
        s.rope = _rope(ctx)
        s.qk, s.qv = (torch.zeros(n_kv, ctx, HEAD, dtype=torch.int8, device="cuda") for _ in range(2))
        s.dk, s.dv = (torch.zeros(n_kv, ctx, 4, dtype=torch.float16, device="cuda") for _ in range(2))
        s.back_k, s.back_v = (torch.zeros(n_kv, n, HEAD, dtype=torch.float16, device="cuda") for _ in range(2))
        return s
    if kind in ("draft", "tree"):
        s.parent, s.path = _tree(case, seed)
        n, rows = case["nodes"], case["past"] + case["nodes"]
        s.depth = [0] * n
        for i, p in enumerate(s.parent):
            s.depth[i] = s.depth[p] + 1 if p >= 0 else 0
    else:
        n, rows = case["n"], case["pos0"] + case["n"]
    if kind == "draft":
        s.rope = _rope(rows)
    else:
        s.q = _normal(g, n, n_head * HEAD)
    s.k, s.dk = _cache(case, g, rows, 1.0)
    s.v, s.dv = _cache(case, g, rows, 4.0)
    s.out = torch.zeros(n, n_head * HEAD, device="cuda")
    return s


# ---- the framework's calls -------------------------------------------------------------------------------------------

_device = None


def _htr():
    at = os.path.join(os.getcwd(), "historic-htr-ocr_amd")  # the working folder is the repository's root
    if at not in sys.path:
        sys.path.insert(0, at)
    import htr

    return htr


def _dev():
    """the program's one device, opened at its first use"""
    global _device
    if _device is None:
        _device = _htr().Device(0)
    return _device


class _Ref:
    """device memory of a torch tensor, as the entry points take it"""

    def __init__(self, t, offset=0):
        self.ptr = t.data_ptr() + offset


class _Held:
    """the handles that a program keeps for a case's buffers: made once, at its first pass"""

    def __init__(self, s):
        htr, c = _htr(), s.case
        n_kv = c["n_kv"]
        ref = lambda t: None if t is None else _Ref(t)  # noqa: E731
        cache = lambda k, v, dk, dv: htr.KvCache.of(k.shape[0], k.shape[1], _Ref(k), _Ref(v), ref(dk), ref(dv))  # noqa: E731
        for name in ("q", "out", "rope", "q_norm", "k_norm"):
            if hasattr(s, name):
                setattr(self, name, _Ref(getattr(s, name)))
        if hasattr(s, "qkv"):
            self.raw = [_Ref(s.qkv, 4 * HEAD * h) for h in (0, c["n_head"], c["n_head"] + n_kv)]
        if hasattr(s, "qk"):
            self.q8 = cache(s.qk, s.qv, s.dk, s.dv)
            self.back = cache(s.back_k, s.back_v, None, None)
        if hasattr(s, "k"):
            self.kv = cache(s.k, s.v, s.dk, s.dv) if hasattr(s, "out") else cache(s.k, s.v, None, None)
        if hasattr(s, "parent"):
            self.tree = htr.Tree(s.parent)


def _run_own(s):
    htr, dev, c, kind = _htr(), _dev(), s.case, s.case["kind"]
    if s.held is None:
        s.held = _Held(s)
    h, scale = s.held, HEAD ** -0.5
    if kind == "park":
        htr.kv_copy(dev, h.kv, 0, h.q8, 0, c["rows"])
        htr.kv_copy(dev, h.q8, 0, h.back, 0, c["rows"])
        return {"k": s.back_k, "v": s.back_v}
    if kind == "write":
        width = s.qkv.shape[1]
        htr.qkv_post_rows(dev, h.raw[0], h.raw[1], h.raw[2], c["n"], h.q_norm, h.k_norm, h.rope, s.rope.shape[0], c["pos0"],
                          c["n_head"], EPS, h.q8, c["pos0"], h.q, q_stride=width, kv_stride=width)
        htr.kv_copy(dev, h.q8, c["pos0"], h.back, 0, c["n"])
        return {"q": s.q, "k": s.back_k, "v": s.back_v}
    if kind == "draft":
        width, past = s.qkv.shape[1], c["past"]
        htr.qkv_post_rows(dev, h.raw[0], h.raw[1], h.raw[2], c["nodes"], h.q_norm, h.k_norm, h.rope, s.rope.shape[0], past,
                          c["n_head"], EPS, h.kv, past, h.q, q_stride=width, kv_stride=width, tree=h.tree)
        htr.tree_attention(dev, h.q, h.tree, past, h.kv, c["n_head"], scale, h.out)
        htr.kv_keep(dev, h.kv, past, s.path)
        return {"q": s.q, "out": s.out, "k": s.k[:, past:], "v": s.v[:, past:]}
    if kind == "tree":
        htr.tree_attention(dev, h.q, h.tree, c["past"], h.kv, c["n_head"], scale, h.out)
        return s.out
    htr.window_attention(dev, h.q, c["n"], c["pos0"], c["window"], c["sink"], h.kv, c["n_head"], scale, h.out)
    return s.out


# ---- the plain forms -------------------------------------------------------------------------------------------------

def _post(x, w, cs):
    """rows x [n, heads, 128]: each head's RMS norm with weights w, then the pairs (i, i + 64) turned by cs [n, 64, 2]. In
    64 bits: the results are rounded to the cache's types, and lie next to a border of theirs now and then"""
    x = x.double()
    y = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
    a, b = y[..., :64], y[..., 64:]
    c, t = cs.double()[:, None, :, 0], cs.double()[:, None, :, 1]
    return torch.cat([a * c - b * t, a * t + b * c], dim=-1)


def _rows(s, pos):
    """the raw rows' queries, keys and values at the positions pos: f64 [n, heads, 128]"""
    c = s.case
    n_head, n_kv = c["n_head"], c["n_kv"]
    x = s.qkv.view(len(pos), n_head + 2 * n_kv, HEAD)
    cs = s.rope[pos]
    return _post(x[:, :n_head], s.q_norm, cs), _post(x[:, n_head:n_head + n_kv], s.k_norm, cs), x[:, n_head + n_kv:].double()


def _attend(q, k, v, seen, n_kv):
    """softmax(q·k / sqrt(128) over the keys that each query sees)·v: q [n, heads·128], k and v [n_kv, keys, 128], seen
    [n, keys]; a query that sees none gets zeros"""
    n, n_head = q.shape[0], q.shape[1] // HEAD
    x = (q.float() * HEAD ** -0.5).view(n, n_kv, n_head // n_kv, HEAD).transpose(0, 1).reshape(n_kv, -1, HEAD)
    score = torch.matmul(x, k.float().transpose(1, 2)).view(n_kv, n, n_head // n_kv, -1)
    score = torch.where(seen[None, :, None, :], score, -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(-3e38)
    p = (score - top).exp()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(1, 2), v.float()).view(n_kv, n, -1, HEAD) / torch.where(total > 0, total, 1.0)
    return o.transpose(0, 1).reshape(n, -1)


def _tree_seen(s):
    """node i sees the committed keys and the nodes on its path from the root, itself among them"""
    n, past = s.case["nodes"], s.case["past"]
    on = np.zeros((n, n), bool)
    for i, p in enumerate(s.parent):
        on[i] = on[p] if p >= 0 else False
        on[i, i] = True
    return torch.cat([torch.ones(n, past, dtype=torch.bool), torch.from_numpy(on)], dim=1).cuda()


def _window_seen(c):
    pos = c["pos0"] + torch.arange(c["n"], device="cuda")[:, None]
    key = torch.arange(c["pos0"] + c["n"], device="cuda")[None, :]
    return (key <= pos) & ((key < c["sink"]) | (key > pos - c["window"]))


def _run_plain(s):
    c, kind = s.case, s.case["kind"]
    if kind == "park":
        for x, q, d, back in ((s.k, s.qk, s.dk, s.back_k), (s.v, s.qv, s.dv, s.back_v)):
            for to, new in zip((q, d), _quantise(x)):
                to.copy_(new)
            back.copy_(_values(q, d))
        return {"k": s.back_k, "v": s.back_v}
    if kind == "write":
        rows = slice(c["pos0"], c["pos0"] + c["n"])
        q, k, v = _rows(s, torch.arange(c["pos0"], c["pos0"] + c["n"], device="cuda"))
        s.q.copy_(q.flatten(1))
        for x, to, d, back in ((k, s.qk, s.dk, s.back_k), (v, s.qv, s.dv, s.back_v)):
            to[:, rows], d[:, rows] = _quantise(x.float().transpose(0, 1))
            back.copy_(_values(to[:, rows], d[:, rows]))
        return {"q": s.q, "k": s.back_k, "v": s.back_v}
    if kind == "draft":
        past, kept = c["past"], len(s.path)
        q, k, v = _rows(s, torch.tensor([past + d for d in s.depth], device="cuda"))
        s.q.copy_(q.flatten(1))
        s.k[:, past:], s.v[:, past:] = k.float().transpose(0, 1), v.float().transpose(0, 1)
        s.out.copy_(_attend(s.q, s.k, s.v, _tree_seen(s), c["n_kv"]))
        at = torch.tensor([past + i for i in s.path], device="cuda")
        s.k[:, past:past + kept], s.v[:, past:past + kept] = s.k[:, at], s.v[:, at]
        return {"q": s.q, "out": s.out, "k": s.k[:, past:], "v": s.v[:, past:]}
    k, v = (s.k, s.v) if s.dk is None else (_values(s.k, s.dk), _values(s.v, s.dv))
    return _attend(s.q, k, v, _tree_seen(s) if kind == "tree" else _window_seen(c), c["n_kv"])


def run(s):
    if own:
        return _run_own(s)
    return _run_plain(s)


# ---- what a case cannot do without -----------------------------------------------------------------------------------

def _row_bytes(t):
    """K and V of one position of one KV head"""
    return 2 * (HEAD + 8 if t == Q8_0 else 2 * HEAD)


def work(case):
    kind, n_kv = case["kind"], case["n_kv"]
    f16, q8 = n_kv * _row_bytes(F16), n_kv * _row_bytes(Q8_0)
    if kind == "park":
        return {"bytes": case["rows"] * (2 * f16 + 2 * q8), "flops": case["rows"] * n_kv * 2 * HEAD * 6}
    n_head = case["n_head"]
    # a row's raw q, k and v, its (cos, sin), its q written; the arithmetic of norm, turn and rounding
    made = 4 * HEAD * (n_head + 2 * n_kv) + 4 * HEAD + 4 * HEAD * n_head
    ops = HEAD * (n_head + 2 * n_kv) * 12
    if kind == "write":
        return {"bytes": case["n"] * (made + 2 * q8 + f16), "flops": case["n"] * ops}
    qo = 2 * 4 * HEAD * n_head
    if kind == "window":
        n, pos0, w, sink = case["n"], case["pos0"], case["window"], case["sink"]
        p = np.arange(pos0, pos0 + n, dtype=np.int64)
        first = np.maximum(p - w + 1, 0)
        pairs = int((p + 1 - first + np.minimum(sink, first)).sum())
        keys = pos0 + n - int(first[0]) + min(sink, int(first[0]))
        return {"bytes": keys * n_kv * _row_bytes(case["type"]) + n * qo, "flops": 4 * HEAD * n_head * pairs}
    n, past = case["nodes"], case["past"]
    flops = 4 * HEAD * n_head * n * (past + 1)
    if kind == "tree":
        return {"bytes": (past + n) * n_kv * _row_bytes(case["type"]) + n * qo, "flops": flops}
    # the nodes' rows are made and written, the attention reads the committed ones and writes its output
    return {"bytes": n * (made + f16) + past * f16 + n * qo // 2, "flops": flops + n * ops}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------

def _exact_blocks(x):
    """what the blocks of x [..., 128] stand for, from the definition: every f16 scale in order, the first that reaches"""
    x = x.double()
    scales = torch.arange(0x7C00, dtype=torch.int16, device=x.device).view(torch.float16).double()
    out = []
    for part in x.split(32, dim=-1):
        top = part.abs().max(dim=-1, keepdim=True).values
        d = scales[torch.searchsorted(scales * 127.0, top.contiguous())]
        n = torch.where(d == 0, torch.zeros_like(part), part / torch.where(d == 0, torch.ones_like(d), d))
        low = n.floor()
        up = (n - low > 0.5) | ((n - low == 0.5) & (low.remainder(2) == 1))
        out.append((low + up) * d)
    return torch.cat(out, dim=-1)


def _exact_heads(x, w, pos):
    """RMS norm and turn of the heads x [n, heads, 128] at the positions pos, as complex numbers"""
    x = x.double()
    x = x * torch.rsqrt((x * x).sum(dim=2, keepdim=True) / HEAD + EPS) * w.double()
    z = torch.complex(x[:, :, :64].contiguous(), x[:, :, 64:].contiguous())
    turn = _rope(int(max(pos)) + 1)[torch.as_tensor(pos, device="cuda")].double()
    z = z * torch.complex(turn[..., 0].contiguous(), turn[..., 1].contiguous())[:, None, :]
    return torch.cat([z.real, z.imag], dim=2)


def _exact_attention(q, k, v, n_head, allowed):
    """one head at a time: q [n, n_head, 128], k and v [n_kv, keys, 128] in 64 bits, allowed [n, keys]"""
    n_kv = k.shape[0]
    out = torch.zeros(q.shape[0], n_head, HEAD, dtype=torch.float64, device="cuda")
    for h in range(n_head):
        j = h * n_kv // n_head
        t = q[:, h].contiguous() @ k[j].t().contiguous() / math.sqrt(HEAD)
        w = torch.softmax(t.masked_fill_(~allowed, -math.inf), dim=1)
        out[:, h] = w @ v[j]
    return out.flatten(1)


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "park":
        return {"k": _exact_blocks(s.k), "v": _exact_blocks(s.v)}
    n_head, n_kv = case["n_head"], case["n_kv"]
    if kind in ("write", "draft"):
        n = s.qkv.shape[0]
        pos = [case["pos0"] + i for i in range(n)] if kind == "write" else [case["past"] + d for d in s.depth]
        q, k, v = s.qkv.view(n, -1, HEAD).split([n_head, n_kv, n_kv], dim=1)
        q, k, v = _exact_heads(q, s.q_norm, pos), _exact_heads(k, s.k_norm, pos).permute(1, 0, 2), v.permute(1, 0, 2)
        if kind == "write":
            return {"q": q.flatten(1), "k": _exact_blocks(k.float()), "v": _exact_blocks(v)}
        past = case["past"]
        s.k[:, past:], s.v[:, past:] = k.float(), v.float()
    if kind == "window":
        i = torch.arange(case["n"], device="cuda").unsqueeze(1) + case["pos0"]
        j = torch.arange(case["pos0"] + case["n"], device="cuda").unsqueeze(0)
        allowed = (j <= i) & ~((j >= case["sink"]) & (i - j >= case["window"]))
    else:
        allowed = torch.zeros(case["nodes"], case["past"] + case["nodes"], dtype=torch.bool)
        allowed[:, :case["past"]] = True
        for i in range(case["nodes"]):
            j = i
            while j >= 0:
                allowed[i, case["past"] + j] = True
                j = s.parent[j]
        allowed = allowed.cuda()
    k, v = s.k.double(), s.v.double()
    if case.get("type") == Q8_0:
        k, v = ((x.unflatten(-1, (4, 32)) * d.double().unsqueeze(-1)).flatten(-2).float().half().double()
                for x, d in ((k, s.dk), (v, s.dv)))
    if kind != "draft":
        return _exact_attention(s.q.double().view(-1, n_head, HEAD), k, v, n_head, allowed)
    out = _exact_attention(q, k, v, n_head, allowed)
    path = [past + i for i in s.path]
    s.k[:, past:past + len(path)], s.v[:, past:past + len(path)] = s.k[:, path], s.v[:, path]
    return {"q": q.flatten(1), "out": out, "k": s.k[:, past:].double(), "v": s.v[:, past:].double()}
