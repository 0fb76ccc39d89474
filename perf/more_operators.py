"""The operators of a step of several reads at once over one cache in pages, as timed cases: the tables and row maps made
on the device from the reads' lengths, the new rows' q / k norm, rotary turn and store at mapped rows, the attention of
each read's new tokens over its own pages, and the log probabilities of the tokens that were chosen.

A cache is one layer's, [n_kv][rows][128], in f16 or as q8_0 blocks of 32 values (int8 quants q and an f16 scale d, which
stand for f16(q·d); d the smallest f16 number with 127·d >= max |x|, q = x / d to the nearest integer, ties to even), its
rows cut into pages of 16 ... 256. A read's row i lies in row i % page of page table[read][i / page]. Free pages wait in a
ring [n_page], the pool's {head, count} say which of it. A read with d_new = -1 ends: its pages go back to the ring's end.

Each operator is here in its plain form too (elementary torch operations), which says what it computes; `own` picks the
framework's kernels. Inputs are synthetic: normed keys and queries ~ N(0, 1), values ~ N(0, 4^2), norm weights 1 + N(0,
0.02^2), as perf/operators.py has them; logits ~ N(0, 2.5^2) with one token of each row raised, as a read's mostly sure
choices have them.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

HEAD, EPS, ROPE_BASE = 128, 1e-6, 1e6
F16, Q8_0 = 1, 8  # the ggml types of a cache's rows
MODEL = dict(n_head=16, n_kv=8)  # the LightOnOCR decoder's heads
VOCAB = 151936  # and its vocabulary


def listed():
    return [
        # the maps of a decode step of 24 reads, all latency, and of the largest batch: 1000 reads of which some end, some
        # start with a page's prompt and some go on with a part of one
        dict(name="map_decode", kind="map", tokens=24, lo=700, hi=2600, chunks=0, chunk=0, past=0, ended=0, page=64, pad=0),
        dict(name="map_large", kind="map", tokens=800, lo=40, hi=6000, chunks=120, chunk=541, past=0, ended=80, page=16, pad=777),
        # the new rows of a decode step of 40 reads into an f16 cache; of a step that takes three pages' prompts in beside
        # 29 reads, into q8_0 rows
        dict(name="rows_decode", kind="rows", type=F16, tokens=40, lo=300, hi=2600, chunks=0, chunk=0, past=0, page=64, pad=8, **MODEL),
        dict(name="rows_prompts", kind="rows", type=Q8_0, tokens=29, lo=300, hi=2600, chunks=3, chunk=1925, past=0, page=32,
             pad=0, **MODEL),
        # one read's next token, all latency; a decode step of 64 reads between early and late, f16 and q8_0 rows; four
        # pages' prompts; a step that takes two chunks of long prompts in beside 61 tokens; many q heads on few KV heads,
        # whose reads are short
        dict(name="attend_token", kind="attend", type=F16, tokens=1, lo=1300, hi=1300, chunks=0, chunk=0, past=0, page=64, pad=0, **MODEL),
        dict(name="attend_reads", kind="attend", type=F16, tokens=64, lo=300, hi=6000, chunks=0, chunk=0, past=0, page=64, pad=0, **MODEL),
        dict(name="attend_reads_q8", kind="attend", type=Q8_0, tokens=64, lo=300, hi=6000, chunks=0, chunk=0, past=0, page=16, pad=0, **MODEL),
        dict(name="attend_prompts", kind="attend", type=F16, tokens=0, lo=0, hi=0, chunks=4, chunk=1925, past=0, page=128, pad=0, **MODEL),
        dict(name="attend_mixed", kind="attend", type=F16, tokens=61, lo=300, hi=2600, chunks=2, chunk=509, past=5003, page=16, pad=5, **MODEL),
        # a token's log probability and its alternatives; those of a decode step's reads; a page's tokens scored at once
        dict(name="score_token", kind="score", n=1, vocab=VOCAB, top=5),
        dict(name="score_reads", kind="score", n=61, vocab=VOCAB, top=20),
        dict(name="score_page", kind="score", n=1925, vocab=VOCAB, top=1),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["map", "rows", "attend", "attend", "attend", "attend", "score", "score"])
    if kind == "score":
        vocab = rng.choice([VOCAB, _log(rng, 257, VOCAB)])
        return dict(kind=kind, n=_log(rng, 1, 1925), vocab=vocab, top=rng.choice([0, 1, 3, 5, 20, 32]))
    lo = _log(rng, 1, 2000)
    b = dict(tokens=_log(rng, 1, 800 if kind == "map" else 64), lo=lo, hi=lo + _log(rng, 1, 4000), page=rng.choice([16, 32, 64, 128, 256]),
             pad=rng.choice([0, 0, rng.randint(1, 40)]), chunks=0, chunk=0, past=0)
    if rng.random() < 0.6:
        b.update(chunks=rng.randint(1, 4), chunk=_log(rng, 2, 1500), past=rng.choice([0, rng.randint(1, 4000)]))
        b["tokens"] = rng.choice([0, b["tokens"]])
    if kind == "map":
        return dict(kind=kind, ended=rng.choice([0, rng.randint(1, 60)]), **b)
    n_kv = rng.choice([1, 2, 4, 8, 8])
    case = dict(kind=kind, type=rng.choice([F16, Q8_0]), n_head=n_kv * rng.choice([1, 2, 2, 3, 4]), n_kv=n_kv, **b)
    while kind == "attend" and case["chunk"] > 2 and work(case)["flops"] > 6e10:  # no more than four pages' prompts
        case["chunk"] //= 2
    return case


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


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


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


def _lengths(case):
    """(rows held, new rows) of each read: the lengths of reads that take one token lie evenly on a log scale from lo to
    hi, chunks have the same past, ended reads a few pages; in an order of the case's own"""
    t, lo, hi = case["tokens"], case["lo"], case["hi"]
    reads = [(round(lo * (hi / lo) ** (i / max(t - 1, 1))), 1) for i in range(t)]
    reads += [(case["past"], case["chunk"] - i % 2) for i in range(case["chunks"])]
    reads += [(lo + 37 * i, -1) for i in range(case.get("ended", 0))]
    random.Random(1000 * t + case["page"] + case["chunk"]).shuffle(reads)
    return reads


def _pages(n, page):
    return -(-n // page)


def _map_inputs(s, seed):
    """the reads' lengths, their tables with the pages they hold, the ring of free pages"""
    c = s.case
    s.reads, page = _lengths(c), c["page"]
    g = _gen(seed, 31)
    s.n_row = sum(max(n, 0) for _, n in s.reads) + c["pad"]
    held = [_pages(p, page) for p, _ in s.reads]
    want = [max(h, _pages(p + max(n, 0), page)) for h, (p, n) in zip(held, s.reads)]
    s.max_pages = max(want) + 2
    s.n_page = sum(want) + 5
    order = torch.randperm(s.n_page, generator=g, device="cuda").int()
    s.table = torch.full((len(s.reads), s.max_pages), -1, dtype=torch.int32, device="cuda")
    here = torch.arange(s.max_pages, device="cuda")[None, :] < _int(held)[:, None]
    s.table[here] = order[:sum(held)]
    free = s.n_page - sum(held)
    head = int(torch.randint(s.n_page, (1,), generator=g, device="cuda"))
    s.ring = torch.full((s.n_page,), -1, dtype=torch.int32, device="cuda")
    s.ring[(head + torch.arange(free, device="cuda")) % s.n_page] = order[sum(held):]
    s.pool = _int([head, free])
    s.len, s.new = _int([p for p, _ in s.reads]), _int([n for _, n in s.reads])
    n = len(s.reads)
    s.start, s.past, s.len_out, s.pool_out = (torch.zeros(k, dtype=torch.int32, device="cuda") for k in (n + 1, n, n, 2))
    s.pos, s.slot = (torch.zeros(s.n_row, dtype=torch.int32, device="cuda") for _ in range(2))


def prepare(case, seed):
    s, kind = _State(case), case["kind"]
    g = _gen(seed, 32)
    if kind == "score":
        n, vocab = case["n"], case["vocab"]
        s.logits = _normal(g, n, vocab, std=2.5)
        sure = torch.randint(vocab, (n, 1), generator=g, device="cuda")
        s.logits.scatter_add_(1, sure, torch.rand(n, 1, generator=g, device="cuda") * 24)
        # the chosen token: the raised one, or any
        any_ = torch.randint(vocab, (n, 1), generator=g, device="cuda")
        s.ids = torch.where(torch.rand(n, 1, generator=g, device="cuda") < 0.8, sure, any_).int().flatten()
        s.logprob, s.entropy = (torch.zeros(n, device="cuda") for _ in range(2))
        s.top_ids = torch.zeros(n, case["top"], dtype=torch.int32, device="cuda")
        s.top_logprob = torch.zeros(n, case["top"], device="cuda")
        return s
    _map_inputs(s, seed)
    if kind == "map":
        return s
    _map_plain(s)  # the step's maps, which every layer's calls take
    n_head, n_kv, rows = case["n_head"], case["n_kv"], s.n_page * case["page"]
    s.out = torch.zeros(s.n_row, n_head * HEAD, device="cuda")
    if kind == "rows":
        s.qkv = _normal(g, s.n_row, (n_head + 2 * n_kv) * HEAD)  # the rows of the fused projections, [q | k | v]
        s.qkv[:, (n_head + n_kv) * HEAD:] *= 4.0
        s.q_norm, s.k_norm = _normal(g, HEAD, mean=1.0, std=0.02), _normal(g, HEAD, mean=1.0, std=0.02)
        s.rope = _rope(max(p + n for p, n in s.reads))
        if case["type"] == Q8_0:
            s.k, s.v = (torch.zeros(n_kv, rows, HEAD, dtype=torch.int8, device="cuda") for _ in range(2))
            s.dk, s.dv = (torch.zeros(n_kv, rows, 4, dtype=torch.float16, device="cuda") for _ in range(2))
            s.back_k, s.back_v = (torch.zeros(n_kv, rows, HEAD, dtype=torch.float16, device="cuda") for _ in range(2))
        else:
            s.k, s.v = (torch.zeros(n_kv, rows, HEAD, dtype=torch.float16, device="cuda") for _ in range(2))
            s.dk = s.dv = None
        return s
    s.q = _normal(g, s.n_row, n_head * HEAD)
    for x, d, std in (("k", "dk", 1.0), ("v", "dv", 4.0)):
        a = _normal(g, n_kv, rows, HEAD, std=std).half()
        a, b = _quantise(a) if case["type"] == Q8_0 else (a, None)
        setattr(s, x, a)
        setattr(s, d, b)
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
        ref = lambda t: None if t is None else _Ref(t)  # noqa: E731
        for name in ("len", "new", "ring", "pool", "len_out", "pool_out", "q", "out", "q_norm", "k_norm", "rope",
                     "logits", "ids", "logprob", "entropy"):
            if hasattr(s, name):
                setattr(self, name, _Ref(getattr(s, name)))
        if c["kind"] == "score":
            self.top_ids, self.top_logprob = (ref(t) if c["top"] else None for t in (s.top_ids, s.top_logprob))
            return
        self.pages = htr.Pages.of(len(s.reads), s.n_row, c["page"], s.max_pages, _Ref(s.start), _Ref(s.past), _Ref(s.table),
                                  _Ref(s.pos), _Ref(s.slot))
        if c["kind"] == "map":
            return
        cache = lambda k, v, dk, dv: htr.KvCache.of(k.shape[0], k.shape[1], _Ref(k), _Ref(v), ref(dk), ref(dv))  # noqa: E731
        self.kv = cache(s.k, s.v, s.dk, s.dv)
        if hasattr(s, "back_k"):
            self.back = cache(s.back_k, s.back_v, None, None)
        if hasattr(s, "qkv"):
            self.raw = [_Ref(s.qkv, 4 * HEAD * h) for h in (0, c["n_head"], c["n_head"] + c["n_kv"])]


def _run_own(s):
    htr, dev, c, kind = _htr(), _dev(), s.case, s.case["kind"]
    if s.held is None:
        s.held = _Held(s)
    h = s.held
    if kind == "map":
        htr.page_map(dev, h.pages, s.n_page, h.len, h.new, h.ring, h.pool, h.len_out, h.pool_out)
        return _map_out(s)
    if kind == "rows":
        width = s.qkv.shape[1]
        htr.qkv_post_pages(dev, h.raw[0], h.raw[1], h.raw[2], h.pages, h.q_norm, h.k_norm, h.rope, s.rope.shape[0], c["n_head"],
                           EPS, h.kv, h.out, q_stride=width, kv_stride=width)
        if s.dk is None:
            return {"q": s.out, "k": s.k, "v": s.v}
        htr.kv_copy(dev, h.kv, 0, h.back, 0, s.back_k.shape[1])
        return {"q": s.out, "k": s.back_k, "v": s.back_v}
    if kind == "attend":
        htr.page_attention(dev, h.q, h.pages, h.kv, c["n_head"], HEAD ** -0.5, h.out)
        return s.out
    htr.token_logprobs(dev, h.logits, c["n"], c["vocab"], h.ids, h.logprob, h.entropy, c["top"], h.top_ids, h.top_logprob)
    return {"logprob": s.logprob, "entropy": s.entropy, "top_ids": s.top_ids, "top_logprob": s.top_logprob}


# ---- the plain forms -------------------------------------------------------------------------------------------------

def _map_out(s):
    return {"start": s.start, "past": s.past, "table": s.table, "pos": s.pos, "slot": s.slot, "ring": s.ring,
            "len": s.len_out, "pool": s.pool_out}


def _map_plain(s):
    """Reads in order: one whose rows fit the table's width and the step's buffers is served if the free pages that it and
    those before it need are there (or it needs none); one that is not keeps its length, its past is -1, and its rows have no
    place. The pages of ended reads go behind the free ones, and are not yet given out."""
    page, mp, npg = s.case["page"], s.max_pages, s.n_page
    length, new = s.len.long(), s.new.long()
    head, count = s.pool.long()
    ends, n = new < 0, new.clamp_min(0)
    end = n.cumsum(0)
    held = (length + page - 1) // page
    fits = ~ends & (length + n <= mp * page) & (end <= s.n_row)
    need = torch.where(fits, (length + n + page - 1) // page - held, 0)
    upto = need.cumsum(0)
    served = fits & ((need == 0) | (upto <= count))
    taken = torch.where(served & (need > 0), upto, 0).amax()
    k = torch.arange(mp, device="cuda")[None, :]
    back = torch.where(ends, held, 0)
    old = s.table.clone()
    fresh = served[:, None] & (k >= held[:, None]) & (k < (held + need)[:, None])
    at = (head + (upto - need - held)[:, None] + k) % npg
    s.table.copy_(torch.where(fresh, s.ring[at], s.table))
    gone = ends[:, None] & (k < held[:, None])
    at = (head + count + (back.cumsum(0) - back)[:, None] + k) % npg
    s.ring[at[gone]] = old[gone]
    s.pool_out.copy_(torch.stack([(head + taken) % npg, count - taken + back.sum()]))
    s.len_out.copy_(torch.where(ends, 0, torch.where(served, length + n, length)))
    s.past.copy_(torch.where(served, length, -1))
    s.start[0] = 0
    s.start[1:] = end.clamp_max(s.n_row)
    row = torch.arange(s.n_row, device="cuda")
    read = torch.searchsorted(s.start[1:].long(), row, right=True)
    there = read < len(s.reads)
    read = read.clamp_max(len(s.reads) - 1)
    there &= s.past[read] >= 0
    pos = s.past[read] + row - s.start[read]
    s.pos.copy_(torch.where(there, pos, -1))
    p = s.pos.clamp_min(0).long()
    s.slot.copy_(torch.where(there, s.table[read, p // page] * page + p % page, -1))


def _post(x, w, cs):
    """rows x [n, heads, 128]: each head's RMS norm with weights w, then the pairs (i, i + 64) turned by cs [n, 64, 2]. In
    64 bits: the results are rounded to the cache's types, and lie next to a border of theirs now and then"""
    x = x.double()
    y = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
    a, b = y[..., :64], y[..., 64:]
    c, t = cs.double()[:, None, :, 0], cs.double()[:, None, :, 1]
    return torch.cat([a * c - b * t, a * t + b * c], dim=-1)


def _rows_plain(s):
    c, n = s.case, s.n_row - s.case["pad"]  # the rows behind the last read are left as they were
    n_head, n_kv = c["n_head"], c["n_kv"]
    pos, slot = s.pos[:n].long(), s.slot[:n].long()
    x, cs = s.qkv[:n].view(n, n_head + 2 * n_kv, HEAD), s.rope[pos]
    s.out[:n] = _post(x[:, :n_head], s.q_norm, cs).flatten(1).float()
    k, v = _post(x[:, n_head:n_head + n_kv], s.k_norm, cs).float(), x[:, n_head + n_kv:]
    if s.dk is None:
        s.k[:, slot], s.v[:, slot] = k.transpose(0, 1).half(), v.transpose(0, 1).half()
        return {"q": s.out, "k": s.k, "v": s.v}
    for y, to, d, back in ((k, s.k, s.dk, s.back_k), (v, s.v, s.dv, s.back_v)):
        to[:, slot], d[:, slot] = _quantise(y.transpose(0, 1))
        back.copy_(_values(to, d))
    return {"q": s.out, "k": s.back_k, "v": s.back_v}


def _attend_plain(s):
    c = s.case
    n_head, n_kv, page = c["n_head"], c["n_kv"], c["page"]
    at = 0
    for i, (past, n) in enumerate(s.reads):
        keys = past + n
        j = torch.arange(keys, device="cuda")
        row = s.table[i, j // page].long() * page + j % page
        k, v = s.k[:, row], s.v[:, row]
        if s.dk is not None:
            k, v = _values(k, s.dk[:, row]), _values(v, s.dv[:, row])
        q = (s.q[at:at + n] * HEAD ** -0.5).view(n, n_kv, n_head // n_kv, HEAD).transpose(0, 1).reshape(n_kv, -1, HEAD)
        score = torch.matmul(q, k.float().transpose(1, 2).contiguous()).view(n_kv, n, n_head // n_kv, keys)
        seen = j[None, :] <= past + torch.arange(n, device="cuda")[:, None]
        score = torch.where(seen[None, :, None, :], score, -math.inf)
        p = (score - score.amax(-1, keepdim=True)).exp()
        o = torch.matmul(p.flatten(1, 2), v.float()).view(n_kv, n, -1, HEAD) / p.sum(-1, keepdim=True)
        s.out[at:at + n] = o.transpose(0, 1).reshape(n, -1)
        at += n
    return s.out


def _score_plain(s):
    """logprob = x - log Σ e^x, entropy = Σ p·(log Σ e^x - x). In 64 bits: a sure token's log probability and entropy are the
    small differences of large numbers; some rows at a time"""
    top = s.case["top"]
    for a in range(0, s.case["n"], 128):
        rows = slice(a, min(a + 128, s.case["n"]))
        x = s.logits[rows].double()
        e = (x - x.amax(-1, keepdim=True)).exp()
        total = e.sum(-1, keepdim=True)
        lp = x - x.amax(-1, keepdim=True) - total.log()
        s.logprob[rows] = lp.gather(1, s.ids[rows, None].long()).flatten().float()
        s.entropy[rows] = -(e / total * lp).sum(-1).float()
        if top:  # the largest logits, of equal ones the lower id first
            b = s.logits[rows].view(torch.int32).long()
            key = torch.where(b < 0, -(b & 0x7FFFFFFF), b) * 2 ** 31 + (2 ** 31 - 1 - torch.arange(x.shape[1], device="cuda"))
            ids = key.topk(top, dim=1).indices
            s.top_ids[rows] = ids.int()
            s.top_logprob[rows] = lp.gather(1, ids).float()
    return {"logprob": s.logprob, "entropy": s.entropy, "top_ids": s.top_ids, "top_logprob": s.top_logprob}


def run(s):
    if own:
        return _run_own(s)
    kind = s.case["kind"]
    if kind == "map":
        _map_plain(s)
        return _map_out(s)
    return _rows_plain(s) if kind == "rows" else _attend_plain(s) if kind == "attend" else _score_plain(s)


# ---- what a case cannot do without -----------------------------------------------------------------------------------

def _row_bytes(t):
    """K and V of one position of one KV head"""
    return 2 * (HEAD + 8 if t == Q8_0 else 2 * HEAD)


def work(case):
    kind = case["kind"]
    if kind == "score":
        n, vocab, top = case["n"], case["vocab"], case["top"]
        return {"bytes": n * (4 * vocab + 12 + 8 * top), "flops": 6 * n * vocab}
    reads, page = _lengths(case), case["page"]
    rows = sum(max(n, 0) for _, n in reads)
    if kind == "map":
        moved = sum(_pages(p, page) if n < 0 else _pages(p + n, page) - _pages(p, page) for p, n in reads)
        # a read's length, new rows, start, past and new length; its pages out of or into the ring; a row's page, place and slot
        return {"bytes": 20 * len(reads) + 8 * moved + 12 * rows + 8 * case["pad"], "flops": 12 * len(reads) + 8 * rows}
    n_head, n_kv = case["n_head"], case["n_kv"]
    if kind == "rows":
        # the raw q, k and v, (cos, sin), position and slot; its q and its cache row written (q8_0 rows are read back too)
        made = 4 * HEAD * (n_head + 2 * n_kv) + 4 * HEAD + 8 + 4 * HEAD * n_head + n_kv * _row_bytes(case["type"])
        if case["type"] == Q8_0:
            made += n_kv * (_row_bytes(Q8_0) + _row_bytes(F16))
        return {"bytes": rows * made, "flops": rows * HEAD * (n_head + 2 * n_kv) * 12}
    keys = sum(p + n for p, n in reads)
    pairs = sum(n * p + n * (n + 1) // 2 for p, n in reads)
    return {"bytes": keys * n_kv * _row_bytes(case["type"]) + 2 * rows * 4 * HEAD * n_head, "flops": 4 * HEAD * n_head * pairs}


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


def _exact_heads(x, w, turn):
    """RMS norm and turn of the heads x [n, heads, 128] by turn [n, 64, 2], as complex numbers"""
    x = x.double()
    x = x * torch.rsqrt((x * x).sum(dim=2, keepdim=True) / HEAD + EPS) * w.double()
    z = torch.complex(x[:, :, :64].contiguous(), x[:, :, 64:].contiguous())
    turn = turn.double()
    z = z * torch.complex(turn[..., 0].contiguous(), turn[..., 1].contiguous())[:, None, :]
    return torch.cat([z.real, z.imag], dim=2)


def _exact_rows(s):
    """row by read: the read's own positions, its pages from the table"""
    c = s.case
    n_head, n_kv, page, q8 = c["n_head"], c["n_kv"], c["page"], c["type"] == Q8_0
    q_out = torch.zeros(s.n_row, n_head * HEAD, dtype=torch.float64, device="cuda")
    kv_out = [torch.zeros(*s.k.shape, dtype=torch.float64, device="cuda") for _ in range(2)]
    at = 0
    for (past, n), pages in zip(s.reads, s.table.tolist()):
        x = s.qkv[at:at + n].unflatten(1, (n_head + 2 * n_kv, HEAD))
        turn = s.rope[past:past + n]
        q_out[at:at + n] = _exact_heads(x[:, :n_head], s.q_norm, turn).flatten(1)
        rows = torch.tensor([pages[p // page] * page + p % page for p in range(past, past + n)], device="cuda")
        for to, y in zip(kv_out, (_exact_heads(x[:, n_head:n_head + n_kv], s.k_norm, turn), x[:, n_head + n_kv:].double())):
            y = y.permute(1, 0, 2)
            to[:, rows] = _exact_blocks(y.float()) if q8 else y
        at += n
    return {"q": q_out, "k": kv_out[0], "v": kv_out[1]}


def _exact_attend(s):
    c = s.case
    n_head, n_kv, page = c["n_head"], c["n_kv"], c["page"]
    out = torch.zeros(s.n_row, n_head, HEAD, dtype=torch.float64, device="cuda")
    at = 0
    for (past, n), pages in zip(s.reads, s.table.tolist()):
        parts = [slice(pages[a // page] * page, pages[a // page] * page + min(page, past + n - a)) for a in range(0, past + n, page)]
        future = torch.arange(past + n, device="cuda") > torch.arange(past, past + n, device="cuda").unsqueeze(1)
        for j in range(n_kv):
            k, v = (torch.cat([x[j, r] for r in parts]).double() for x in (s.k, s.v))
            if c["type"] == Q8_0:
                dk, dv = (torch.cat([x[j, r] for r in parts]).double().repeat_interleave(32, dim=1) for x in (s.dk, s.dv))
                k, v = (k * dk).float().half().double(), (v * dv).float().half().double()
            kt = k.t().contiguous()
            for h in range(j * n_head // n_kv, (j + 1) * n_head // n_kv):
                t = s.q[at:at + n, h * HEAD:(h + 1) * HEAD].double() @ kt / math.sqrt(HEAD)
                out[at:at + n, h] = torch.softmax(t.masked_fill_(future, -math.inf), dim=1) @ v
        at += n
    return out.flatten(1)


def _exact_score(s):
    out = {"logprob": [], "entropy": [], "top_ids": None, "top_logprob": []}
    for a in range(0, s.case["n"], 256):
        lp = torch.log_softmax(s.logits[a:a + 256].double(), dim=1)
        out["logprob"].append(lp[torch.arange(lp.shape[0], device="cuda"), s.ids[a:a + 256].long()])
        out["entropy"].append(-(lp.exp() * lp).sum(1))
        out["top_logprob"].append(lp.topk(s.case["top"], dim=1).values if s.case["top"] else lp[:, :0])
    return {k: v if v is None else torch.cat(v) for k, v in out.items()}


def exact(case, seed):
    kind = case["kind"]
    if kind == "map":
        return None  # whole numbers: the plain form's
    s = prepare(case, seed)
    return _exact_rows(s) if kind == "rows" else _exact_attend(s) if kind == "attend" else _exact_score(s)
