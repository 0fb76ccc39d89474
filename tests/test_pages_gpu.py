"""The operators of a step of several reads over a cache in pages on the GPU against plain numpy in 64 bits: the tables and row
maps, rows stored at mapped slots, each read's attention over its pages, and a serving loop of them together, eager and replayed
as one recorded step."""
import os
import re

import numpy as np
import pytest

import htr
from test_kernel_waits import PKG
from test_kv_ops_gpu import BAR, EPS, SCALE, Cache, attention, bits, blocks, cache, heads, normal, rel_rows, strided, values

pytestmark = pytest.mark.gpu


# ---- plain forms ----------------------------------------------------------------------------------------------------------

def cdiv(a, b):
    return -(-a // b)


class Serving:
    """the state of a program that serves reads, and htr_page_map's definition on it, read by read"""

    def __init__(self, n_seq, n_row, page, max_pages, n_page, seed=0):
        self.n_seq, self.n_row, self.page, self.max_pages, self.n_page = n_seq, n_row, page, max_pages, n_page
        rng = np.random.default_rng(seed)
        self.ring = rng.permutation(n_page).astype(np.int32)
        self.head, self.count = int(rng.integers(n_page)), n_page
        self.len = np.zeros(n_seq, np.int64)
        self.table = np.full((n_seq, max_pages), -1, np.int32)

    def step(self, new):
        """→ start, past, pos, slot; the state after the step"""
        start, past = np.zeros(self.n_seq + 1, np.int64), np.full(self.n_seq, -1, np.int64)
        ask, taken, back, total = 0, 0, [], 0
        for b, n in enumerate(new):
            held = cdiv(max(int(self.len[b]), 0), self.page)
            if n < 0:
                back += list(self.table[b, :min(held, self.max_pages)])
                self.len[b] = 0
            else:
                total += int(n)
                want = cdiv(int(self.len[b] + n), self.page)
                if self.len[b] >= 0 and self.len[b] + n <= self.max_pages * self.page and total <= self.n_row:
                    ask += want - held
                    if want == held or ask <= self.count:
                        for k in range(held, want):
                            self.table[b, k] = self.ring[(self.head + ask - (want - k)) % self.n_page]
                        if want > held:
                            taken = ask
                        past[b] = self.len[b]
                        self.len[b] += n
            start[b + 1] = min(total, self.n_row)
        for i, p in enumerate(back):
            self.ring[(self.head + self.count + i) % self.n_page] = p
        self.head, self.count = (self.head + taken) % self.n_page, self.count - taken + len(back)
        pos, slot = np.full(self.n_row, -1, np.int64), np.full(self.n_row, -1, np.int64)
        for b in range(self.n_seq):
            if past[b] >= 0:
                for i, r in enumerate(range(start[b], start[b + 1])):
                    pos[r] = past[b] + i
                    p = self.table[b, pos[r] // self.page]
                    slot[r] = p * self.page + pos[r] % self.page if 0 <= p < self.n_page else -1
        return start, past, pos, slot


class OnDevice:
    """the same state on the device; in place: the lengths and the pool are replaced by a step's"""

    def __init__(self, dev, s, in_place=True):
        self.dev, self.s = dev, s
        self.pages = htr.Pages(dev, s.n_seq, s.n_row, s.page, s.max_pages)
        self.pages.table.upload(s.table)
        up = lambda a: dev.upload(np.ascontiguousarray(a, np.int32))  # noqa: E731
        self.len, self.new, self.ring, self.pool = up(s.len), up(np.zeros(s.n_seq)), up(s.ring), up([s.head, s.count])
        self.len_out, self.pool_out = (self.len, self.pool) if in_place else (up(np.zeros(s.n_seq)), up([0, 0]))

    def map(self):
        htr.page_map(self.dev, self.pages, self.s.n_page, self.len, self.new, self.ring, self.pool, self.len_out, self.pool_out)

    def step(self, new):
        self.new.upload(np.ascontiguousarray(new, np.int32))
        self.map()

    def check(self, want):
        s, p = self.s, self.pages
        for buf, w, what in zip((p.start, p.past, p.pos, p.slot), want, ("start", "past", "pos", "slot")):
            np.testing.assert_array_equal(buf.download(np.int32, w.size), w, err_msg=what)
        np.testing.assert_array_equal(p.table.download(np.int32, s.table.size).reshape(s.table.shape), s.table)
        np.testing.assert_array_equal(self.len_out.download(np.int32, s.n_seq), s.len)
        np.testing.assert_array_equal(self.pool_out.download(np.int32, 2), [s.head, s.count])
        np.testing.assert_array_equal(self.ring.download(np.int32, s.n_page), s.ring)

    def free(self):
        for b in {id(b): b for b in (self.len, self.new, self.ring, self.pool, self.len_out, self.pool_out)}.values():
            b.free()
        self.pages.free()


# ---- tables and maps ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("n_seq,n_row,page,max_pages,n_page,steps", [
    (1, 1, 16, 1, 1, [[1], [1], [0], [-1], [1]]),
    (3, 40, 16, 4, 5, [[17, 0, 16], [1, 3, 1], [-1, 20, 0], [5, 1, 40], [30, -1, 1], [0, 0, 0], [-1, -1, -1], [40, 0, 0]]),
    # the second read is too long for the table, the third for the step, the fourth finds no pages left, the fifth needs none
    (6, 70, 32, 2, 4, [[40, 65, 64, 20, 0, 2], [24, 1, 7, 20, 0, 2], [1, 1, 1, 1, 1, 1], [-1, 64, 0, 6, 0, 0], [3, 3, 3, 3, 3, 3]]),
    (65, 5000, 64, 9, 300, [[(7 * i) % 97 for i in range(65)], [1] * 65, [-1 if i % 3 == 0 else 2 for i in range(65)],
                            [64 if i % 3 == 0 else 1 for i in range(65)]]),
    (1024, 4096, 16, 3, 2100, [[i % 5 for i in range(1024)], [1] * 1024, [-1] * 1024, [4] * 1024]),
    (1000, 40000, 128, 4, 1500, [[37 + i % 4 for i in range(1000)], [(31 * i) % 60 - 1 for i in range(1000)], [1] * 1000])])
@pytest.mark.parametrize("in_place", [True, False])
def test_map(dev, n_seq, n_row, page, max_pages, n_page, steps, in_place):
    s = Serving(n_seq, n_row, page, max_pages, n_page, seed=n_seq)
    d = OnDevice(dev, s, in_place)
    for new in steps:
        want = s.step(new)
        d.step(new)
        d.check(want)
        if not in_place:
            d.map()  # the same step again, over the same lengths: the same tables
            d.check(want)
            d.len, d.len_out, d.pool, d.pool_out = d.len_out, d.len, d.pool_out, d.pool
    d.free()


def test_map_of_lengths_and_pools_that_are_none(dev):
    """lengths below 0 and past the table, a pool of more pages than there are, new rows whose sum passes 32 bits: each read
    as the definition has it, nothing written past an array"""
    s = Serving(5, 50, 16, 4, 8, seed=3)
    s.len[:] = [-5, 65, 2 ** 31 - 1, 10, -7]
    s.table[3, 0] = 6
    d = OnDevice(dev, s)
    for b in (d.ring, d.pages.table):
        assert b is not None
    want = s.step([1, 1, 2 ** 31 - 1, 7, -1])
    d.step([1, 1, 2 ** 31 - 1, 7, -1])
    assert want[1].tolist() == [-1, -1, -1, -1, -1]  # (the third read's rows fill the step)
    d.check(want)
    d.free()
    s = Serving(2, 50, 16, 4, 8, seed=4)
    d = OnDevice(dev, s)
    d.pool.upload(np.array([s.head + 8, 100], np.int32))
    want = s.step([20, 30])
    d.step([20, 30])
    d.check(want)
    s.table[1, 1] = 8  # (a page that the cache does not have)
    d.pages.table.upload(s.table)
    want = s.step([1, 2])
    assert want[3].tolist()[:3] == [int(s.table[0, 1]) * 16 + 4, -1, -1]
    d.step([1, 2])
    d.check(want)
    d.free()


# ---- rows -----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("q8_0", [False, True], ids=["f16", "q8_0"])
@pytest.mark.parametrize("n_row,n_head,n_kv,page,gap,in_place", [
    (1, 16, 8, 64, 0, False), (1, 1, 1, 16, 4, False), (67, 6, 2, 16, 12, False), (200, 4, 4, 32, 0, True), (333, 16, 8, 128, 8, False)])
def test_rows_at_slots(dev, q8_0, n_row, n_head, n_kv, page, gap, in_place):
    """bit for bit what the rows are by the definition; rows without a place, q outputs of rows without a position and all else
    of the cache stay as they were"""
    rng = np.random.default_rng(n_row + n_head)
    n_page, n_pos = cdiv(n_row, page) + 3, 2 * n_row + 5
    n_ctx = n_page * page + 7
    pos = rng.permutation(n_pos)[:n_row].astype(np.int32)
    slot = rng.permutation(n_ctx)[:n_row].astype(np.int32)
    if n_row > 1:
        pos[3], pos[n_row - 1], pos[7] = -1, n_pos, -2 ** 31
        slot[5], slot[n_row // 2], slot[8] = -1, n_ctx, 2 ** 31 - 1
    x = normal(n_row, n_row, n_head + 2 * n_kv, 128)
    x[:, n_head + n_kv:] *= 4
    qn, kn = 1 + 0.02 * normal(1, 128), 1 + 0.02 * normal(2, 128)
    ang = np.arange(n_pos)[:, None] * 1e6 ** (-np.arange(64) / 64.0)
    rope = np.stack([np.cos(ang), np.sin(ang)], axis=2).astype(np.float32)
    has_pos = (pos >= 0) & (pos < n_pos)
    kept = has_pos & (slot >= 0) & (slot < n_ctx)
    cs = rope[np.where(has_pos, pos, 0)]
    q, k = heads(x[:, :n_head], qn, cs), heads(x[:, n_head:n_head + n_kv], kn, cs)
    c = cache(dev, 5, n_kv, n_ctx, q8_0)
    want = {"k": c.rows("k"), "v": c.rows("v")}
    for w, y in (("k", k), ("v", x[:, n_head + n_kv:])):
        y = y[kept].transpose(1, 0, 2)
        for to, new in zip(want[w] if q8_0 else (want[w],), blocks(y) if q8_0 else (y.astype(np.float16),)):
            to[:, slot[kept]] = new
    raw = [np.ascontiguousarray(a.reshape(n_row, -1)) for a in (x[:, :n_head], x[:, n_head:n_head + n_kv], x[:, n_head + n_kv:])]
    bufs = [strided(dev, a, 0 if in_place else gap) for a in raw]
    before = raw[0] if in_place else normal(9, n_row, n_head * 128)
    out = bufs[0] if in_place else dev.upload(before)
    others = [dev.upload(a) for a in (qn.astype(np.float32), kn.astype(np.float32), rope, pos, slot)]
    p = htr.Pages.of(1, n_row, page, n_page, others[3], others[3], others[3], others[3], others[4])
    g = 0 if in_place else gap
    htr.qkv_post_pages(dev, *bufs, p, others[0], others[1], others[2], n_pos, n_head, EPS, c.kv, out,
                       q_stride=n_head * 128 + g, kv_stride=n_kv * 128 + g)
    got = out.download(np.float32, n_row * n_head * 128).reshape(n_row, -1)
    ulp = np.spacing(np.abs(q.reshape(n_row, -1)))
    assert np.all(np.abs(got - q.reshape(n_row, -1))[has_pos] <= ulp[has_pos])
    np.testing.assert_array_equal(bits(got)[~has_pos], bits(before)[~has_pos])
    for w in "kv":
        for a, b in zip(*((c.rows(w), want[w]) if q8_0 else ((c.rows(w),), (want[w],)))):
            np.testing.assert_array_equal(bits(a), bits(b))
    for b in (*bufs, *others, *(() if in_place else (out,))):
        b.free()
    c.free()


# ---- attention ------------------------------------------------------------------------------------------------------------

class Reads:
    """reads of (past, new) rows with pages in an order of their own, over caches whose other rows are NaN"""

    def __init__(self, dev, reads, page, n_kv, q8_0=False, seed=0, spare=2, pad=0, std=1.0):
        self.dev, self.reads, self.page = dev, reads, page
        rng = np.random.default_rng(seed)
        n_pages = [cdiv(max(p, 0) + n, page) for p, n in reads]
        self.n_page, self.max_pages = sum(n_pages) + spare, max(max(n_pages), 1)
        order = rng.permutation(self.n_page).astype(np.int32)
        self.table, at = np.full((len(reads), self.max_pages), -1, np.int32), 0
        for b, n in enumerate(n_pages):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.start = np.concatenate([[0], np.cumsum([n for _, n in reads])]).astype(np.int32)
        self.n = int(self.start[-1])
        self.n_row = max(self.n + pad, 1)
        n_ctx = self.n_page * page
        seen = np.zeros(n_ctx, bool)
        self.rows = []
        for b, (p, n) in enumerate(reads):
            j = np.arange(max(p, 0) + n)
            self.rows.append(self.table[b, j // page] * page + j % page)
            seen[self.rows[-1]] = True
        k, v = normal(seed, n_kv, n_ctx, 128, std=std).astype(np.float16), normal(seed + 1, n_kv, n_ctx, 128, std=4.0).astype(np.float16)
        k[:, ~seen], v[:, ~seen] = np.nan, np.inf
        self.cache = Cache(dev, k, v, q8_0)
        up = lambda a: dev.upload(np.ascontiguousarray(a, np.int32))  # noqa: E731
        self.bufs = [up(self.start), up([p for p, _ in reads]), up(self.table)]
        self.pages = htr.Pages.of(len(reads), self.n_row, page, self.max_pages, *self.bufs)

    def want(self, q, scale):
        out = np.zeros((self.n, q.shape[1] * 128))
        for b, (p, n) in enumerate(self.reads):
            if p < 0 or n == 0:
                continue
            r = self.rows[b]
            seen = np.arange(p + n)[None, :] <= p + np.arange(n)[:, None]
            out[self.start[b]:self.start[b + 1]] = attention(q[self.start[b]:self.start[b + 1]], self.cache.k[:, r], self.cache.v[:, r],
                                                             seen, scale)
        return out

    def run(self, q, n_head, scale=SCALE, gap=0, fill=7.5):
        full = np.full((self.n_row, n_head * 128), np.nan, np.float32)  # rows behind the last read are read by nobody
        full[:self.n] = q.reshape(self.n, n_head * 128)
        qb = strided(self.dev, full, gap)
        out = self.dev.upload(np.full((self.n_row, n_head * 128), fill, np.float32))
        htr.page_attention(self.dev, qb, self.pages, self.cache.kv, n_head, scale, out, q_stride=n_head * 128 + gap)
        got = out.download(np.float32, self.n_row * n_head * 128).reshape(self.n_row, -1)
        qb.free()
        out.free()
        assert np.all(got[self.n:] == np.float32(fill))  # those rows stay as they were
        return got[:self.n]

    def free(self):
        for b in self.bufs:
            b.free()
        self.cache.free()


BATCHES = [
    # one token of one read: its own key alone, a page's border, a long read
    ([(0, 1)], 16, 2, 1), ([(15, 1)], 16, 2, 1), ([(16, 1)], 16, 2, 1), ([(1000, 1)], 64, 16, 8), ([(12345, 1)], 32, 4, 2),
    # tokens of many reads, some of which have no new rows or are not served
    ([(37 * i % 611, 1) for i in range(70)], 16, 16, 8), ([(100, 1), (5, 0), (-1, 3), (0, 1), (255, 1), (-1, 0), (63, 1)], 64, 6, 2),
    ([(-1, 2), (-1, 1)], 16, 2, 2), ([(0, 0), (9, 0)], 16, 2, 2), ([(3, 1)] + [(9, 0)] * 130 + [(300, 1), (17, 2)], 16, 4, 4),
    # prompts, chunks over rows held, all lengths around the tiles
    ([(0, 31), (0, 32), (0, 33), (0, 1), (0, 15), (0, 16), (0, 17)], 32, 4, 2), ([(0, 200)], 128, 16, 8), ([(500, 77), (64, 64)], 64, 8, 8),
    ([(0, 3), (129, 65), (1000, 1), (31, 34), (-1, 40), (2, 190)], 16, 12, 4),
    # other groups of q heads, a KV head alone, more KV heads than the card has parts for
    ([(70, 5), (0, 9), (333, 1)], 32, 5, 1), ([(70, 5), (0, 9), (333, 1)], 32, 40, 1), ([(40, 3), (7, 1)], 16, 600, 600),
    ([(600, 1), (17, 4)], 1024, 7, 7), ([(2000, 130), (3000, 1), (2999, 1)], 256, 6, 2),
]


@pytest.mark.parametrize("q8_0", [False, True], ids=["f16", "q8_0"])
@pytest.mark.parametrize("reads,page,n_head,n_kv", BATCHES, ids=[f"{i}" for i in range(len(BATCHES))])
def test_attention(dev, reads, page, n_head, n_kv, q8_0):
    """against 64 bits; what a row does not see is NaN or an infinity; rows behind the last read stay as they were"""
    r = Reads(dev, reads, page, n_kv, q8_0, seed=len(reads) + page, pad=3)
    q = normal(77, r.n, n_head, 128)
    got = r.run(q, n_head, gap=4)
    if r.n:
        assert rel_rows(got, r.want(q, SCALE)) < BAR
        assert np.array_equal(bits(got), bits(r.run(q, n_head)))  # the same bits every time
    r.free()


@pytest.mark.parametrize("q8_0", [False, True], ids=["f16", "q8_0"])
@pytest.mark.parametrize("n_head,n_kv,reads", [
    (16, 8, [(9000, 1)]), (16, 8, [(5000, 1), (-1, 1), (3000, 2), (0, 1), (17, 3), (700, 1)]), (8, 8, [(4000, 32)]),
    (48, 16, [(2100, 1), (2100, 1), (33, 2), (6000, 3)]), (64, 8, [(2500, 1), (1300, 3)]), (24, 24, [(1700, 1)] * 30),
    # reads of many rows among those of few: several tiles to a read
    (16, 8, [(300, 50)] + [(5, 0)] * 14 + [(900, 1)]), (8, 8, [(2, 0)] * 30 + [(-1, 1), (0, 100), (1900, 20)]),
    (16, 8, [(37 * i % 900, 1) for i in range(190)] + [(700, 30), (0, 12)]), (16, 8, [(9, 0)] * 70 + [(2500, 33), (64, 40), (-1, 9)]),
    (8, 8, [(9, 0)] * 70 + [(2500, 33), (64, 40), (-1, 9)] + [(3, 1)] * 30)])
def test_attention_of_few_rows(dev, n_head, n_kv, reads, q8_0):
    """rows that one launch takes: the parts of a cut tile joined by the last of its workgroups, call after call, eager and replayed"""
    r = Reads(dev, reads, 32, n_kv, q8_0, seed=n_head)
    q = normal(31, r.n, n_head, 128)
    got = r.run(q, n_head)
    assert rel_rows(got, r.want(q, SCALE)) < BAR
    qb, out = dev.upload(q), dev.alloc(q.nbytes)
    dev.capture_begin()
    htr.page_attention(dev, qb, r.pages, r.cache.kv, n_head, SCALE, out)
    g = dev.capture_end()
    for i in range(5):
        out.upload(np.full(q.size, 2.5, np.float32))
        for _ in range(8):
            g.launch()
        np.testing.assert_array_equal(bits(out.download(np.float32, q.size)), bits(got.ravel()))
        np.testing.assert_array_equal(bits(r.run(q, n_head)), bits(got))
    for b in (g, qb, out):
        b.free()
    r.free()


def test_attention_of_many_reads(dev):
    """1024 reads, of which the last 24 hold more rows"""
    reads = [(i % 40, 1) for i in range(1000)] + [(400 + 13 * i, 1 + i % 3) for i in range(24)]
    r = Reads(dev, reads, 16, 2, seed=8)
    q = normal(5, r.n, 4, 128)
    assert rel_rows(r.run(q, 4), r.want(q, SCALE)) < BAR
    r.free()


@pytest.mark.parametrize("q8_0", [False, True], ids=["f16", "q8_0"])
@pytest.mark.parametrize("reads,n_head,n_kv", [
    ([(20000, 300)], 2, 1),                 # wide tiles cut into many parts each, and the rows behind them
    ([(9000, 16)], 2, 1),                   # a narrow one of 32 rows
    ([(7000, 64), (3, 1), (0, 66)], 2, 1),  # whole tiles of 128 rows and one of 4 more
    ([(5000, 1), (30, 130), (6000, 1)], 2, 1)])
def test_attention_of_tiles_in_many_parts(dev, reads, n_head, n_kv, q8_0):
    r = Reads(dev, reads, 64, n_kv, q8_0, seed=21, pad=1)
    q = normal(22, r.n, n_head, 128)
    got = r.run(q, n_head)
    assert rel_rows(got, r.want(q, SCALE)) < BAR
    assert np.array_equal(bits(got), bits(r.run(q, n_head)))
    r.free()


@pytest.mark.parametrize("seed", range(8))
def test_attention_of_any_batch(dev, seed):
    rng = np.random.default_rng(seed)
    n_kv = int(rng.choice([1, 2, 3, 8]))
    n_head = n_kv * int(rng.choice([1, 2, 3, 5, 17]))
    reads = []
    for _ in range(int(rng.integers(1, 30))):
        kind = rng.random()
        past = int(2 ** rng.uniform(0, 11)) - 1
        reads.append((past, 1) if kind < 0.5 else (past, int(2 ** rng.uniform(0, 7))) if kind < 0.85 else (past, 0) if kind < 0.92 else
                     (-1, int(rng.integers(0, 5))))
    r = Reads(dev, reads, int(rng.choice([16, 32, 64, 256])), n_kv, bool(rng.integers(2)), seed=seed, pad=int(rng.integers(3)))
    q = normal(40 + seed, r.n, n_head, 128)
    if r.n:
        assert rel_rows(r.run(q, n_head, gap=4 * int(rng.integers(2))), r.want(q, SCALE)) < BAR
    r.free()


def test_attention_of_arrays_that_are_none(dev):
    """starts below 0 and past the buffers, a past beyond the table: each read has the rows that are there, over the rows that
    the table has room for"""
    page, n_kv, n_head, n_row = 16, 2, 4, 10
    table = np.array([[2, 0], [1, 1], [4, 3]], np.int32)
    start, past = np.array([-4, 2, 2, 100], np.int32), np.array([2 ** 31 - 1, 5, 3], np.int32)
    c = cache(dev, 3, n_kv, 5 * page)
    bufs = [dev.upload(a) for a in (start, past, table)]
    q = normal(1, n_row, n_head, 128)
    qb, out = dev.upload(q), dev.alloc(q.nbytes)
    htr.page_attention(dev, qb, htr.Pages.of(3, n_row, page, 2, *bufs), c.kv, n_head, SCALE, out)
    got = out.download(np.float32, q.size).reshape(n_row, -1)
    j = np.arange(2 * page)
    rows = table[:, j // page] * page + j % page
    want = np.zeros((n_row, n_head * 128))
    want[:2] = attention(q[:2], c.k[:, rows[0]], c.v[:, rows[0]], np.ones((2, 32), bool), SCALE)
    want[2:] = attention(q[2:], c.k[:, rows[2]], c.v[:, rows[2]], j[None, :] <= 3 + np.arange(8)[:, None], SCALE)
    assert rel_rows(got, want) < BAR
    for b in (*bufs, qb, out):
        b.free()
    c.free()


def test_recorded_calls_share_the_scratch(dev):
    """two recorded attentions of different batches replayed in turn, with eager work between: each gives its eager bits"""
    batches = [Reads(dev, reads, page, 2, q8_0, seed=seed) for reads, page, q8_0, seed in
               (([(900, 1), (20, 1)], 16, False, 1), ([(1500, 150), (40, 1)], 64, True, 2))]
    runs = []
    for r in batches:
        q = normal(r.n, r.n, 4, 128)
        qb, out = dev.upload(q), dev.alloc(q.nbytes)
        want = r.run(q, 4)
        dev.capture_begin()
        htr.page_attention(dev, qb, r.pages, r.cache.kv, 4, SCALE, out)
        runs.append((r, q, qb, out, want, dev.capture_end()))
    for i in range(4):
        for r, q, qb, out, want, g in runs[::1 if i % 2 else -1]:
            out.upload(np.full(q.size, 3.5, np.float32))
            g.launch()
            if i == 2:
                dev.sync()
        for r, q, qb, out, want, g in runs:
            np.testing.assert_array_equal(bits(out.download(np.float32, q.size)), bits(want.ravel()))
            np.testing.assert_array_equal(bits(r.run(q, 4)), bits(want))
    for r, q, qb, out, want, g in runs:
        g.free()
        qb.free()
        out.free()
        r.free()


def test_attention_of_scores_of_every_size(dev):
    """keys and scales that put most of a row's weight on few keys, or on one: the weights' reference moves"""
    for std, scale in ((8.0, SCALE), (1.0, 1.0), (30.0, 0.3), (1.0, -0.2), (1e-3, 1e-3), (1.0, 0.0)):
        r = Reads(dev, [(700, 1), (90, 40), (0, 70)], 32, 2, seed=3, std=std)
        q = normal(6, r.n, 4, 128)
        got, want = r.run(q, 4, scale), r.want(q, scale)
        # a score's own error is relative to its size: 2^-20 of |q|·|k|·scale, in the exponent
        top = np.max(np.abs(scale) * np.linalg.norm(q, axis=2)) * np.max(np.linalg.norm(np.nan_to_num(r.cache.k.astype(np.float64), nan=0.0), axis=2))
        assert rel_rows(got, want) < BAR + top * 2.0 ** -20
        r.free()


@pytest.mark.parametrize("q8_0", [False, True], ids=["f16", "q8_0"])
def test_attention_without_pages(dev, q8_0):
    """a table entry outside the cache stands for no rows: at the read's first page, in the middle, at its last; a read none of
    whose pages is there gets zeros; one with more rows than the table is wide sees those that it has"""
    page, reads = 16, [(100, 2), (50, 40), (20, 1), (70, 1), (33, 3)]
    r = Reads(dev, reads, page, 2, q8_0, seed=12, spare=0)
    gone = {0: [0], 1: [2, 5], 2: [0, 1], 3: [4], 4: [1]}
    table = r.table.copy()
    for i, (b, ks) in enumerate(gone.items()):
        for k in ks:
            table[b, k] = (-1, r.n_page, 2 ** 31 - 1, -2 ** 31, r.n_page + 5)[(i + k) % 5]
    r.bufs[2].upload(table)
    q = normal(2, r.n, 4, 128)
    got = r.run(q, 4)
    want = np.zeros((r.n, 4 * 128))
    for b, (p, n) in enumerate(reads):
        j = np.arange(p + n)
        here = ~np.isin(j // page, gone[b])
        seen = (j[None, :] <= p + np.arange(n)[:, None]) & here[None, :]
        at = slice(r.start[b], r.start[b + 1])
        want[at] = attention(q[at], r.cache.k[:, r.rows[b]], r.cache.v[:, r.rows[b]], seen, SCALE)
    assert not want[r.start[2]:r.start[3]].any()
    assert rel_rows(got, want) < BAR
    # the table cut to 3 pages: rows from 48 on are not there
    cut = dev.upload(np.ascontiguousarray(r.table[:, :3]))
    r.pages = htr.Pages.of(len(reads), r.n_row, page, 3, r.bufs[0], r.bufs[1], cut)
    got = r.run(q, 4)
    for b, (p, n) in enumerate(reads):
        j = np.arange(p + n)
        seen = (j[None, :] <= p + np.arange(n)[:, None]) & (j < 48)[None, :]
        at = slice(r.start[b], r.start[b + 1])
        want[at] = attention(q[at], r.cache.k[:, r.rows[b]], r.cache.v[:, r.rows[b]], seen, SCALE)
    assert rel_rows(got, want) < BAR
    cut.free()
    r.free()


@pytest.mark.parametrize("q8_0", [False, True], ids=["f16", "q8_0"])
def test_attention_of_values_that_are_not_finite(dev, q8_0):
    """a value that is not finite makes the outputs of the rows that see it not finite, and of no other"""
    r = Reads(dev, [(70, 50), (40, 1), (200, 1)], 32, 2, q8_0, seed=4)
    v = r.cache.v.copy()
    for b, j in ((0, 90), (2, 7)):
        v[1, r.rows[b][j], 5] = np.inf if b else np.nan
    k = r.cache.k
    r.cache.free()
    r.cache = Cache(dev, k, v, q8_0)
    q = normal(3, r.n, 4, 128)
    got = r.run(q, 4).reshape(r.n, 4, 128)
    bad = np.zeros((r.n, 4), bool)
    bad[90 - 70:50, 2:] = True  # read 0's rows from position 90 on, of KV head 1
    bad[51, 2:] = True
    finite = np.isfinite(got)
    block = slice(0, 32) if q8_0 else slice(5, 6)  # (a q8_0 block has one scale)
    assert not finite[bad][:, block].any()
    rest = np.ones(128, bool)
    rest[block] = False
    assert finite[~bad].all() and finite[bad][:, rest].all()
    clean = np.where(np.isfinite(r.cache.v), r.cache.v, 0)
    r.cache.v = clean
    want = r.want(q, SCALE).reshape(r.n, 4, 128)
    assert rel_rows(got[~bad], want[~bad]) < BAR
    assert np.allclose(got[bad][:, rest], want[bad][:, rest], atol=1e-4)
    r.free()


@pytest.mark.parametrize("reads", [[(60, 50), (500, 1)], [(60, 8), (500, 1)]], ids=["wide", "narrow"])
@pytest.mark.parametrize("scale", [511.75, 512.0, 65504.0])
def test_attention_of_quants_of_minus_128(dev, reads, scale):
    """a q8_0 cache made elsewhere may hold the quant -128, which with a scale of 512 and more is an infinity: rows that do not see
    it are as they were"""
    r = Reads(dev, reads, 32, 2, True, seed=21)
    n_ctx, j = r.cache.k.shape[1], 60 + reads[0][1] // 2  # seen from the middle row of the first read on
    qv = r.cache.bufs[1].download(np.int8, 2 * n_ctx * 128).reshape(2, n_ctx, 128)
    dv = r.cache.bufs[3].download(np.float16, 2 * n_ctx * 4).reshape(2, n_ctx, 4)
    qv[1, r.rows[0][j], 32:64], dv[1, r.rows[0][j], 1] = 1, scale
    qv[1, r.rows[0][j], 37] = -128
    r.cache.bufs[1].upload(qv)
    r.cache.bufs[3].upload(dv)
    with np.errstate(over="ignore"):
        r.cache.v = values(qv, dv)
    assert np.isfinite(r.cache.v[1, r.rows[0][j], 37]) == (scale < 512)
    q = normal(22, r.n, 4, 128)
    got = r.run(q, 4).reshape(r.n, 4, 128)
    r.cache.v = np.where(np.isfinite(r.cache.v), r.cache.v, 0)
    want = r.want(q, SCALE).reshape(r.n, 4, 128)
    sees = np.zeros((r.n, 4, 128), bool)
    sees[reads[0][1] // 2:reads[0][1], 2:, 37] = scale >= 512
    assert not np.isfinite(got[sees]).any() and np.isfinite(got[~sees]).all()
    clean = ~sees.any(axis=2)
    assert rel_rows(got[clean], want[clean]) < BAR
    assert np.allclose(got[~sees], want[~sees], rtol=1e-4, atol=1e-3)
    r.free()


def test_attention_over_a_long_cache(dev):
    """pages whose bytes lie past 4 GiB of a plane: row numbers times a row's bytes pass 32 bits"""
    page, n_ctx = 1024, (1 << 24) + 4096
    kb, vb = (dev.alloc(2 * n_ctx * 256) for _ in range(2))
    n, pages_ = 1500, np.array([[n_ctx // page - 1, n_ctx // page - 3]], np.int32)
    k, v = normal(1, 2, n, 128).astype(np.float16), normal(2, 2, n, 128, std=4.0).astype(np.float16)
    for buf, x in ((kb, k), (vb, v)):
        for h in range(2):
            for i, pg in enumerate(pages_[0]):
                part = np.ascontiguousarray(x[h, i * page:(i + 1) * page])
                htr._check(htr.lib().htr_upload(dev.h, buf.ptr + 256 * (h * n_ctx + int(pg) * page), part.ctypes.data, part.nbytes))
    arrays = [dev.upload(np.array(a, np.int32)) for a in ([0, 3], [n - 3], pages_)]
    q = normal(3, 3, 4, 128)
    qb, out = dev.upload(q), dev.alloc(q.nbytes)
    kv = htr.KvCache.of(2, n_ctx, kb, vb)
    htr.page_attention(dev, qb, htr.Pages.of(1, 3, page, 2, *arrays), kv, 4, SCALE, out)
    got = out.download(np.float32, q.size)
    seen = np.arange(n)[None, :] <= n - 3 + np.arange(3)[:, None]
    assert rel_rows(got, attention(q, k, v, seen, SCALE)) < BAR
    for b in (kb, vb, qb, out, *arrays):
        b.free()


@pytest.mark.parametrize("q8_0", [False, True], ids=["f16", "q8_0"])
@pytest.mark.parametrize("n_row", [1, 40])
def test_attention_up_to_the_last_row_that_is_counted(dev, q8_0, n_row):
    """a table of 2^27 − 1 pages of 16 rows of which the first and the last two are there, and rows whose keys end at 2^31 − 17, the
    last that it has room for"""
    page, max_pages = 16, 2 ** 27 - 1
    table = np.full(max_pages, -1, np.int32)
    table[0], table[-2], table[-1] = 1, 2, 0
    past = max_pages * page - n_row
    c = Cache(dev, normal(9, 1, 48, 128).astype(np.float16), normal(10, 1, 48, 128, std=4.0).astype(np.float16), q8_0)
    arrays = [dev.upload(np.array(a, np.int32)) for a in ([0, n_row], [past], table)]
    q = normal(3, n_row, 1, 128)
    qb, out = dev.upload(q), dev.alloc(q.nbytes)
    htr.page_attention(dev, qb, htr.Pages.of(1, n_row, page, max_pages, *arrays), c.kv, 1, SCALE, out)
    got = out.download(np.float32, q.size).reshape(n_row, 128)
    rows = np.concatenate([np.arange(16, 48), np.arange(16)])
    at = np.concatenate([np.arange(16), np.arange(max_pages * page - 32, max_pages * page)])
    seen = at[None, :] <= past + np.arange(n_row)[:, None]
    assert rel_rows(got, attention(q, c.k[:, rows], c.v[:, rows], seen, SCALE)) < BAR
    for b in (*arrays, qb, out):
        b.free()
    c.free()


# ---- the operators together -----------------------------------------------------------------------------------------------

def _loop(dev, q8_0, replay):
    """several reads through a layer's cache in pages: prompts in chunks, tokens, ends and new reads in their place. Each step's
    attention against a plain one over the rows that the read has had so far, and its q / k / v rows by the definition"""
    n_head, n_kv, page, n_seq, n_row, n_page = 4, 2, 16, 5, 90, 24
    s = Serving(n_seq, n_row, page, 12, n_page, seed=1)
    d = OnDevice(dev, s)
    n_pos, qw, kw = 200, n_head * 128, n_kv * 128
    ang = np.arange(n_pos)[:, None] * 1e6 ** (-np.arange(64) / 64.0)
    rope = np.stack([np.cos(ang), np.sin(ang)], axis=2).astype(np.float32)
    qn, kn = 1 + 0.02 * normal(1, 128), 1 + 0.02 * normal(2, 128)
    wq, wk, rb = (dev.upload(a.astype(np.float32)) for a in (qn, kn, rope))
    kv = htr.KvCache(dev, n_kv, n_page * page, q8_0)
    raw, q, out = dev.alloc(4 * n_row * (qw + 2 * kw)), dev.alloc(4 * n_row * qw), dev.alloc(4 * n_row * qw)
    parts = [type("Ref", (), {"ptr": raw.ptr + 4 * o}) for o in (0, qw, qw + kw)]

    def layer():
        d.map()
        htr.qkv_post_pages(dev, *parts, d.pages, wq, wk, rb, n_pos, n_head, EPS, kv, q, q_stride=qw + 2 * kw, kv_stride=qw + 2 * kw)
        htr.page_attention(dev, q, d.pages, kv, n_head, SCALE, out)

    graph = None
    had = [([], []) for _ in range(n_seq)]  # each read's K and V rows
    steps = [[40, 0, 7, 0, 0], [33, 1, 1, 16, 0], [1, 1, 1, 1, 30], [1, -1, 1, 15, 1], [1, 50, -1, 1, 1], [-1, 1, 90, 1, 1],
             [80, 1, 3, 1, 1], [1, 1, 1, -1, -1], [1, 1, 1, 60, 9]]
    refused = 0
    for i, new in enumerate(steps):
        start, past, pos, slot = want = s.step(new)
        x = normal(100 + i, n_row, n_head + 2 * n_kv, 128)
        x[:, n_head + n_kv:] *= 4
        raw.upload(x)
        d.new.upload(np.array(new, np.int32))
        if replay and i == 1:  # (the first step's call has made the scratch)
            dev.capture_begin()
            layer()
            graph = dev.capture_end()
        if graph:
            graph.launch()
        else:
            layer()
        d.check(want)
        got = out.download(np.float32, n_row * qw).reshape(n_row, -1)
        got_q = q.download(np.float32, n_row * qw).reshape(n_row, n_head, 128)
        for b in range(n_seq):
            if new[b] < 0:
                had[b] = ([], [])
            at = slice(start[b], start[b + 1])
            n = start[b + 1] - start[b]
            if n == 0:
                continue
            if past[b] < 0:
                refused += 1
                assert not got[at].any()
                continue
            cs = rope[pos[at]]
            wq_, wk_ = heads(x[at, :n_head], qn, cs), heads(x[at, n_head:n_head + n_kv], kn, cs)
            assert np.all(np.abs(got_q[at] - wq_) <= np.spacing(np.abs(wq_)))
            for rows, y in zip(had[b], (wk_, x[at, n_head + n_kv:])):
                rows.extend(values(*blocks(y)) if q8_0 else y.astype(np.float16))
            k, v = (np.array(rows).transpose(1, 0, 2) for rows in had[b])
            assert k.shape[1] == past[b] + n
            seen = np.arange(past[b] + n)[None, :] <= past[b] + np.arange(n)[:, None]
            assert rel_rows(got[at], attention(got_q[at], k, v, seen, SCALE)) < BAR
    assert refused >= 1  # (by the plain form: 52 + 80 rows and more in a step of 90)
    if graph:
        graph.free()
    for b in (wq, wk, rb, kv, raw, q, out, d):
        b.free()


@pytest.mark.parametrize("q8_0", [False, True], ids=["f16", "q8_0"])
@pytest.mark.parametrize("replay", [False, True], ids=["eager", "replayed"])
def test_serving_loop(dev, q8_0, replay):
    _loop(dev, q8_0, replay)


def test_freed_pages_are_refused(dev):
    p = htr.Pages(dev, 2, 3, 16, 2)
    p.free()
    b = dev.alloc(4096)
    with pytest.raises(htr.HtrError, match="null start"):
        htr.page_map(dev, p, 1, b, b, b, b, b, b)
    b.free()


@pytest.fixture(scope="module")
def poisoned():
    """another device handle on the same GPU, with a stream and scratch of its own, whose memory starts as NaN"""
    with pytest.MonkeyPatch.context() as env:
        env.setenv("HTR_POISON", "1")
        d = htr.Device(0)
    yield d
    d.close()


@pytest.mark.parametrize("n_head,n_kv,reads", [(4, 2, [(2500, 1), (300, 140), (4000, 1), (-1, 2)]),
                                               (16, 8, [(2500, 1), (300, 6), (4000, 1), (-1, 2)])], ids=["chunks", "tokens"])
def test_two_devices_at_once(dev, poisoned, n_head, n_kv, reads):
    """calls of two handles that overlap, eager and replayed, each with tiles and rows in parts: the bits of either alone, where
    scratch was NaN before its first use too"""
    vocab, top = 151936, 7
    logits = normal(4, 3, vocab, std=2.5)
    sides = []
    for d in (dev, poisoned):
        r = Reads(d, reads, 32, n_kv, seed=6)
        q = normal(8, r.n, n_head, 128)
        b = [d.upload(a) for a in (q, logits, np.array([5, 70000, vocab - 1], np.int32))]
        out = [d.alloc(4 * n) for n in (q.size, 3, 3, 3 * top, 3 * top)]

        def call(d=d, r=r, b=b, out=out):
            htr.page_attention(d, b[0], r.pages, r.cache.kv, n_head, SCALE, out[0])
            htr.token_logprobs(d, b[1], 3, vocab, b[2], out[1], out[2], top, out[3], out[4])

        sides.append((d, r, q, b, out, call))
    want = []
    for d, r, q, b, out, call in sides:
        call()
        want.append([o.download(np.uint32, o.nbytes // 4) for o in out])
    for x, y in zip(*want):
        np.testing.assert_array_equal(x, y)
    d, r, q, *_ = sides[0]
    assert rel_rows(want[0][0].view(np.float32).reshape(r.n, -1), r.want(q, SCALE)) < BAR
    graphs = []
    for d, r, q, b, out, call in sides:
        d.capture_begin()
        call()
        graphs.append(d.capture_end())
    for i in range(6):
        for (d, r, q, b, out, call), g in zip(sides, graphs):
            for _ in range(4):
                g.launch() if i % 2 else call()
        for d, r, q, b, out, call in sides:
            for o, w in zip(out, want[0]):
                np.testing.assert_array_equal(o.download(np.uint32, w.size), w)
    for g in graphs:
        g.free()
    for d, r, q, b, out, call in sides:
        for o in (*b, *out):
            o.free()
        r.free()


def test_a_recording_cannot_make_the_scratch(dev):
    """on a new handle the first call of a graph fails with the reason; after an eager one, of tokens or of chunks, both are
    recorded"""
    reads = [[(900, 1), (40, 1)], [(500, 70)]]
    d = htr.Device(0)
    runs = []
    for seed, r in enumerate(reads):
        r = Reads(d, r, 16, 8, seed=seed)
        q = normal(seed, r.n, 16, 128)
        runs.append((r, q, d.upload(q), d.alloc(q.nbytes)))

    def call(i):
        r, q, qb, out = runs[i]
        htr.page_attention(d, qb, r.pages, r.cache.kv, 16, SCALE, out)

    for i in range(2):
        d.capture_begin()
        with pytest.raises(htr.HtrError, match="captured"):
            call(i)
        d.capture_end().free()
    call(0)
    for i, (r, q, qb, out) in enumerate(runs):
        d.capture_begin()
        call(i)
        g = d.capture_end()
        for _ in range(3):
            out.upload(np.full(q.size, 9.0, np.float32))
            g.launch()
            assert rel_rows(out.download(np.float32, q.size).reshape(r.n, -1), r.want(q, SCALE)) < BAR
        g.free()
    for r, q, qb, out in runs:
        qb.free()
        out.free()
        r.free()
    d.close()


# ---- the order of the two kinds of tiles ----------------------------------------------------------------------------------

def source_constants(*names):
    with open(os.path.join(PKG, "csrc", "page_attention.hip")) as f:
        text = f.read()
    return [float(re.search(rf"\b{n} = ([0-9.]+)f?\b", text)[1]) for n in names]


def lines(reads, group):
    """the lengths of the lines of wide and of narrow tiles (keys and 128 more to a tile; a wide one's by the heads of a group)"""
    wide, narrow = 0, 0
    for past, n in reads:
        rows = n * group
        rest, tiles, held = rows % 128, rows // 128 + (rows % 128 > 32), max(past, 0) + 128
        wide += tiles * (held * group + 64 * tiles)
        narrow += held + n if 0 < rest <= 32 else 0
    return wide, narrow


def beside_tokens(past, n, tokens):
    """chunks of n and n - 1 rows over past keys, beside tokens over some 500, in an order of their own"""
    reads = [(430 + 7 * i % 150, 1) for i in range(tokens)]
    return reads[:tokens // 3] + [(past, n)] + reads[tokens // 3:-2] + [(past - 11, n - 1)] + reads[-2:]


@pytest.mark.parametrize("n_head,n_kv,reads,turns", [
    (16, 8, beside_tokens(2500, 300, 60), True), (14, 7, beside_tokens(2700, 300, 60), True),  # (7 KV heads: an odd number of pieces)
    (14, 7, beside_tokens(2600, 330, 200), True), (12, 4, beside_tokens(6000, 260, 90), True),
    # the bounds' other sides: little to do for the narrow tiles, for the wide ones, for either
    (16, 8, beside_tokens(4000, 300, 6), False), (16, 8, [(2500, 150)] + [(3000, 1)] * 70, False), (14, 7, beside_tokens(300, 130, 20), False)])
def test_attention_of_kinds_in_turn(dev, n_head, n_kv, reads, turns):
    """f16 rows: half of the workgroups of wide tiles, half of those of narrow ones, and what is left of each; and one kind behind the
    other. The outputs start as infinities: a piece that nobody took would be seen"""
    low, high, pieces_of, least = source_constants("TURNS_FROM", "TURNS_TO", "TURNS_PIECES", "LEAST")
    wide, narrow = lines(reads, n_head // n_kv)
    pieces = 2 * dev.info()[1] // n_kv
    assert turns == (low * wide < narrow < high * wide and wide > pieces_of * least * (n_head // n_kv) * pieces)
    r = Reads(dev, reads, 32, n_kv, seed=n_kv, pad=2)
    q = normal(n_head, r.n, n_head, 128)
    got = r.run(q, n_head, fill=np.inf)
    assert dev.last_kernel() == "k_page_attn_join"
    assert rel_rows(got, r.want(q, SCALE)) < BAR
    assert np.array_equal(bits(got), bits(r.run(q, n_head)))
    r.free()


@pytest.mark.parametrize("q8_0", [False, True], ids=["f16", "q8_0"])
@pytest.mark.parametrize("n_head,n_kv,reads", [
    # a full tile of 32 rows in many parts, on 8 KV heads, whose workgroups share an XCD, and on 4 and 1, whose do not
    (8, 8, [(4000, 32)] + [(0, 0)] * 7), (4, 4, [(4000, 32)] + [(0, 0)] * 7), (1, 1, [(9000, 32)] + [(0, 0)] * 7),
    # 120 rows of many reads; several tiles to a read
    (8, 8, [(37 * i % 900, 1) for i in range(90)] + [(700, 30), (0, 7)]), (3, 3, [(37 * i % 900, 1) for i in range(90)] + [(700, 30), (0, 7)]),
    (16, 8, [(9, 0)] * 40 + [(2500, 33), (64, 20), (-1, 9)]), (2, 1, [(9, 0)] * 40 + [(2500, 33), (64, 20), (-1, 9)])])
def test_attention_in_one_launch(dev, n_head, n_kv, reads, q8_0):
    """steps that one launch takes (by the rule on sizes, and by the kernel that ran): a cut tile's parts joined by the last of its
    workgroups, call after call, replayed among others that leave other parts and tickets"""
    few, = source_constants("FEW")
    n = sum(new for _, new in reads)
    assert n * n_head // n_kv <= few and n <= 4 * len(reads)
    r = Reads(dev, reads, 32, n_kv, q8_0, seed=n_head)
    q = normal(33, r.n, n_head, 128)
    got = r.run(q, n_head, fill=np.inf)
    assert dev.last_kernel().startswith("k_page_few<")
    assert rel_rows(got, r.want(q, SCALE)) < BAR
    other = Reads(dev, [(1500, 1), (40, 1), (3000, 1)], 16, n_kv, not q8_0, seed=5)
    oq = normal(34, other.n, n_head, 128)
    other_got = other.run(oq, n_head)
    assert dev.last_kernel().startswith("k_page_few<")
    qb, out = dev.upload(q), dev.alloc(q.nbytes)
    dev.capture_begin()
    htr.page_attention(dev, qb, r.pages, r.cache.kv, n_head, SCALE, out)
    g = dev.capture_end()
    for i in range(4):
        out.upload(np.full(q.size, 2.5, np.float32))
        g.launch()
        np.testing.assert_array_equal(bits(other.run(oq, n_head)), bits(other_got))
        g.launch()
        np.testing.assert_array_equal(bits(out.download(np.float32, q.size)), bits(got.ravel()))
    for b in (g, qb, out, r, other):
        b.free()


# ---- nothing written past an array ----------------------------------------------------------------------------------------

class Guarded:
    """an int32 array on the device between words of a pattern"""
    GUARD, WORD = 300, 0x5EED5EED

    def __init__(self, dev, a):
        self.dev, self.n = dev, np.size(a)
        words = np.full(self.n + 2 * self.GUARD, self.WORD, np.int32)
        words[self.GUARD:self.GUARD + self.n] = np.ravel(a)
        self.buf = dev.upload(words)
        self.ptr = self.buf.ptr + 4 * self.GUARD

    def upload(self, a):
        a = np.ascontiguousarray(a, np.int32)
        assert a.size == self.n
        htr._check(htr.lib().htr_upload(self.dev.h, self.ptr, a.ctypes.data, a.nbytes))

    def download(self, dtype, count):
        words = self.buf.download(np.int32)
        for guard in (words[:self.GUARD], words[self.GUARD + self.n:]):
            np.testing.assert_array_equal(guard, self.WORD)
        assert count == self.n
        return words[self.GUARD:self.GUARD + self.n].view(dtype)

    def free(self):
        self.buf.free()


class GuardedDevice(OnDevice):
    """OnDevice on guarded arrays, whose guards each check looks at (those that a call only reads too)"""

    def __init__(self, dev, s, in_place):
        g = lambda a: Guarded(dev, np.asarray(a, np.int64).astype(np.int32))  # noqa: E731
        self.dev, self.s = dev, s
        rows = [np.full(n, 77) for n in (s.n_seq + 1, s.n_seq)]
        self.arrays = [g(rows[0]), g(rows[1]), g(s.table), g(np.full(s.n_row, 77)), g(np.full(s.n_row, 77))]
        self.pages = htr.Pages.of(s.n_seq, s.n_row, s.page, s.max_pages, *self.arrays)
        self.len, self.new, self.ring, self.pool = g(s.len), g(np.zeros(s.n_seq)), g(s.ring), g([s.head, s.count])
        self.len_out, self.pool_out = (self.len, self.pool) if in_place else (g(np.zeros(s.n_seq)), g([0, 0]))

    def check(self, want):
        super().check(want)
        for a in (self.len, self.new, self.pool):
            a.download(np.int32, a.n)

    def free(self):
        super().free()
        for a in self.arrays:
            a.free()


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("n_seq,n_row,page,max_pages", [(1, 1, 16, 1), (5, 50, 16, 4), (256, 512, 16, 3), (257, 512, 32, 2), (1024, 4096, 16, 5),
                                                        (1000, 5000, 64, 7), (3, 9000, 1024, 9)])
def test_nothing_is_written_past_a_map_s_arrays(dev, n_seq, n_row, page, max_pages, in_place):
    """lengths below 0, past the table, at the end of 32 bits; new rows whose sums pass 32 bits, ends of any number below 0; tables
    without pages: as the definition has it, and nothing in front of or behind an array"""
    rng = np.random.default_rng(n_seq + n_row)
    cap = page * max_pages
    lengths = np.array([-5, -2 ** 31, 0, 1, page, cap - 1, cap, cap + 1, 2 ** 31 - 1, 2 ** 31 - page])
    news = np.array([0, 1, 1, 7, page, cap, n_row, 2 ** 31 - 1, -1, -7, -2 ** 31])
    for usual, usual_new in ((0.5, 1.0), (0.9, 0.995), (0.0, 0.0)):
        s = Serving(n_seq, n_row, page, max_pages, n_seq * max_pages + 3, seed=n_seq)
        s.len[:] = np.where(rng.random(n_seq) < usual, rng.integers(0, cap + 1, n_seq), rng.choice(lengths, n_seq))
        s.table[:] = np.where(rng.random(s.table.shape) < 0.8, rng.integers(0, s.n_page, s.table.shape), -1)
        new = np.where(rng.random(n_seq) < usual_new, rng.integers(0, max(2, n_row // n_seq), n_seq), rng.choice(news, n_seq))
        held = np.minimum(-(-np.maximum(s.len, 0) // page), max_pages)
        s.count = min(s.n_page - int(held[new < 0].sum()), max(2, n_seq // 2))  # (room in the ring for what comes back)
        d = GuardedDevice(dev, s, in_place)
        d.new.upload(new.astype(np.int32))
        want = s.step(new)
        d.map()
        d.check(want)
        d.free()


# ---- what shares a device's scratch; rows far apart -----------------------------------------------------------------------

def test_all_ways_of_joining_in_one_recording(dev):
    """tokens on 8 KV heads, whose workgroups share an XCD, on 3 and on 1, whose do not, and chunks by two launches, one after another
    over the same tickets and scratch, recorded as one graph and replayed: the bits of each alone"""
    runs = []
    for seed, (reads, n_head, n_kv, q8_0, kernel) in enumerate([
            ([(5000, 1), (300, 2)], 16, 8, False, "k_page_few<f16>"), ([(4000, 2), (70, 1)], 6, 3, True, "k_page_few<q8_0>"),
            ([(2000, 150), (900, 1)], 16, 8, False, "k_page_attn_join"), ([(9000, 3)], 2, 1, False, "k_page_few<f16>"),
            ([(3000, 40), (20, 200)], 4, 1, True, "k_page_attn_join"), ([(5000, 1), (300, 2)], 16, 8, True, "k_page_few<q8_0>")]):
        r = Reads(dev, reads, 32, n_kv, q8_0, seed=seed)
        q = normal(50 + seed, r.n, n_head, 128)
        want = r.run(q, n_head)
        assert dev.last_kernel() == kernel
        assert rel_rows(want, r.want(q, SCALE)) < BAR
        runs.append((r, q, n_head, want, dev.upload(q), dev.alloc(q.nbytes)))
    dev.capture_begin()
    for _ in range(2):
        for r, q, n_head, want, qb, out in runs:
            htr.page_attention(dev, qb, r.pages, r.cache.kv, n_head, SCALE, out)
    g = dev.capture_end()
    for i in range(6):
        for r, q, n_head, want, qb, out in runs:
            out.upload(np.full(q.size, -3.5, np.float32))
        g.launch()
        for r, q, n_head, want, qb, out in runs[::-1 if i % 2 else 1]:
            np.testing.assert_array_equal(bits(out.download(np.float32, q.size)), bits(want.ravel()))
            if i % 3 == 0:
                np.testing.assert_array_equal(bits(r.run(q, n_head)), bits(want))
    g.free()
    for r, q, n_head, want, qb, out in runs:
        for b in (qb, out, r):
            b.free()


def test_rows_past_32_bits(dev):
    """q, k and v rows 2^30 + 4 floats apart (the fifth 17 GB behind the first), attended by the kernels of one launch and of two, and
    stored: as rows without a gap"""
    n, n_head, n_kv, page, gap = 5, 4, 2, 16, 2 ** 30 + 4
    x = normal(11, n, n_head + 2 * n_kv, 128)
    q = x[:, :n_head]
    big = dev.alloc(4 * ((n - 1) * gap + x[0].size))
    for i in range(n):
        row = np.ascontiguousarray(x[i])
        htr._check(htr.lib().htr_upload(dev.h, big.ptr + 4 * gap * i, row.ctypes.data, row.nbytes))
    out = dev.alloc(q.nbytes)
    for reads, kernel in (([(40, 2), (100, 1), (3, 2)], "k_page_few<f16>"), ([(90, 5)], "k_page_attn_join")):
        r = Reads(dev, reads, page, n_kv, seed=9)
        want = r.run(q, n_head)
        assert rel_rows(want, r.want(q, SCALE)) < BAR
        htr.page_attention(dev, big, r.pages, r.cache.kv, n_head, SCALE, out, q_stride=gap)
        assert dev.last_kernel() == kernel
        np.testing.assert_array_equal(bits(out.download(np.float32, q.size)), bits(want.ravel()))
        r.free()
    n_pos = 50
    ang = np.arange(n_pos)[:, None] * 1e6 ** (-np.arange(64) / 64.0)
    others = [dev.upload(a) for a in (np.full(128, 1.25, np.float32), np.stack([np.cos(ang), np.sin(ang)], axis=2).astype(np.float32),
                                      np.array([7, 0, 49, 3, 20], np.int32), np.array([31, 4, 0, 17, 16], np.int32))]
    w, rope, pos, slot = others
    p = htr.Pages.of(1, n, page, 2, pos, pos, pos, pos, slot)
    got = []
    near = dev.upload(x)
    for base, stride in ((near, x[0].size), (big, gap)):
        c = cache(dev, 6, n_kv, 2 * page, True)
        at = [type("Ref", (), {"ptr": base.ptr + 512 * o}) for o in (0, n_head, n_head + n_kv)]
        out.upload(np.zeros(q.size, np.float32))
        htr.qkv_post_pages(dev, *at, p, w, w, rope, n_pos, n_head, EPS, c.kv, out, q_stride=stride, kv_stride=stride)
        got.append([out.download(np.uint32, q.size), *c.rows("k"), *c.rows("v")])
        c.free()
    assert got[0][0].any()
    for a, b in zip(*got):
        np.testing.assert_array_equal(a, b)
    for b in (big, near, out, *others):
        b.free()
