"""The operators on a layer's KV cache on the GPU against plain numpy in 64 bits: rows normed, turned and stored, copies
between cache types, rows kept, attention of a drafted tree and of a sliding window, and a drafted step of them together."""
import ctypes as C
import threading

import numpy as np
import pytest

import htr
import oracle as orc

pytestmark = pytest.mark.gpu
EPS = 1e-6
SCALE = float(np.float32(1 / np.sqrt(128)))


# ---- plain forms ----------------------------------------------------------------------------------------------------------

def heads(x, w, cs):
    """rows x [n, heads, 128] normed with w and turned by cs [n, 64, 2], in f64, as f32"""
    x = x.astype(np.float64)
    y = x / np.sqrt(np.mean(x * x, axis=2, keepdims=True) + np.float64(np.float32(EPS))) * w.astype(np.float64)
    c, s = (cs[:, None, :, i].astype(np.float64) for i in (0, 1))
    a, b = y[:, :, :64], y[:, :, 64:]
    return np.concatenate([a * c - b * s, a * s + b * c], axis=2).astype(np.float32)


F16_UP = np.arange(0x7C00, dtype=np.uint16).view(np.float16).astype(np.float64)  # 0 and the positive f16 numbers in order


def blocks(x):
    """q8_0 blocks of rows x [..., 128]: int8 quants and f16 scales [..., 4]"""
    x = np.clip(x.astype(np.float64), -127 * 515.5, 127 * 515.5, where=np.isfinite(x), out=x.astype(np.float64))
    b = x.reshape(*x.shape[:-1], 4, 32)
    bad = ~np.isfinite(b).all(axis=-1)
    b = np.where(bad[..., None], 0.0, b)
    d = F16_UP[np.searchsorted(F16_UP * 127, np.abs(b).max(axis=-1))]
    q = np.rint(np.divide(b, d[..., None], out=np.zeros_like(b), where=d[..., None] > 0))
    assert np.abs(q).max() <= 127
    d = np.where(bad, np.nan, d).astype(np.float16)
    return q.astype(np.int8).reshape(x.shape), d


def values(q, d):
    """f16(q·d)"""
    return (q.reshape(*d.shape, 32).astype(np.float32) * d[..., None].astype(np.float32)).astype(np.float16).reshape(q.shape)


def attention(q, k, v, seen, scale):
    """q [n, n_head, 128], k and v [n_kv, keys, 128], seen [n, keys] → [n, n_head·128] in f64; what a query does not see is
    not there; zeros where it sees nothing"""
    n, n_head = q.shape[:2]
    out = np.zeros((n, n_head, 128))
    for t in range(n):
        at = np.flatnonzero(seen[t])
        if at.size == 0:
            continue
        kt, vt = k[:, at].astype(np.float64), v[:, at].astype(np.float64)
        for h in range(n_head):
            j = h * k.shape[0] // n_head
            s = kt[j] @ q[t, h].astype(np.float64) * np.float64(np.float32(scale))
            p = np.exp(s - s.max())
            out[t, h] = p @ vt[j] / p.sum()
    return out.reshape(n, -1)


def rel_rows(got, want):
    """the largest relative error of a head's 128 values"""
    g, w = got.reshape(-1, 128).astype(np.float64), want.reshape(-1, 128)
    n = np.linalg.norm(w, axis=1)
    e = np.linalg.norm(g - w, axis=1)
    assert np.all(np.isfinite(g)) and np.all(g[n == 0] == 0)
    return float(np.max(np.divide(e, n, out=np.zeros_like(e), where=n > 0)))


# What the attention may be off by. q is held to 2^-22 of its row's largest value a (11 bits, and 11 more in the rest), its
# product with scale rounded once (2^-24): a score errs by at most (2^-22 + 2^-24)·a·scale·Σ|k|, and its f32 sum of 256
# products by 2^-24·√256 of its terms' size. For q, k ~ N(0, 1): a ≤ 4.5, Σ|k| ≤ 130, so 1.6e-5 if every element erred its most
# and one way; the errors are independent and even, so √128 of them instead of 128: 1.4e-6, four deviations of it 2e-6 at most.
# The softmax turns a score's error into as much of p; p's own pair, exponential and sums add 2^-21. 1e-5 leaves room.
BAR = 1e-5


# ---- buffers --------------------------------------------------------------------------------------------------------------

class Cache:
    """a cache on the device with values x_k, x_v f16 [n_kv, rows, 128], in either type; .k / .v: what its rows stand for"""

    def __init__(self, dev, k, v, q8_0=False):
        self.dev = dev
        if q8_0:
            (qk, dk), (qv, dv) = blocks(k), blocks(v)
            self.bufs = [dev.upload(a) for a in (qk, qv, dk, dv)]
            self.k, self.v = values(qk, dk), values(qv, dv)
        else:
            self.bufs = [dev.upload(a) for a in (k, v)]
            self.k, self.v = k, v
        self.kv = htr.KvCache.of(k.shape[0], k.shape[1], *self.bufs)

    def rows(self, which="k"):
        """the rows as they are on the device"""
        c = self.kv
        i = 0 if which == "k" else 1
        if not c.q8_0:
            return self.bufs[i].download(np.float16, c.n_kv * c.n_ctx * 128).reshape(c.n_kv, c.n_ctx, 128)
        return (self.bufs[i].download(np.int8, c.n_kv * c.n_ctx * 128).reshape(c.n_kv, c.n_ctx, 128),
                self.bufs[2 + i].download(np.float16, c.n_kv * c.n_ctx * 4).reshape(c.n_kv, c.n_ctx, 4))

    def free(self):
        for b in self.bufs:
            b.free()


def bits(a):
    return a.view({2: np.uint16, 4: np.uint32, 1: np.uint8}[a.dtype.itemsize])


def normal(seed, *shape, std=1.0):
    return (np.random.default_rng(seed).standard_normal(shape) * std).astype(np.float32)


def cache(dev, seed, n_kv, rows, q8_0=False, **kw):
    return Cache(dev, normal(seed, n_kv, rows, 128, **kw).astype(np.float16),
                 normal(seed + 1, n_kv, rows, 128, std=4.0).astype(np.float16), q8_0)


def strided(dev, x, gap):
    """rows x [n, m] on the device with gap floats of NaN between them"""
    return dev.upload(np.concatenate([x, np.full((x.shape[0], gap), np.nan, np.float32)], axis=1))


# ---- rows normed, turned and stored ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("q8_0", [False, True], ids=["f16", "q8_0"])
@pytest.mark.parametrize("n,n_head,n_kv,pos0,row0,fused,drafted", [
    (1, 16, 8, 700, 3, True, False), (1, 1, 1, 0, 0, False, False), (7, 6, 2, 5, 11, True, True), (64, 16, 8, 40, 0, True, True),
    (129, 4, 4, 0, 2, False, False), (333, 16, 8, 17, 17, True, False)])
def test_rows_are_normed_turned_and_stored(dev, q8_0, n, n_head, n_kv, pos0, row0, fused, drafted):
    """the cache's rows bit for bit (the kernel's f64 rounds to the same f32 as numpy's: two f64 sums differ by 2^-50, which
    a border of f32 separates once in 2^26 values); q to an f32 ulp; nothing else of the cache is written"""
    rng = np.random.default_rng(n * 31 + n_head)
    width = (n_head + 2 * n_kv) * 128
    x = normal(n + n_kv, n, n_head + 2 * n_kv, 128, std=3.0)
    x[0, -1, 32:64] = 0.0
    x[-1, -1, 64:96] *= np.float32(2.0 ** -22)  # a block whose scale is among the last f16 numbers
    qn, kn = normal(1, 128, std=0.1) + 1, normal(2, 128, std=0.1) + 1
    n_pos = pos0 + 64 + n
    cs = orc.rope_table(1e6, 128, n_pos).reshape(n_pos, 64, 2)
    tree = htr.Tree([-1] + [int(rng.integers(-1, i)) for i in range(1, n)]) if drafted else None
    pos = pos0 + (tree.depths if drafted else np.arange(n))
    n_ctx = row0 + n + 5
    c = cache(dev, 50, n_kv, n_ctx, q8_0)
    before = [c.rows(w) for w in "kv"]
    q_out = dev.upload(np.full((n + 1, n_head * 128), 7.0, np.float32))
    parts = [x[:, :n_head], x[:, n_head:n_head + n_kv], x[:, n_head + n_kv:]]
    if fused:
        raw = dev.upload(x)
        at = [raw.ptr, raw.ptr + n_head * 512, raw.ptr + (n_head + n_kv) * 512]
        strides = dict(q_stride=width, kv_stride=width)
        bufs = [raw]
    else:
        bufs = [dev.upload(np.ascontiguousarray(p)) for p in parts]
        at, strides = [b.ptr for b in bufs], {}

    class At:
        def __init__(self, ptr):
            self.ptr = ptr

    htr.qkv_post_rows(dev, *map(At, at), n, dev.upload(qn), dev.upload(kn), dev.upload(cs), n_pos, pos0, n_head, EPS, c.kv,
                      row0, q_out, tree=tree, **strides)
    want_q = heads(parts[0], qn, cs[pos])
    got_q = q_out.download(np.float32).reshape(n + 1, n_head * 128)
    assert np.all(got_q[n] == 7.0)
    assert np.all(np.abs(got_q[:n] - want_q.reshape(n, -1)) <= 2.0 ** -23 * np.abs(want_q.reshape(n, -1)))
    for w, rows, old in zip("kv", (heads(parts[1], kn, cs[pos]), parts[2]), before):
        rows, got = rows.transpose(1, 0, 2), c.rows(w)
        want = blocks(rows) if q8_0 else (rows.astype(np.float16),)
        for g, o, y in zip(got if q8_0 else (got,), old if q8_0 else (old,), want):
            o = o.copy()
            o[:, row0:row0 + n] = y
            assert np.array_equal(bits(g), bits(o))
    c.free()


def test_rows_in_place_and_not_finite(dev):
    """q_out on q's rows; V rows with infinities and NaN: f16 holds them as they are, a q8_0 block is NaN, its neighbours
    are not; values past f16's largest saturate in q8_0"""
    n, n_head, n_kv = 3, 2, 1
    q, k, v = normal(1, n, n_head, 128), normal(2, n, n_kv, 128), normal(3, n, n_kv, 128)
    v[0, 0, 5], v[1, 0, 40], v[2, 0, 70], v[2, 0, 100] = np.inf, np.nan, 7e4, -3e38
    cs = orc.rope_table(1e6, 128, 8).reshape(8, 64, 2)
    one = np.ones(128, np.float32)
    for q8_0 in (False, True):
        c = cache(dev, 9, n_kv, n, q8_0)
        qb = dev.upload(q)
        htr.qkv_post_rows(dev, qb, dev.upload(k), dev.upload(v), n, dev.upload(one), dev.upload(one), dev.upload(cs), 8, 2, n_head,
                          EPS, c.kv, 0, qb)
        want = heads(q, one, cs[2:5])
        assert np.all(np.abs(qb.download(np.float32).reshape(q.shape) - want) <= 2.0 ** -23 * np.abs(want))
        got = c.rows("v")
        if q8_0:
            wq, wd = blocks(v.transpose(1, 0, 2))
            assert np.array_equal(got[0], wq) and np.array_equal(got[1], wd, equal_nan=True)
            assert np.isnan(wd).sum() == 2 and wd[0, 2, 2] == np.float16(515.5) and wd[0, 2, 3] == np.float16(515.5)
        else:
            with np.errstate(over="ignore"):
                assert np.array_equal(got, v.transpose(1, 0, 2).astype(np.float16), equal_nan=True)
        c.free()


# ---- copies ---------------------------------------------------------------------------------------------------------------

def hard_rows(seed, n_kv, rows):
    """f16 rows of all sizes: whole blocks of zeros, of the smallest numbers, of ties between two quants, of the largest"""
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((n_kv, rows, 4, 32)) * 2.0 ** rng.integers(-26, 13, (n_kv, rows, 4, 1))).astype(np.float16)
    kind = rng.integers(0, 8, (n_kv, rows, 4))
    x[kind == 0] = 0
    tie = (rng.integers(-253, 254, x.shape) / 2.0).astype(np.float16)  # 127 and halves of the scale 1
    tie[..., 0] = 127
    x = np.where((kind == 1)[..., None], tie, x)
    x = np.where((kind == 2)[..., None], rng.integers(-9, 10, x.shape) * np.float16(2.0 ** -24), x).astype(np.float16)
    x[kind == 3] = np.float16(65504)
    return x.reshape(n_kv, rows, 128)


@pytest.mark.parametrize("n_kv,rows,src_ctx,src_row,dst_ctx,dst_row", [
    (1, 1, 1, 0, 1, 0), (2, 63, 70, 7, 66, 1), (3, 64, 64, 0, 90, 26), (8, 1000, 1003, 2, 1001, 1)])
def test_copies_quantise_and_read_back(dev, n_kv, rows, src_ctx, src_row, dst_ctx, dst_row):
    """bit for bit: every quant and scale, every value read back; the other rows stay as they are. A block's values are
    within half a scale and f16's rounding of q·d"""
    c = Cache(dev, hard_rows(1, n_kv, src_ctx), hard_rows(2, n_kv, src_ctx))
    q = cache(dev, 5, n_kv, dst_ctx, True)
    old = {w: q.rows(w) for w in "kv"}
    htr.kv_copy(dev, c.kv, src_row, q.kv, dst_row, rows)
    back = cache(dev, 7, n_kv, src_ctx + 3)
    held = {w: back.rows(w).copy() for w in "kv"}
    htr.kv_copy(dev, q.kv, dst_row, back.kv, 3, rows)
    again = cache(dev, 8, n_kv, rows + 1, True)
    htr.kv_copy(dev, q.kv, dst_row, again.kv, 1, rows)
    half = cache(dev, 9, n_kv, rows + 2)
    htr.kv_copy(dev, back.kv, 3, half.kv, 2, rows)
    htr.kv_copy(dev, c.kv, 0, q.kv, 0, 0)  # no rows: nothing
    for w, x in (("k", c.k), ("v", c.v)):
        x = x[:, src_row:src_row + rows]
        wq, wd = blocks(x)
        gq, gd = q.rows(w)
        eq, ed = old[w][0].copy(), old[w][1].copy()
        eq[:, dst_row:dst_row + rows], ed[:, dst_row:dst_row + rows] = wq, wd
        assert np.array_equal(gq, eq) and np.array_equal(bits(gd), bits(ed))
        e = held[w].copy()
        e[:, 3:3 + rows] = values(wq, wd)
        assert np.array_equal(bits(back.rows(w)), bits(e))
        off = np.abs(values(wq, wd).astype(np.float64) - x.astype(np.float64)).reshape(*wd.shape, 32)
        room = wd.astype(np.float64)[..., None] / 2 + 2.0 ** -11 * np.abs(x.astype(np.float64)).reshape(off.shape) * 1.01 + 2.0 ** -25
        assert np.all(off <= room)
        aq, ad = again.rows(w)
        assert np.array_equal(aq[:, 1:], wq) and np.array_equal(bits(ad[:, 1:]), bits(wd))
        assert np.array_equal(bits(half.rows(w)[:, 2:]), bits(values(wq, wd)))
    for x in (c, q, back, again, half):
        x.free()


def test_copies_of_values_that_are_not_finite(dev):
    k = normal(3, 1, 4, 128).astype(np.float16)
    k[0, 0, 3], k[0, 2, 127] = np.nan, -np.inf
    c, q, back = Cache(dev, k, k), cache(dev, 1, 1, 4, True), cache(dev, 2, 1, 4)
    htr.kv_copy(dev, c.kv, 0, q.kv, 0, 4)
    htr.kv_copy(dev, q.kv, 0, back.kv, 0, 4)
    wq, wd = blocks(k)
    assert np.array_equal(q.rows("k")[0], wq) and np.array_equal(q.rows("k")[1], wd, equal_nan=True)
    assert np.array_equal(back.rows("v"), values(wq, wd), equal_nan=True)
    assert np.isnan(back.rows("v")).sum() == 64
    for x in (c, q, back):
        x.free()


def test_copies_within_one_cache(dev):
    for q8_0 in (False, True):
        c = cache(dev, 4, 3, 40, q8_0)
        old = c.rows("k")
        htr.kv_copy(dev, c.kv, 2, c.kv, 20, 18)
        for g, o in zip(c.rows("k") if q8_0 else (c.rows("k"),), old if q8_0 else (old,)):
            e = o.copy()
            e[:, 20:38] = o[:, 2:20]
            assert np.array_equal(bits(g), bits(e))
        c.free()


@pytest.mark.parametrize("q8_0", [False, True], ids=["f16", "q8_0"])
@pytest.mark.parametrize("row0,idx", [(5, [0, 2, 3, 9]), (0, [63] * 64), (7, list(range(40, 0, -1))), (60, [39]), (0, [])])
def test_rows_kept(dev, q8_0, row0, idx):
    """every row read before any is written, whatever their order; the rest stays"""
    c = cache(dev, 6, 8, 100, q8_0)
    old = {w: c.rows(w) for w in "kv"}
    htr.kv_keep(dev, c.kv, row0, idx)
    for w in "kv":
        for g, o in zip(c.rows(w) if q8_0 else (c.rows(w),), old[w] if q8_0 else (old[w],)):
            e = o.copy()
            e[:, row0:row0 + len(idx)] = o[:, [row0 + i for i in idx]]
            assert np.array_equal(bits(g), bits(e))
    c.free()


# ---- attention --------------------------------------------------------------------------------------------------------------

def run_tree(dev, q, c, tree, past, scale=SCALE, gap=0):
    n, n_head = q.shape[:2]
    out = dev.upload(np.full((n + 1, n_head * 128), 7.0, np.float32))
    qb = strided(dev, q.reshape(n, -1), gap)
    htr.tree_attention(dev, qb, tree, past, c.kv, n_head, scale, out, q_stride=n_head * 128 + gap)
    got = out.download(np.float32).reshape(n + 1, -1)
    assert np.all(got[n] == 7.0)
    for b in (out, qb):
        b.free()
    return got[:n]


def run_window(dev, q, c, pos0, window, sink, scale=SCALE, gap=0):
    n, n_head = q.shape[:2]
    out = dev.upload(np.full((n + 1, n_head * 128), 7.0, np.float32))
    qb = strided(dev, q.reshape(n, -1), gap)
    htr.window_attention(dev, qb, n, pos0, window, sink, c.kv, n_head, scale, out, q_stride=n_head * 128 + gap)
    got = out.download(np.float32).reshape(n + 1, -1)
    assert np.all(got[n] == 7.0)
    for b in (out, qb):
        b.free()
    return got[:n]


def tree_seen(masks, past, rows):
    n = len(masks)
    seen = np.zeros((n, rows), bool)
    seen[:, :past] = True
    for i, m in enumerate(masks):
        for j in range(n):
            seen[i, past + j] = (int(m) >> j) & 1
    return seen


def window_seen(n, pos0, window, sink, rows):
    p, j = pos0 + np.arange(n)[:, None], np.arange(rows)[None, :]
    return (j <= p) & ((j < sink) | (j > p - window))


def random_tree(seed, n):
    rng = np.random.default_rng(seed)
    return htr.Tree([-1] + [int(rng.integers(max(-1, i - 4), i)) for i in range(1, n)])


@pytest.mark.parametrize("q8_0", [False, True], ids=["f16", "q8_0"])
@pytest.mark.parametrize("n,past,n_kv,group,gap", [
    (1, 0, 1, 1, 0), (1, 1, 8, 2, 0), (1, 31, 2, 2, 4), (1, 300, 8, 2, 512), (2, 32, 2, 3, 0), (5, 0, 1, 7, 0), (16, 63, 8, 2, 0),
    (17, 511, 2, 2, 128), (33, 100, 3, 1, 0), (64, 0, 2, 2, 0), (64, 1000, 8, 2, 0), (61, 200, 1, 16, 0), (40, 33, 1, 40, 0)])
def test_tree_attention(dev, q8_0, n, past, n_kv, group, gap):
    tree, rows = random_tree(n, n), past + n + 3
    c = cache(dev, 100 + n, n_kv, rows, q8_0)
    for b in c.bufs[:2]:  # what lies past the draft is not there
        a = b.download(np.uint8).reshape(n_kv, rows, -1)
        a[:, past + n:] = 0xFF if not q8_0 else 0x7F
        b.upload(a)
    q = normal(n, n, n_kv * group, 128)
    got = run_tree(dev, q, c, tree, past, gap=gap)
    want = attention(q, c.k, c.v, tree_seen(tree.masks, past, rows), SCALE)
    e = rel_rows(got, want)
    print(f"\n[tree {n} on {past}, {n_kv} x {group}] {e:.2e}", flush=True)
    assert e < BAR
    if n > 1:  # a chain without masks is a chain's tree
        a = run_tree(dev, q, c, n, past)
        assert np.array_equal(bits(a), bits(run_tree(dev, q, c, htr.Tree(np.arange(n) - 1), past)))
    c.free()


@pytest.mark.parametrize("past", [0, 20])
def test_tree_masks_of_any_kind(dev, past):
    """masks that are no tree's: rows that see nothing (zeros, where no key is committed), one row for all, later rows"""
    n, n_kv = 37, 2
    rng = np.random.default_rng(past)
    masks = np.array([int(rng.integers(0, 2 ** n)) & int(rng.integers(0, 2 ** n)) for _ in range(n)], np.uint64)
    masks[[3, 11, 36]] = 0
    masks[5] = 1 << 36
    c, q = cache(dev, 11, n_kv, past + n), normal(12, n, 4, 128)
    got = run_tree(dev, q, c, htr.Tree.of_masks(masks), past)
    want = attention(q, c.k, c.v, tree_seen(masks, past, past + n), SCALE)
    assert rel_rows(got, want) < BAR
    assert np.all(got[[3, 11, 36]] == 0) == (past == 0)
    empty = run_tree(dev, q[:2], c, htr.Tree.of_masks([0, 0]), 0)
    assert np.all(empty == 0)
    c.free()


@pytest.mark.parametrize("q8_0", [False, True], ids=["f16", "q8_0"])
@pytest.mark.parametrize("n,pos0,window,sink,n_kv,group,gap", [
    (1, 0, 1, 0, 1, 1, 0), (1, 0, 5, 3, 2, 2, 0), (1, 500, 64, 4, 8, 2, 128), (1, 500, 1, 0, 2, 1, 0), (3, 29, 2, 40, 2, 2, 0),
    (33, 0, 8, 0, 2, 2, 0), (40, 100, 33, 1, 1, 5, 0), (65, 31, 32, 64, 2, 2, 4), (130, 0, 1000, 0, 8, 2, 0), (200, 70, 50, 33, 1, 3, 0),
    (300, 11, 97, 5, 2, 4, 0), (257, 0, 2 ** 31 - 1, 2 ** 31 - 1, 1, 2, 0), (70, 40, 1, 2, 2, 2, 0),
    (150, 100, 33, 40, 64, 3, 4), (131, 0, 2 ** 31 - 1, 0, 128, 2, 0), (99, 7, 50, 0, 128, 2, 0)])
def test_window_attention(dev, q8_0, n, pos0, window, sink, n_kv, group, gap):
    rows = pos0 + n + 2
    c = cache(dev, 200 + n, n_kv, rows, q8_0)
    for b in c.bufs[:2]:
        a = b.download(np.uint8).reshape(n_kv, rows, -1)
        a[:, pos0 + n:] = 0xFF if not q8_0 else 0x7F
        b.upload(a)
    q = normal(n + 1, n, n_kv * group, 128)
    got = run_window(dev, q, c, pos0, window, sink, gap=gap)
    want = attention(q, c.k, c.v, window_seen(n, pos0, window, sink, rows), SCALE)
    e = rel_rows(got, want)
    print(f"\n[window {window}+{sink}, {n} from {pos0}, {n_kv} x {group}] {e:.2e}", flush=True)
    assert e < BAR
    c.free()


def test_attention_over_q8_0_is_that_over_its_read_back(dev):
    """bit for bit, from one token to a long prompt: a q8_0 element stands for f16(q·d)"""
    c = cache(dev, 31, 8, 3000, True)
    back = cache(dev, 33, 8, 3000)
    htr.kv_copy(dev, c.kv, 0, back.kv, 0, 3000)
    q = normal(34, 2000, 16, 128)
    for n, past in ((1, 2900), (64, 2900), (13, 7)):
        t = random_tree(n, n)
        assert np.array_equal(bits(run_tree(dev, q[:n], c, t, past)), bits(run_tree(dev, q[:n], back, t, past)))
    for n, pos0, w, s in ((1, 2000, 500, 4), (700, 1000, 300, 4), (700, 2300, 2 ** 20, 0),
                          (2000, 1000, 300, 4), (2000, 1000, 2 ** 20, 0)):
        assert np.array_equal(bits(run_window(dev, q[:n], c, pos0, w, s)), bits(run_window(dev, q[:n], back, pos0, w, s)))
    c.free()
    back.free()


def test_attention_agrees_with_the_decode_and_prefill_attention(dev):
    """one token as htr_decode_attention, a window past the whole cache as htr_causal_attention. Both sides of the first are
    within BAR. htr_causal_attention holds a q element whose f32 product with the scale is a tie between two f16 values an
    f16 ulp off (5e-5 of the elements, so every two hundredth head or so has one): 2^-10·|q·scale| at most, times |k| in a
    key's score; the softmax turns a score's error into as much of its weight, and the weights' sum into as much again"""
    n_head, n_kv, rows = 16, 8, 700
    c, q = cache(dev, 41, n_kv, rows), normal(42, 300, n_head, 128)
    out = dev.alloc(q.nbytes)
    qb = dev.upload(q)
    htr.decode_attention(dev, qb, c.bufs[0], c.bufs[1], n_head, n_kv, rows, rows, SCALE, out)
    one = out.download(np.float32, n_head * 128)
    assert rel_rows(run_tree(dev, q[:1], c, 1, rows - 1), one.astype(np.float64)) < 2 * BAR
    htr.causal_attention(dev, qb, c.bufs[0], c.bufs[1], 300, 400, n_head, n_kv, rows, SCALE, out)
    many = out.download(np.float32).reshape(300, -1)
    ulp = 2.0 ** -10 * float(np.abs(q).max()) * SCALE * float(np.abs(c.k).max())
    assert rel_rows(run_window(dev, q, c, 400, rows, 0), many.astype(np.float64)) < 2 * BAR + 2 * ulp
    c.free()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_rows_that_are_not_seen_do_not_matter(dev, bad):
    """K and V rows that some queries see and others do not: those that do not are bit for bit as without them; those that
    do get values that are not finite. So too in blocks that are wholly out of the window"""
    n, past, n_kv = 40, 50, 2
    tree = random_tree(7, n)
    k, v = normal(1, n_kv, past + n, 128).astype(np.float16), normal(2, n_kv, past + n, 128).astype(np.float16)
    q = normal(3, n, 6, 128)
    hit = 4
    sees = (tree.masks >> np.uint64(hit)) & np.uint64(1) != 0
    assert 0 < sees.sum() < n
    for which in (0, 1):
        kk, vv = k.copy(), v.copy()
        (kk, vv)[which][:, past + hit, 17] = bad
        c, clean = Cache(dev, kk, vv), Cache(dev, k, v)
        got, want = run_tree(dev, q, c, tree, past), run_tree(dev, q, clean, tree, past)
        plain = attention(q, k, v, tree_seen(tree.masks, past, past + n), SCALE)
        # (where V is not finite the block's products are summed one by one: another order)
        assert rel_rows(got[~sees], plain[~sees]) < BAR
        if which == 0:
            assert np.array_equal(bits(got[~sees]), bits(want[~sees]))
        col = got[sees].reshape(-1, 128)[:, 17]
        assert not np.any(np.isfinite(col)) if which else True
        c.free()
        clean.free()
    rows, w = 200, 30
    k, v = normal(1, 1, rows, 128).astype(np.float16), normal(2, 1, rows, 128).astype(np.float16)
    q = normal(4, rows, 2, 128)
    seen = window_seen(rows, 0, w, 2, rows)
    for at in (2, 40, 100, rows - 1):
        kk, vv = k.copy(), v.copy()
        kk[0, at], vv[0, at, ::3] = bad, bad
        c = Cache(dev, kk, vv)
        got = run_window(dev, q, c, 0, w, 2)
        free = ~seen[:, at]
        assert rel_rows(got[free], attention(q, k, v, seen, SCALE)[free]) < BAR
        assert not np.any(np.isfinite(got[~free].reshape(-1, 128)[:, 0]))
        c.free()


@pytest.mark.parametrize("size", [2.0 ** -140, 2.0 ** -60, 2.0 ** -20, 40.0, 3000.0, 2.0 ** 25])
def test_queries_of_any_size(dev, size):
    """q from subnormals, whose weights are equal, to scores of 1e9, whose softmax is one key's. A score s errs by 2^-21·|s|
    (q's pair and product, the sum), and as much of p: the bar grows with the largest score; where that leaves nothing of the
    smaller weights, keys far apart are taken, and the largest's values are the answer"""
    n, past, n_kv = 6, 90, 2
    c = cache(dev, 61, n_kv, past + n)
    q = normal(62, n, 4, 128) * np.float32(size)
    seen = tree_seen(htr.Tree(np.arange(n) - 1).masks, past, past + n)
    want = attention(q, c.k, c.v, seen, SCALE)
    got = run_tree(dev, q, c, n, past)
    s = np.abs(np.einsum("thd,hkd->thk", q.astype(np.float64), np.repeat(c.k, 2, axis=0).astype(np.float64))) * SCALE
    worst = 0.0
    for t in range(n):
        for h in range(4):
            at = np.sort(s[t, h][seen[t]])
            bar = BAR * max(1.0, at[-1] / 8)
            if bar > 1e-2:  # the two largest scores are far apart here, beside what they err by
                z = np.sort((c.k[h // 2][seen[t]].astype(np.float64) @ q[t, h].astype(np.float64)) * SCALE)
                assert z[-1] - z[-2] > 40 + 2.0 ** -19 * at[-1]
                bar = BAR
            g, w = got[t].reshape(4, 128)[h], want[t].reshape(4, 128)[h]
            worst = max(worst, np.linalg.norm(g - w) / np.linalg.norm(w) / bar)
    assert worst < 1.0, worst
    c.free()


# (queries, q heads to a KV head, KV heads): each of the kernels that a call may take
WAYS = [(3, 2, 2), (11, 2, 8), (40, 3, 2), (200, 2, 64)]


@pytest.mark.parametrize("n,group,n_kv", WAYS)
@pytest.mark.parametrize("q8_0", [False, True], ids=["f16", "q8_0"])
def test_scores_that_grow_and_fall(dev, n, group, n_kv, q8_0):
    """the largest score moves with almost every block, up and down by hundreds, so that every sum is taken again and again to
    another reference: a score of size s errs by 2^-21·s (see the sizes below), and as much its weight"""
    rows, window = 900, 700
    k = normal(1, n_kv, rows, 128, std=0.3)
    k[..., 0] = np.float32(40.0) * np.sin(np.arange(rows) / 37.0).astype(np.float32)
    c = Cache(dev, k.astype(np.float16), normal(2, n_kv, rows, 128, std=4.0).astype(np.float16), q8_0)
    q = normal(3, n, n_kv * group, 128)
    q[..., 0] = np.where(np.arange(n) % 2, 6.0, -6.0)[:, None]
    pos0 = rows - n
    got = run_window(dev, q, c, pos0, window, 20, 1.0)
    heads_seen = slice(0, 2) if n_kv == 64 else slice(0, n_kv)  # (the plain form is slow)
    keep = q.reshape(n, n_kv, group, 128)[:, heads_seen].reshape(n, -1, 128)
    want = attention(keep, c.k[heads_seen], c.v[heads_seen], window_seen(n, pos0, window, 20, rows), 1.0)
    assert rel_rows(got.reshape(n, n_kv, group * 128)[:, heads_seen].reshape(n, -1), want) < BAR * 250 / 8
    c.free()


@pytest.mark.parametrize("n,group,n_kv", WAYS)
@pytest.mark.parametrize("q8_0", [False, True], ids=["f16", "q8_0"])
def test_values_that_are_not_finite_in_every_kernel(dev, n, group, n_kv, q8_0):
    """a row of V with a NaN that the first queries do not see yet, one that has left the last ones' window, and one among the
    first keys: those that see none of them are as the plain form, the others not finite in those dims alone"""
    rows, window, sink = n + 300, 150, 3
    k, v = normal(1, n_kv, rows, 128).astype(np.float16), normal(2, n_kv, rows, 128).astype(np.float16)
    pos0 = rows - n
    bad = [(rows - 2, 5), (pos0 - window + 2, 70), (rows - n // 2 - 1, 100)]
    vv = v.copy()
    for r, d in bad:
        vv[:, r, d] = np.nan
    c = Cache(dev, k, vv, q8_0)
    kk, clean = (values(*blocks(x)) if q8_0 else x for x in (k, v))
    q = normal(3, n, n_kv * group, 128)
    got = run_window(dev, q, c, pos0, window, sink).reshape(n, n_kv * group, 128)
    seen = window_seen(n, pos0, window, sink, rows)
    hs = min(n_kv, 2)
    want = attention(q[:, :hs * group], kk[:hs], clean[:hs], seen, SCALE).reshape(n, hs * group, 128)
    for t in range(n):
        hit = {d2 for r, d in bad if seen[t, r] for d2 in (range(d // 32 * 32, d // 32 * 32 + 32) if q8_0 else (d,))}
        fine = [d for d in range(128) if d not in hit]
        assert not hit or not np.any(np.isfinite(got[t][:, sorted(hit)])), t
        assert np.all(np.isfinite(got[t][:, fine])), t
        if t % 7 == 0 or n < 20:
            e = np.linalg.norm(got[t, :hs * group][:, fine] - want[t][:, fine], axis=1) / np.linalg.norm(want[t][:, fine], axis=1)
            assert np.all(e < BAR), t
    c.free()


@pytest.mark.parametrize("q8_0", [False, True], ids=["f16", "q8_0"])
def test_trees_of_very_many_heads(dev, q8_0):
    """512 q heads on 128: the kernel of many rows, on a tree"""
    n, past, n_kv = 64, 77, 128
    t = random_tree(5, n)
    c, q = cache(dev, 121, n_kv, past + n, q8_0), normal(122, n, 512, 128)
    got = run_tree(dev, q, c, t, past).reshape(n, n_kv, 512)
    want = attention(q[:, 8:16], c.k[2:4], c.v[2:4], tree_seen(t.masks, past, past + n), SCALE)
    assert rel_rows(got[:, 2:4].reshape(n, -1), want) < BAR
    c.free()


@pytest.mark.parametrize("n,group,n_kv", WAYS)
def test_queries_that_are_not_finite(dev, n, group, n_kv):
    """a query with a NaN and one with an infinity: their outputs are not finite, every other bit for bit as without them"""
    rows = 400
    c, q = cache(dev, 161, n_kv, rows), normal(162, n, n_kv * group, 128)
    want = run_window(dev, q, c, rows - n, 170, 3).reshape(n, -1, 128)
    q[1, 0, 5], q[n - 1, -1, 127] = np.nan, -np.inf
    got = run_window(dev, q, c, rows - n, 170, 3).reshape(n, -1, 128)
    assert not np.any(np.isfinite(got[1, 0])) and not np.any(np.isfinite(got[n - 1, -1]))
    got[1, 0], got[n - 1, -1] = want[1, 0], want[n - 1, -1]
    assert np.array_equal(bits(got), bits(want))
    c.free()


def test_calls_of_changing_shapes_share_the_scratch(dev):
    """one call after another over caches of 8, 2 and 16 KV heads (partial sums and tickets in an XCD's L2, and through the
    coherence point), of one to 64 nodes: each as alone"""
    for i, (n, past, n_kv, group) in enumerate([(1, 3000, 8, 2), (1, 3000, 2, 2), (20, 2000, 8, 1), (64, 900, 16, 1), (1, 1000, 16, 3), (9, 5000, 8, 1),
                                                (1, 4000, 8, 2), (30, 3000, 1, 2), (1, 700, 8, 4), (60, 1500, 4, 4), (64, 3000, 2, 2),
                                                (33, 900, 1, 8), (60, 1100, 4, 4), (2, 900, 3, 2)]):
        t = random_tree(i, n)
        c, q = cache(dev, 130 + i, n_kv, past + n, i % 2 == 1), normal(140 + i, n, n_kv * group, 128)
        assert rel_rows(run_tree(dev, q, c, t, past), attention(q, c.k, c.v, tree_seen(t.masks, past, past + n), SCALE)) < BAR, i
        c.free()


def test_graphs_outlive_the_scratch_they_were_recorded_over(dev):
    """many queries over a q8_0 cache read rows back into scratch: a graph recorded over it replays right after a larger call
    has made it anew, and a call that would make it cannot be recorded"""
    d = htr.Device(0)
    n_kv, n = 64, 200
    c, q = cache(d, 151, n_kv, 700, True), normal(152, n, 2 * n_kv, 128)
    qb, out = d.upload(q), d.alloc(q.nbytes)
    call = lambda cc, pos0: htr.window_attention(d, qb, n, pos0, 300, 4, cc.kv, 2 * n_kv, SCALE, out)  # noqa: E731
    d.capture_begin()
    with pytest.raises(htr.HtrError, match="captured"):
        call(c, 500)
    d.capture_end().free()
    call(c, 500)
    want = out.download(np.float32)
    d.capture_begin()
    call(c, 500)
    g = d.capture_end()
    big = Cache(d, *(np.zeros((n_kv, 9000, 128), np.float16) for _ in range(2)), True)
    before = d.mem_live()["work"]
    htr.window_attention(d, qb, n, 8000, 9000, 4, big.kv, 2 * n_kv, SCALE, out)
    assert d.mem_live()["work"] > before
    for _ in range(3):
        out.upload(np.zeros(q.size, np.float32))
        g.launch()
        assert np.array_equal(bits(out.download(np.float32)), bits(want))
    g.free()
    d.close()


def test_negative_and_zero_scale(dev):
    c, q = cache(dev, 71, 1, 80), normal(72, 3, 2, 128)
    seen = tree_seen(htr.Tree(np.arange(3) - 1).masks, 77, 80)
    for scale in (-0.1, 0.0, 1.5):
        assert rel_rows(run_tree(dev, q, c, 3, 77, scale), attention(q, c.k, c.v, seen, scale)) < BAR * 8
    c.free()


def test_long_caches(dev):
    """70001 keys (every workgroup has a part) of both types, one token and a tree; a window at their end"""
    past, n_kv = 70001, 2
    for q8_0 in (False, True):
        c = cache(dev, 81, n_kv, past + 20, q8_0)
        q = normal(82, 20, 4, 128)
        for n in (1, 20):
            t = random_tree(n, n)
            assert rel_rows(run_tree(dev, q[:n], c, t, past), attention(q[:n], c.k, c.v, tree_seen(t.masks, past, past + 20), SCALE)) < BAR
        assert rel_rows(run_window(dev, q, c, past, 5000, 40), attention(q, c.k, c.v, window_seen(20, past, 5000, 40, past + 20), SCALE)) < BAR
        c.free()


def test_rows_past_four_gib(dev):
    """a cache of 2^24 + 200 rows (its bytes pass 32 bits): rows written, copied, kept and attended to at its end"""
    rows, n = 2 ** 24 + 200, 9
    big = htr.KvCache(dev, 1, rows)
    end = rows - n
    k, v = normal(1, 1, n, 128).astype(np.float16), normal(2, 1, n, 128).astype(np.float16)
    small, back = Cache(dev, k, v), cache(dev, 5, 1, n)
    htr.kv_copy(dev, small.kv, 0, big, end, n)
    htr.kv_keep(dev, big, end, [0, 1, 2, 8, 7])
    order = [0, 1, 2, 8, 7, 5, 6, 7, 8]
    htr.kv_copy(dev, big, end, back.kv, 0, n)
    assert np.array_equal(bits(back.rows("k")), bits(k[:, order])) and np.array_equal(bits(back.rows("v")), bits(v[:, order]))
    q = normal(3, n, 2, 128)
    got = run_window(dev, q, type("c", (), {"kv": big}), end, 5, 0)
    ko, vo = (np.concatenate([np.zeros((1, 8, 128), np.float16), x[:, order]], axis=1) for x in (k, v))
    assert rel_rows(got, attention(q, ko, vo, window_seen(n, 8, 5, 0, 8 + n), SCALE)) < BAR
    # a tree on the zeros before it: 2^24 + 191 scores of 0, whose equal weights f32 sums exactly (8 each, 2^24 of them)
    t = random_tree(4, n)
    got = run_tree(dev, q, type("c", (), {"kv": big}), t, end)
    seen, want = tree_seen(t.masks, 0, n), np.zeros((n, 2, 128))
    for i in range(n):
        for h in range(2):
            s = np.where(seen[i], k[0, order].astype(np.float64) @ q[i, h].astype(np.float64) * SCALE, -np.inf)
            want[i, h] = np.exp(s) @ v[0, order].astype(np.float64) / (end + np.exp(s).sum())
    assert rel_rows(got, want.reshape(n, -1)) < BAR
    for b in (small, back):
        b.free()
    big.free()


# ---- together -----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("q8_0", [False, True], ids=["f16", "q8_0"])
def test_a_drafted_step_together_and_as_graphs(dev, q8_0):
    """rows made and stored, the draft's attention, the accepted path kept; then two captured graphs of such steps, which
    share the scratch of partial sums, replayed in turn with eager calls between them: every output as the eager one's"""
    n_head, n_kv, past = 16, 8, 1300
    L = []
    for i, n in enumerate((23, 64)):
        tree = random_tree(i + 1, n)
        rows = past + n + 1
        x = normal(90 + i, n, n_head + 2 * n_kv, 128)
        c = cache(dev, 91 + i, n_kv, rows, q8_0)
        cs = orc.rope_table(1e6, 128, rows + 64).reshape(-1, 64, 2)
        w = normal(93, 128, std=0.02) + 1
        path, j = [], n - 1
        while j >= 0:
            path.append(j)
            up = [p for p in range(j) if (int(tree.masks[j]) >> p) & 1]
            j = up[-1] if up else -1
        L.append(dict(n=n, tree=tree, c=c, path=path[::-1], raw=dev.upload(x), w=dev.upload(w), cs=dev.upload(cs), n_pos=cs.shape[0],
                      q=dev.alloc(n * n_head * 512), out=dev.alloc(n * n_head * 512), x=x, wh=w, csh=cs))

    class At:
        def __init__(self, ptr):
            self.ptr = ptr

    def step(s):
        r, width = s["raw"].ptr, (n_head + 2 * n_kv) * 128
        htr.qkv_post_rows(dev, At(r), At(r + n_head * 512), At(r + (n_head + n_kv) * 512), s["n"], s["w"], s["w"], s["cs"], s["n_pos"],
                          past, n_head, EPS, s["c"].kv, past, s["q"], q_stride=width, kv_stride=width, tree=s["tree"])
        htr.tree_attention(dev, s["q"], s["tree"], past, s["c"].kv, n_head, SCALE, s["out"])
        htr.kv_keep(dev, s["c"].kv, past, s["path"])

    def result(s):
        rows = [r for w in "kv" for r in (s["c"].rows(w) if q8_0 else (s["c"].rows(w),))]
        return [s["q"].download(np.float32), s["out"].download(np.float32)] + rows

    for s in L:
        step(s)
        s["want"] = result(s)
        n, pos = s["n"], past + s["tree"].depths
        q = heads(s["x"][:, :n_head], s["wh"], s["csh"][pos])
        k, v = heads(s["x"][:, n_head:-n_kv], s["wh"], s["csh"][pos]).transpose(1, 0, 2), s["x"][:, -n_kv:].transpose(1, 0, 2)
        k, v = ((values(*blocks(a)) if q8_0 else a.astype(np.float16)) for a in (k, v))
        ko, vo = s["c"].k.copy(), s["c"].v.copy()
        ko[:, past:past + n], vo[:, past:past + n] = k, v
        want = attention(q, ko, vo, tree_seen(s["tree"].masks, past, past + n + 1), SCALE)
        assert rel_rows(s["want"][1].reshape(n, -1), want) < BAR
    graphs = []
    for s in L:
        dev.capture_begin()
        step(s)
        graphs.append(dev.capture_end())
    one = normal(99, 1, n_head, 128)
    for rep in range(3):
        for g, s in zip(graphs, L):
            s["out"].upload(np.full(s["n"] * n_head * 128, np.nan, np.float32))
            g.launch()
            run_tree(dev, one, L[0]["c"], 1, past - 1)  # an eager call with partial sums of its own
            for a, b in zip(result(s), s["want"]):
                assert np.array_equal(bits(a), bits(b)), rep
    # both graphs in one go, nothing waiting between them
    for g in graphs + graphs[::-1]:
        g.launch()
    for s in L:
        for a, b in zip(result(s), s["want"]):
            assert np.array_equal(bits(a), bits(b))
    for g in graphs:
        g.free()
    for s in L:
        s["c"].free()


def test_window_attention_as_a_graph(dev):
    """captured at sizes that split the keys and that do not; replays equal the eager outputs, and calls repeat bit for bit"""
    c = cache(dev, 111, 8, 2600)
    q = dev.upload(normal(112, 600, 16, 128))
    for n, pos0 in ((1, 2500), (600, 2000)):
        out = dev.alloc(n * 16 * 512)
        htr.window_attention(dev, q, n, pos0, 1000, 4, c.kv, 16, SCALE, out)
        want = out.download(np.float32)
        dev.capture_begin()
        htr.window_attention(dev, q, n, pos0, 1000, 4, c.kv, 16, SCALE, out)
        g = dev.capture_end()
        for _ in range(3):
            out.upload(np.zeros(n * 16 * 128, np.float32))
            g.launch()
            assert np.array_equal(bits(out.download(np.float32)), bits(want))
        g.free()
    c.free()


def test_poisoned_scratch_and_another_thread(dev):
    """a second device object, its memory poisoned, driven from another thread: the same bits"""
    import os

    q, k, v = normal(1, 9, 16, 128), normal(2, 8, 400, 128).astype(np.float16), normal(3, 8, 400, 128).astype(np.float16)
    c = Cache(dev, k, v)
    want = run_tree(dev, q, c, 9, 391), run_window(dev, q, c, 300, 64, 4)
    got, keep = [], os.environ.get("HTR_POISON")

    def other():
        os.environ["HTR_POISON"] = "1"
        try:
            d = htr.Device(0)
        finally:
            os.environ.pop("HTR_POISON") if keep is None else os.environ.update(HTR_POISON=keep)
        oc = Cache(d, k, v)
        got.extend((run_tree(d, q, oc, 9, 391), run_window(d, q, oc, 300, 64, 4)))
        d.close()

    t = threading.Thread(target=other)
    t.start()
    t.join()
    assert len(got) == 2
    for a, b in zip(got, want):
        assert np.array_equal(bits(a), bits(b))
    c.free()


def test_a_session_s_layer_as_a_cache(dev):
    """a prefilled session's f16 layer: put aside in q8_0, read back into the session, and attended to as it lies"""
    from helpers import tiny_prompt, tiny_text_model, to_htr_cfg

    cfg, te, on, layers = tiny_text_model()
    m = htr.TextModel(dev, to_htr_cfg(cfg), te, on, layers)
    prompt = tiny_prompt()
    s = m.session(prompt.size + 8)
    s.prefill(prompt)
    view = s.kv_view()

    class At:
        def __init__(self, ptr):
            self.ptr = ptr

    layer = 3
    off = 2 * layer * view.layer_stride
    kv = htr.KvCache.of(view.n_kv, view.n_ctx, At(view.d_k + off), At(view.d_v + off))
    f16, q8 = htr.KvCache(dev, view.n_kv, prompt.size), htr.KvCache(dev, view.n_kv, prompt.size, q8_0=True)
    htr.kv_copy(dev, kv, 0, f16, 0, prompt.size)
    htr.kv_copy(dev, kv, 0, q8, 0, prompt.size)
    rows = f16.k.download(np.float16).reshape(view.n_kv, -1, 128)
    vals = f16.v.download(np.float16).reshape(view.n_kv, -1, 128)
    q = normal(5, 1, cfg["n_head"], 128)
    got = run_tree(dev, q, type("c", (), {"kv": kv}), 1, prompt.size - 1)
    assert rel_rows(got, attention(q, rows, vals, np.ones((1, prompt.size), bool), SCALE)) < BAR
    htr.kv_copy(dev, q8, 0, kv, 0, prompt.size)
    htr.kv_copy(dev, kv, 0, f16, 0, prompt.size)
    assert np.array_equal(bits(f16.k.download(np.float16).reshape(rows.shape)), bits(values(*blocks(rows))))
    logits = s.step(int(prompt[0]))
    assert np.all(np.isfinite(logits))
    for x in (f16, q8, s, m):
        x.free()


def test_capture_before_the_scratch_exists_is_refused(dev):
    """a call that would make the scratch fails while the stream is captured, and the device stays alive"""
    d = htr.Device(0)
    c, q = cache(d, 1, 8, 600), normal(2, 1, 16, 128)
    qb, out = d.upload(q), d.alloc(16 * 512)
    d.capture_begin()
    with pytest.raises(htr.HtrError, match="captured"):
        htr.tree_attention(d, qb, 1, 599, c.kv, 16, SCALE, out)
    d.capture_end().free()
    d.alive()
    htr.tree_attention(d, qb, 1, 599, c.kv, 16, SCALE, out)
    assert rel_rows(out.download(np.float32), attention(q, c.k, c.v, np.ones((1, 600), bool), SCALE)) < BAR
    d.close()


# ---- what a row sees, and nothing else, makes its output --------------------------------------------------------------------

@pytest.mark.parametrize("n,group,n_kv", WAYS)
@pytest.mark.parametrize("scale", [511.75, 512.0, 515.5, 65504.0])
def test_quants_of_minus_128_at_scales_that_overflow(dev, n, group, n_kv, scale):
    """a q8_0 cache may hold the quant -128 (this library writes none): with a scale of 512 and more f16(q·d) is an infinity.
    V rows with such an element that the first queries do not see yet, and one just before every query's window: those that
    see none of them get the clean cache's bits, and all of them those over the cache's read-back"""
    rows, window, sink = n + 300, 150, 3
    (qk, dk), (qv, dv) = (blocks(normal(s, n_kv, rows, 128).astype(np.float16)) for s in (1, 2))
    pos0 = rows - n
    at = [(rows - 2, 5), (pos0 - window, 70), (rows - n // 2 - 1, 100)]
    bq, bd = qv.copy(), dv.copy()
    for r, d in at:
        bq[:, r, d // 32 * 32:d // 32 * 32 + 32], bq[:, r, d], bd[:, r, d // 32] = 1, -128, scale
    q = normal(3, n, n_kv * group, 128)
    got = []
    for v, d in ((bq, bd), (qv, dv)):
        bufs = [dev.upload(a) for a in (qk, v, dk, d)]
        kv = htr.KvCache.of(n_kv, rows, *bufs)
        back = htr.KvCache(dev, n_kv, rows)
        htr.kv_copy(dev, kv, 0, back, 0, rows)
        for c in (kv, back):
            got.append(run_window(dev, q, type("c", (), {"kv": c}), pos0, window, sink))
        for b in bufs + [back]:
            b.free()
    assert np.array_equal(got[0], got[1], equal_nan=True) and np.array_equal(bits(got[2]), bits(got[3]))
    seen = window_seen(n, pos0, window, sink, rows)
    free = ~seen[:, [r for r, _ in at]].any(axis=1)
    assert 0 < free.sum() < n
    assert np.array_equal(bits(got[0][free]), bits(got[2][free]))
    for r, d in at:
        hit = got[0][seen[:, r]].reshape(-1, 128)[:, d]
        assert np.all(np.isfinite(hit)) if scale < 512 else not np.any(np.isfinite(hit))


def test_a_quant_of_minus_128_in_a_draft(dev):
    """the same in trees: of one node's row (few rows, and more), with the masks of its siblings without it"""
    for n, n_kv, group in ((5, 2, 2), (40, 2, 3)):
        past, hit = 50, 2
        (qk, dk), (qv, dv) = (blocks(normal(s, n_kv, past + n, 128).astype(np.float16)) for s in (1, 2))
        bq, bd = qv.copy(), dv.copy()
        bq[:, past + hit, :32], bd[:, past + hit, 0] = -128, 513.5
        masks = np.array([(2 << i) - 1 if i % 2 else ((2 << i) - 1) & ~(1 << hit) for i in range(n)], np.uint64)
        q, got = normal(3, n, n_kv * group, 128), []
        for v, d in ((bq, bd), (qv, dv)):
            bufs = [dev.upload(a) for a in (qk, v, dk, d)]
            got.append(run_tree(dev, q, type("c", (), {"kv": htr.KvCache.of(n_kv, past + n, *bufs)}), htr.Tree.of_masks(masks), past))
            for b in bufs:
                b.free()
        sees = (masks >> np.uint64(hit)) & np.uint64(1) != 0
        assert np.array_equal(bits(got[0][~sees]), bits(got[1][~sees])), n
        assert not np.any(np.isfinite(got[0][sees].reshape(-1, 128)[:, :32])), n


@pytest.mark.parametrize("n,group,n_kv,window", [(3, 2, 8, 300), (11, 2, 8, 600), (40, 3, 2, 600), (200, 2, 64, 700)])
@pytest.mark.parametrize("q8_0", [False, True], ids=["f16", "q8_0"])
def test_a_key_moves_only_the_rows_that_see_it(dev, n, group, n_kv, window, q8_0):
    """a key that the later queries see, with a score far above all others or an infinite one in some of them: the outputs of
    the queries before it are bit for bit as with an ordinary key there, though the kernels take their rows together"""
    rows, sink = 900, 20
    pos0, r = rows - n, rows - 1 - n // 2
    k, v = normal(1, n_kv, rows, 128).astype(np.float16), normal(2, n_kv, rows, 128).astype(np.float16)
    q = normal(3, n, n_kv * group, 128)
    c = Cache(dev, k, v, q8_0)
    want = run_window(dev, q, c, pos0, window, sink)
    c.free()
    before = pos0 + np.arange(n) < r
    assert 0 < before.sum() < n
    for change in (2.0, np.inf):
        kk = k.copy()
        if change == 2.0:
            kk[:, r] = change * q[n - 1].reshape(n_kv, group, 128)[:, 0]
        else:
            kk[:, r, 40] = change
        c = Cache(dev, kk, v, q8_0)
        got = run_window(dev, q, c, pos0, window, sink)
        c.free()
        assert np.array_equal(bits(got[before]), bits(want[before])), change
        assert not np.array_equal(bits(got[~before]), bits(want[~before]))


@pytest.mark.parametrize("kind", ["few", "split", "many"])
@pytest.mark.parametrize("q8_0", [False, True], ids=["f16", "q8_0"])
def test_small_weights_of_many_keys_count(dev, kind, q8_0):
    """a few first keys take the largest weights, 2^28 times those of the many others: each of those is nothing beside them,
    2^13 … 2^15 of them in a wave's run are not. A weight is held to 2^-22 of itself or 2^-35 of the largest, so the values'
    sum of N of them errs by N·2^-35 of the largest value (2^-20 at most here), beside the exponential's and the f32 sums'
    2^-21: 2^-18 leaves room. The keys' scores are exact: the queries have one dim that is not 0"""
    if kind == "few":  # one token; a part of 2^13 keys to a workgroup, a large key at each one's start
        n, rows, large = 1, 2 ** 19, np.arange(0, 2 ** 19, 2 ** 13)
    elif kind == "split":  # a wave takes every eighth block of 32 keys: one large key in each of the first eight
        n, rows, large = 32 * 129, 2 ** 16 + 32 * 129, 32 * np.arange(8)
    else:  # a wave takes every other block
        n, rows, large = 32 * 3 * 256 + 64, 2 ** 15 + 32 * 3 * 256 + 64, 32 * np.arange(2)
    x = np.ones((1, rows, 128), np.float16)  # K and V alike: dim 0 makes the scores, the others are the values
    x[0, :, :32], x[0, large] = 0, 0
    x[0, large, 0] = 16
    scale = 28.03 / 16 / np.log2(np.e)
    if q8_0:
        qx, dx = blocks(x)
        x = values(qx, dx)
        bufs = [dev.upload(qx), dev.upload(dx)]
        kv = htr.KvCache.of(1, rows, bufs[0], bufs[0], bufs[1], bufs[1])
    else:
        bufs = [dev.upload(x)]
        kv = htr.KvCache.of(1, rows, bufs[0], bufs[0])
    q = np.zeros((n, 1, 128), np.float32)
    q[..., 0] = 1.0
    c = type("c", (), {"kv": kv})
    if kind == "few":
        got = run_tree(dev, q, c, 1, rows - 1, scale)
    else:
        got = run_window(dev, q, c, rows - n, rows, 0, scale)
    keys = rows - n + 1 + np.arange(n)
    w = np.exp(-float(x[0, 0, 0]) * float(np.float32(scale)))
    small = (keys - large.size) * w / (large.size + (keys - large.size) * w)
    tail = float(x[0, 1, 127])
    assert np.all(x[0, 1, 32:] == x[0, 1, 127]) and small.min() > 2.0 ** -17  # (more than the bar: that they count is seen)
    off = np.abs(got[:, 32:].astype(np.float64) - small[:, None] * tail)
    print(f"\n[{kind}] the small ones' share {small.max():.2e}, off by {off.max():.2e}", flush=True)
    assert off.max() < 2.0 ** -18 * tail
    for b in bufs:
        b.free()


def test_scratch_that_cannot_double_is_what_the_call_needs(dev):
    """room for rows read back is doubled when it grows, and exactly what the call needs where the doubled size is not there:
    the call goes on, and the device stays alive"""
    n_kv, n, gib = 64, 200, 1 << 30
    d = htr.Device(0)
    try:
        c = htr.KvCache(d, n_kv, 75000, q8_0=True)
        some = cache(d, 171, n_kv, 300, True)
        htr.kv_copy(d, some.kv, 0, c, 59700, 300)
        htr.kv_copy(d, some.kv, 0, c, 74700, 300)
        q = normal(172, n, 2 * n_kv, 128)
        at = type("c", (), {"kv": c})
        run_window(d, q, at, 60000 - n, 75000, 0)  # 2 · 64 · 60000 rows of 256 bytes: 1.83 GiB
        need, doubled = 2 * n_kv * 75000 * 256, 2 * 2 * n_kv * 60000 * 256
        free, total = C.c_size_t(), C.c_size_t()
        assert htr.lib().hipMemGetInfo(C.byref(free), C.byref(total)) == 0
        left = (need + doubled) // 2  # 0.7 GiB more than the call needs, as much less than it would like
        held = free.value - left
        while held > 0:
            d.alloc(min(held, 8 * gib))
            held -= 8 * gib
        before = d.mem_live()["work"]
        got = run_window(d, q, at, 75000 - n, 75000, 0)
        d.alive()
        assert d.mem_live()["work"] - before == need
        few = run_window(d, q[n - 4:], at, 74996, 75000, 0)  # (by a kernel that reads no rows back)
        assert rel_rows(got[n - 4:], few.astype(np.float64)) < 2 * BAR
    finally:
        d.close()


@pytest.mark.parametrize("sink", [0, 1, 33, 64])
@pytest.mark.parametrize("pos0,window", [(1500, 100), (1503, 1), (1520, 65)])
def test_windows_read_back_as_two_ranges(dev, pos0, window, sink):
    """many queries over a q8_0 cache whose first keys and window are far apart: the rows between are not read back, and the
    blocks past them lie further down than their keys say. The first row group's window starts on the second range's first
    block. What lies between is not finite, and what is seen as over the whole cache's read-back, bit for bit"""
    n, n_kv, group = 200, 64, 2
    rows = pos0 + n + 3
    first, from_row = (sink + 31) // 32 * 32, (pos0 - window + 1) // 32 * 32
    assert from_row - first > (pos0 + n) // 4
    k, v = (normal(s, n_kv, rows, 128).astype(np.float16) for s in (1, 2))
    c = Cache(dev, k, v, True)
    back = cache(dev, 3, n_kv, rows)
    htr.kv_copy(dev, c.kv, 0, back.kv, 0, rows)
    for b in c.bufs[2:]:
        d = b.download(np.float16).reshape(n_kv, rows, 4)
        d[:, first:from_row] = np.nan
        b.upload(d)
    q = normal(4, n, n_kv * group, 128)
    got, want = (run_window(dev, q, x, pos0, window, sink) for x in (c, back))
    assert np.array_equal(bits(got), bits(want))
    plain = attention(q[:, :4], c.k[:2], c.v[:2], window_seen(n, pos0, window, sink, rows), SCALE)
    assert rel_rows(got.reshape(n, -1, 128)[:, :4].reshape(n, -1), plain) < BAR
    c.free()
    back.free()


@pytest.mark.parametrize("n,group,n_kv", WAYS)
@pytest.mark.parametrize("q8_0", [False, True], ids=["f16", "q8_0"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_rows_that_are_not_seen_leave_every_bit(dev, n, group, n_kv, q8_0, bad):
    """K or V rows with a value that is not finite: the queries that do not see them are bit for bit as without, in every
    kernel, and of V the other dims of those that do too. A V value gives one that is not finite in its dims; a K value a
    score of NaN, and so outputs of NaN, or of an infinity, of which −∞ takes the key's weight"""
    rows, window, sink = n + 300, 150, 3
    k, v = normal(1, n_kv, rows, 128).astype(np.float16), normal(2, n_kv, rows, 128).astype(np.float16)
    pos0, r, d = rows - n, rows - n // 2 - 1, 100
    dims = list(range(96, 128)) if q8_0 else [d]
    seen = window_seen(n, pos0, window, sink, rows)
    sees = seen[:, r].copy()
    assert 0 < sees.sum() < n
    q = normal(3, n, n_kv * group, 128)
    clean = Cache(dev, k, v, q8_0)
    want = run_window(dev, q, clean, pos0, window, sink).reshape(n, -1, 128)
    seen[:, r] = False
    hs = min(n_kv, 2)
    without = attention(q[:, :hs * group], clean.k[:hs], clean.v[:hs], seen, SCALE).reshape(n, -1, 128)
    clean.free()
    for which in (0, 1):
        x = [k.copy(), v.copy()]
        x[which][:, r, d] = bad
        c = Cache(dev, *x, q8_0)
        got = run_window(dev, q, c, pos0, window, sink).reshape(n, -1, 128)
        c.free()
        assert np.array_equal(bits(got[~sees]), bits(want[~sees]))
        if which:
            others = [i for i in range(128) if i not in dims]
            assert not np.any(np.isfinite(got[sees][..., dims]))
            assert np.array_equal(bits(got[sees][..., others]), bits(want[sees][..., others]))
            continue
        nan = np.isnan(got[sees]).all(axis=2)
        if np.isnan(bad) or q8_0:  # (a q8_0 block with an infinity is NaN)
            assert nan.all()
            continue
        assert np.array_equal(nan, ~np.isfinite(got[sees]).all(axis=2))
        rest, plain, nan = got[sees][:, :hs * group], without[sees], nan[:, :hs * group]
        off = np.linalg.norm(rest - plain, axis=2) / np.linalg.norm(plain, axis=2)
        assert np.all(off[~nan] < BAR)


def test_rows_beside_those_of_a_decode_step(dev):
    """the same raw rows by htr_qkv_post, one at a time, and by htr_qkv_post_rows: V bit for bit; q and K within what the
    step's f32 norm and turn err by, some 16 roundings, 2^-20 of the pair's size, and, of K, an f16 ulp where a border lies
    between the two"""
    n, n_head, n_kv, pos0, n_ctx = 37, 16, 8, 611, 700
    x = normal(5, n, n_head + 2 * n_kv, 128, std=3.0)
    qn, kn = normal(6, 128, std=0.1) + 1, normal(7, 128, std=0.1) + 1
    cs = orc.rope_table(1e6, 128, n_ctx)
    w = [dev.upload(a) for a in (qn, kn, cs)]
    step, rows = cache(dev, 8, n_kv, n_ctx), cache(dev, 8, n_kv, n_ctx)
    q_step = np.empty((n, n_head, 128), np.float32)
    for t in range(n):
        raw = dev.upload(x[t])
        htr.qkv_post(dev, raw, *w, n_head, n_kv, pos0 + t, n_ctx, EPS, *step.bufs)
        q_step[t] = raw.download(np.float32, n_head * 128).reshape(n_head, 128)
        raw.free()
    raw, q_out, width = dev.upload(x), dev.alloc(n * n_head * 512), (n_head + 2 * n_kv) * 128

    class At:
        def __init__(self, ptr):
            self.ptr = ptr

    htr.qkv_post_rows(dev, raw, At(raw.ptr + n_head * 512), At(raw.ptr + (n_head + n_kv) * 512), n, *w, n_ctx, pos0, n_head, EPS,
                      rows.kv, pos0, q_out, q_stride=width, kv_stride=width)
    assert np.array_equal(bits(step.rows("v")), bits(rows.rows("v")))

    def pair(y):  # the size of each value's pair, a dim and the one 64 further on
        s = np.abs(y[..., :64].astype(np.float64)) + np.abs(y[..., 64:])
        return 2.0 ** -20 * np.concatenate([s, s], axis=-1)

    q_rows = q_out.download(np.float32).reshape(n, n_head, 128)
    assert np.all(np.abs(q_rows.astype(np.float64) - q_step) <= pair(q_rows))
    a, b = step.rows("k").astype(np.float64), rows.rows("k").astype(np.float64)
    ulp = 2.0 ** -10 * np.maximum(np.abs(a), np.abs(b)) + 2.0 ** -24
    assert np.all(np.abs(a - b) <= ulp + pair(b))
    print(f"\n[K rows that differ] {np.mean(a != b):.1e} of the cache's values", flush=True)
    for y in (step, rows, raw, q_out, *w):
        y.free()
