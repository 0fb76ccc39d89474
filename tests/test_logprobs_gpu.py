"""Log probabilities of given tokens, entropies and alternatives on the GPU against numpy in 64 bits."""
import numpy as np
import pytest

import htr

pytestmark = pytest.mark.gpu

# What the results may be off by. A term e^(x − m), of x − m ≥ −17 (below, all terms of a row together are 2^-7 of one such),
# errs by 17·2^-24 from the rounded difference and 2^-23 from the exponential; a sum of N terms in runs of N / 256 and fewer
# by √(N / 256)·2^-24, 25 of them for the largest vocabulary. Together below 64·2^-24 of r, and of W with one product more.
# log(1 + r) passes r's error on as r / (1 + r) of it; the last operations round three times.
DELTA = 64 * 2.0 ** -24


def reference(x, ids, top):
    """→ logprob, entropy, ids and log probabilities of the top, each with what it may be off by"""
    x64 = x.astype(np.float64)
    n, vocab = x.shape
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = np.max(np.where(np.isnan(x64), -np.inf, x64), axis=1, keepdims=True)
        broken = ~np.all(x64 < np.inf, axis=1)
        empty = ~broken & (m[:, 0] == -np.inf)
        first = np.argmax(x64 == m, axis=1)
        e = np.exp(np.where(np.isfinite(m), x64 - m, -np.inf))
        e[np.arange(n), first] = 0
        r = np.where(broken, np.nan, e.sum(axis=1))
        w = np.where(e > 0, e * (m - x64), 0).sum(axis=1)
        ln = np.log1p(r)

        def lp(v, rows=slice(None)):
            y = (v - m[rows, 0]) - ln[rows]
            y = np.where(empty[rows], -np.inf, np.where(broken[rows], np.nan, y))
            return y, DELTA * (r / (1 + r))[rows] + 2.0 ** -22 * np.abs(np.where(np.isfinite(y), y, 0)) + 1e-36

        ok = (ids >= 0) & (ids < vocab)
        got = lp(x64[np.arange(n), np.where(ok, ids, 0)])
        logprob = (np.where(ok, got[0], np.nan), got[1])
        h = np.where(empty, 0, ln + w / (1 + r))
        entropy = (h, 4 * DELTA * np.where(np.isfinite(h), h, 0) + 1e-36)
        order = np.lexsort((np.broadcast_to(np.arange(vocab), x.shape), -np.where(np.isnan(x64), -np.inf, x64), np.isnan(x64)), axis=1)[:, :top]
        tops = [lp(x64[np.arange(n), order[:, k]]) for k in range(top)]
    return logprob, entropy, order, tops


def run(dev, x, ids, top, gap=0, shift=0):
    n, vocab = x.shape
    full = np.full((n, vocab + gap), np.nan, np.float32)
    full[:, :vocab] = x
    flat = np.concatenate([np.full(shift, np.nan, np.float32), full.ravel()])
    xb = dev.upload(flat)
    at = type("Ref", (), {"ptr": xb.ptr + 4 * shift})
    ib = dev.upload(np.asarray(ids, np.int32))
    fill = np.full(n * max(top, 1) + 4, 7.5, np.float32)  # nothing is written behind the outputs
    lp, h, ti, tl = (dev.upload(fill) for _ in range(4))
    htr.token_logprobs(dev, at, n, vocab, ib, lp, h, top, ti if top else None, tl if top else None, stride=vocab + gap)
    out = [b.download(np.float32, fill.size) for b in (lp, h, ti, tl)]
    after = xb.download(np.float32, flat.size)
    assert np.array_equal(after.view(np.uint32), flat.view(np.uint32))  # the logits stay as they are
    for b in (xb, ib, lp, h, ti, tl):
        b.free()
    for a, k in zip(out, (n, n, n * top, n * top)):
        assert np.all(a[k:] == 7.5)
    return out[0][:n], out[1][:n], out[2].view(np.int32)[:n * top].reshape(n, top), out[3][:n * top].reshape(n, top)


def check(dev, x, ids, top, **kw):
    got = run(dev, x, ids, top, **kw)
    logprob, entropy, order, tops = reference(x, ids, top)
    np.testing.assert_array_equal(got[2], order)
    for g, (want, off) in [(got[0], logprob), (got[1], entropy)] + [(got[3][:, k], t) for k, t in enumerate(tops)]:
        special = ~np.isfinite(want)
        np.testing.assert_array_equal(g[special], want[special].astype(np.float32))
        assert np.all(np.abs(g[~special] - want[~special]) <= off[~special]), np.max(np.abs(g[~special] - want[~special]) / off[~special])
    again = run(dev, x, ids, top, **kw)
    for a, b in zip(got, again):
        np.testing.assert_array_equal(a.view(np.uint32), b.view(np.uint32))  # the same bits every time


def logits(seed, n, vocab, sure=True, std=2.5):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((n, vocab)) * std).astype(np.float32)
    at = rng.integers(vocab, size=n)
    if sure:
        x[np.arange(n), at] += (rng.random(n) * 40).astype(np.float32)
    return x, np.where(rng.random(n) < 0.7, at, rng.integers(vocab, size=n)).astype(np.int32)


@pytest.mark.parametrize("n,vocab,top", [(1, 1, 1), (3, 1, 0), (2, 2, 2), (5, 3, 3), (4, 33, 32), (9, 255, 5), (2, 256, 1), (7, 257, 20),
                                         (1, 1000, 32), (300, 1000, 5), (3, 4099, 7), (1, 8192, 32), (1, 151936, 5), (1, 151936, 0),
                                         (2, 151936, 32), (61, 20001, 20), (700, 5003, 1), (5, 151936, 1)])
def test_logprobs(dev, n, vocab, top):
    x, ids = logits(n + vocab, n, vocab)
    check(dev, x, ids, top)


@pytest.mark.parametrize("gap,shift", [(1, 0), (3, 1), (0, 2), (5, 3), (4, 0)])
@pytest.mark.parametrize("n,vocab", [(3, 1000), (2, 30011)])
def test_strides_and_alignment(dev, gap, shift, n, vocab):
    x, ids = logits(gap + 10 * shift, n, vocab)
    check(dev, x, ids, 5, gap=gap, shift=shift)


@pytest.mark.parametrize("vocab", [70, 4096, 151936])
def test_order_of_equal_and_sorted_logits(dev, vocab):
    """rows where all logits are equal, where few values repeat, rising and falling ones, ±0, the largest ones next to each
    other in memory or far apart by the width of a workgroup"""
    rng = np.random.default_rng(vocab)
    x = np.zeros((8, vocab), np.float32)
    x[0] = -3.25
    x[1] = rng.integers(4, size=vocab)
    x[2] = np.linspace(-9, 9, vocab)
    x[3] = np.linspace(9, -9, vocab)
    x[4] = np.where(rng.random(vocab) < 0.5, 0.0, -0.0)
    x[5] = rng.standard_normal(vocab)
    x[5, vocab // 2:vocab // 2 + 33] = 5 + np.arange(33) % 7
    x[6] = rng.standard_normal(vocab)
    x[6, 3::64] += 6
    x[7] = rng.standard_normal(vocab)
    x[7, 5::1024] += 8
    check(dev, x, np.arange(8) * (vocab // 9), 32)


@pytest.mark.parametrize("vocab", [40, 9000])
def test_values_that_are_not_finite(dev, vocab):
    x, ids = logits(vocab, 9, vocab)
    x[0] = -np.inf
    x[1, ::2] = -np.inf
    x[2] = -np.inf
    x[2, vocab - 1] = -4.0
    x[3, 17] = np.nan
    x[4, 5] = np.inf
    x[5] = np.nan
    x[6, :] = -np.inf
    x[6, 7] = np.nan
    x[7] = -3.4028235e38  # a mask of the type's lowest value
    x[7, 30:33] = (1.0, 2.0, 1.0)
    x[8, 20] = x[8, 21] = np.inf
    ids[2], ids[7], ids[4] = vocab - 1, 30, 5
    check(dev, x, ids, 32)
    ids[:] = (0, -1, vocab, 2 ** 31 - 1, -2 ** 31, 3, 7, 0, 20)
    check(dev, x, ids, 3)


def test_sure_and_wide_rows(dev):
    """a choice of probability 1 − 10^-13 … and logits from the smallest to the largest: the leading digits stay"""
    vocab = 3000
    x = np.random.default_rng(1).standard_normal((6, vocab)).astype(np.float32)
    x[:5] += np.float32(0)
    for i, up in enumerate((8, 16, 30, 60, 86)):
        x[i, 100 * i] = up
    x[5] *= np.float32(1e30)
    check(dev, x, np.arange(6) * 100, 4)


def test_replayed_with_other_rows(dev):
    """one recorded call over buffers that change, beside another of another shape that shares the device's scratch"""
    a, b = logits(1, 3, 40000), logits(2, 1, 151936)
    bufs = [[dev.upload(x), dev.upload(i), *(dev.alloc(4 * x.shape[0] * k) for k in (1, 1, 5, 5))] for x, i in (a, b)]

    def call(s, x):
        htr.token_logprobs(dev, s[0], x.shape[0], x.shape[1], s[1], s[2], s[3], 5, s[4], s[5])

    graphs = []
    for s, (x, _) in zip(bufs, (a, b)):
        call(s, x)
        dev.capture_begin()
        call(s, x)
        graphs.append(dev.capture_end())
    for seed in range(3):
        new = [logits(10 + seed, *a[0].shape), logits(20 + seed, *b[0].shape)]
        for s, (x, i) in zip(bufs, new):
            s[0].upload(x), s[1].upload(i)
        for g in graphs:
            g.launch()
        for s, (x, i) in zip(bufs, new):
            want = run(dev, x, i, 5)  # eager, between the replays
            n = x.shape[0]
            for buf, w in zip(s[2:], want):
                np.testing.assert_array_equal(buf.download(np.uint32, w.size), w.view(np.uint32).ravel())
        for g in graphs[::-1]:
            g.launch()
        dev.sync()
    for g in graphs:
        g.free()
    for s in bufs:
        for x in s:
            x.free()


@pytest.mark.parametrize("n,vocab,top", [(1200, 20001, 32), (700, 20001, 32), (500, 30011, 20), (330, 45011, 5), (330, 45011, 32),
                                         (1200, 4096, 32), (600, 4090, 32)])
def test_several_chunks_to_a_workgroup(dev, n, vocab, top):
    """so many rows that a workgroup takes several chunks of one (on 256 CUs three, two of a row in two parts, …): rising and falling
    logits, equal ones, few values, ±0, random ones with a NaN or an infinity in a later chunk. Rows of a kind are alike"""
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((11, vocab)).astype(np.float32)
    x[0] = -3.25
    x[1] = rng.integers(4, size=vocab)
    x[2] = np.linspace(-9, 9, vocab)
    x[3] = np.linspace(9, -9, vocab)
    x[4] = np.where(rng.random(vocab) < 0.5, 0.0, -0.0)
    x[5, -40:] += 9
    x[6, ::3] = -np.inf
    x[7, vocab - 5] = np.nan
    x[8] = -np.inf
    x[8, vocab - 2] = 1.0
    x[9, vocab - 9] = np.inf
    ids = np.array([0, 5, vocab - 1, 0, 7, vocab - 3, 1, 4, vocab - 2, 3, 70], np.int32)
    kind = np.arange(n) % 11
    got = run(dev, x[kind], ids[kind], top)
    logprob, entropy, order, tops = reference(x, ids, top)
    np.testing.assert_array_equal(got[2], order[kind])
    for g, (want, off) in [(got[0], logprob), (got[1], entropy)] + [(got[3][:, k], t) for k, t in enumerate(tops)]:
        special = ~np.isfinite(want)[kind]
        np.testing.assert_array_equal(g[special], want[kind][special].astype(np.float32))
        assert np.all(np.abs(g[~special] - want[kind][~special]) <= off[kind][~special])


def upload_at(dev, ptr, a):
    a = np.ascontiguousarray(a)
    htr._check(htr.lib().htr_upload(dev.h, ptr, a.ctypes.data, a.nbytes))


def test_rows_past_32_bits(dev):
    """rows 2^31 + 5 logits apart: the third lies 17 GB behind the first"""
    vocab, stride, top = 9001, 2 ** 31 + 5, 6
    x, ids = logits(3, 3, vocab)
    xb = dev.alloc(4 * (2 * stride + vocab))
    for i in range(3):
        upload_at(dev, xb.ptr + 4 * stride * i, x[i])
    ib, lp, h = dev.upload(ids), dev.alloc(12), dev.alloc(12)
    ti, tl = dev.alloc(12 * top), dev.alloc(12 * top)
    htr.token_logprobs(dev, xb, 3, vocab, ib, lp, h, top, ti, tl, stride=stride)
    want = run(dev, x, ids, top)
    # (another alignment of the rows: the sums' order and so their last bits differ)
    logprob, entropy, order, tops = reference(x, ids, top)
    np.testing.assert_array_equal(ti.download(np.int32, 3 * top).reshape(3, top), order)
    for g, (w, off) in ((lp.download(np.float32, 3), logprob), (h.download(np.float32, 3), entropy)):
        assert np.all(np.abs(g - w) <= off)
    np.testing.assert_array_equal(want[2], order)
    for b in (xb, ib, lp, h, ti, tl):
        b.free()


def test_the_largest_vocabulary(dev):
    """2^28 logits of a row, all -10 but four. Of 64 parts' 256 threads each sums 2^14 equal terms one after another, each sum off by
    2^-24 of it at most: 2^-10 of r and W, beside DELTA"""
    vocab, top = 2 ** 28, 5
    x = np.full(vocab, -10.0, np.float32)
    at = {5: 1.0, vocab - 1: 2.0, 2 ** 27 + 3: 1.0, vocab - 8192: 1.5}
    for i, v in at.items():
        x[i] = v
    xb, ib = dev.upload(x), dev.upload(np.array([vocab - 8192], np.int32))
    lp, h, ti, tl = dev.alloc(4), dev.alloc(4), dev.alloc(4 * top), dev.alloc(4 * top)
    htr.token_logprobs(dev, xb, 1, vocab, ib, lp, h, top, ti, tl)
    e = [np.exp(v - 2.0) for v in (1.0, 1.0, 1.5)]
    r = (vocab - 4) * np.exp(-12.0) + sum(e)
    w = (vocab - 4) * np.exp(-12.0) * 12 + e[0] + e[1] + 0.5 * e[2]
    off = 2.0 ** -10 + DELTA
    assert ti.download(np.int32, top).tolist() == [vocab - 1, vocab - 8192, 5, 2 ** 27 + 3, 0]
    assert abs(lp.download(np.float32, 1)[0] - (-0.5 - np.log1p(r))) <= off
    assert np.all(np.abs(tl.download(np.float32, top) - (np.array([0, -0.5, -1, -1, -12]) - np.log1p(r))) <= off)
    assert abs(h.download(np.float32, 1)[0] - (np.log1p(r) + w / (1 + r))) <= off * (1 + 2 * w / (1 + r))
    for b in (xb, ib, lp, h, ti, tl):
        b.free()
