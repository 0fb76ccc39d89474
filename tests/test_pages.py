"""The operators of a step over a cache in pages and the log probabilities without a GPU: the refusals, which the entry points
give before they look at the device (a null one here, so that nothing can be launched)."""
import ctypes as C
import re

import pytest

import htr

M = 16 << 20  # addresses that no call follows, far apart
Q8 = dict(type=8, kd=3 << 20, vd=4 << 20)


def kv(type=1, n_kv=2, n_ctx=640, k=1 << 20, v=2 << 20, kd=0, vd=0):
    return htr.KvC(type, n_kv, n_ctx, k, v, kd, vd)


def pages(n_seq=3, n_row=10, page=16, max_pages=5, start=20 * M, past=21 * M, table=22 * M, pos=23 * M, slot=24 * M):
    return htr.PagesC(n_seq, n_row, page, max_pages, start, past, table, pos, slot)


BAD_PAGES = [(dict(n_seq=0), "0 reads"), (dict(n_seq=1025), "1025 reads"), (dict(n_row=0), "of 0 rows"),
             (dict(n_row=2 ** 21 + 1), "2097153 rows"), (dict(page=8), "pages of 8 rows"), (dict(page=48), "pages of 48 rows"),
             (dict(page=2048), "pages of 2048"), (dict(page=0), "pages of 0"), (dict(max_pages=0), "table of 0 pages"),
             (dict(max_pages=2 ** 27), "table of 134217728 pages"), (dict(n_seq=1000, max_pages=2 ** 22), "table of 4194304 pages")]
TABLES = [(dict(start=0), "null start"), (dict(past=0), "null start"), (dict(table=0), "null start"),
          (dict(start=20 * M + 2), "4-byte aligned"), (dict(table=22 * M + 1), "4-byte aligned")]
ROWS = [(dict(pos=0), "null positions"), (dict(slot=0), "null positions"), (dict(slot=24 * M + 3), "4-byte aligned")]


def page_map(p=None, n_page=40, length=M, new=2 * M, ring=3 * M, pool=4 * M, length_out=5 * M, pool_out=6 * M):
    p = pages() if p is None else p
    return htr.lib().htr_page_map(None, C.addressof(p) if p else None, n_page, length, new, ring, pool, length_out, pool_out)


def post(p=None, c=None, q=M, qs=512, k=2 * M, v=3 * M, ks=256, qn=4 * M, kn=5 * M, rope=6 * M, n_pos=200, n_head=4, out=7 * M):
    p, c = pages() if p is None else p, kv() if c is None else c
    return htr.lib().htr_qkv_post_pages(None, q, qs, k, v, ks, C.addressof(p) if p else None, qn, kn, rope, n_pos, n_head, 1e-6,
                                        C.addressof(c), out)


def attend(p=None, c=None, q=M, qs=512, n_head=4, out=2 * M):
    p, c = pages() if p is None else p, kv() if c is None else c
    return htr.lib().htr_page_attention(None, q, qs, C.addressof(p) if p else None, C.addressof(c), n_head, 0.1, out)


def score(x=M, stride=1000, n=3, vocab=1000, ids=2 * M, lp=3 * M, h=4 * M, top=5, top_ids=5 * M, top_lp=6 * M):
    return htr.lib().htr_token_logprobs(None, x, stride, n, vocab, ids, lp, h, top, top_ids, top_lp)


def refused(rc, match):
    assert rc < 0 and re.search(match, htr.last_error()), htr.last_error()


def test_good_arguments_reach_the_device():
    for call in (page_map, post, attend, score):
        refused(call(), "null device")
    for c in (kv(), kv(**Q8)):
        refused(attend(c=c), "null device")
        refused(post(c=c), "null device")
    refused(page_map(length_out=M, pool_out=4 * M), "null device")  # in place
    refused(post(q=M, out=M), "null device")
    refused(attend(p=pages(pos=0, slot=0)), "null device")  # each call wants the arrays that it uses
    refused(post(p=pages(start=0, past=0, table=0)), "null device")
    refused(score(top=0, top_ids=0, top_lp=0), "null device")
    refused(score(x=M + 4, lp=3 * M + 4), "null device")
    for page in (16, 32, 1024):
        refused(attend(p=pages(page=page), c=kv(n_ctx=1024)), "null device")


@pytest.mark.parametrize("change,match", BAD_PAGES)
def test_sizes_of_pages(change, match):
    for call in (page_map, post, attend):
        refused(call(pages(**change)), match)


def test_null_pages():
    for call in (page_map, post, attend):
        refused(call(p=False), "null pages")


@pytest.mark.parametrize("change,match", TABLES)
def test_tables(change, match):
    refused(page_map(pages(**change)), match)
    refused(attend(pages(**change)), match)


@pytest.mark.parametrize("change,match", ROWS)
def test_rows(change, match):
    refused(page_map(pages(**change)), match)
    refused(post(pages(**change)), match)


@pytest.mark.parametrize("change,match", [
    (dict(length=0), "null argument"), (dict(pool_out=0), "null argument"), (dict(ring=0), "null argument"),
    (dict(n_page=0), "0 pages"), (dict(n_page=2 ** 27), "at most 2"), (dict(new=2 * M + 2), "4-byte aligned"),
    (dict(length_out=M + 4), "overlap"), (dict(length_out=2 * M), "overlap"), (dict(ring=22 * M), "overlap"),
    (dict(pool_out=4 * M + 4), "overlap"), (dict(pool=M, pool_out=M), "overlap"), (dict(length=21 * M), "overlap"),
    (dict(new=23 * M + 36), "overlap"), (dict(ring=24 * M - 156), "overlap"), (dict(pool=20 * M + 12), "overlap")])
def test_map(change, match):
    refused(page_map(**change), match)


@pytest.mark.parametrize("change,match", [
    (dict(q=0), "null argument"), (dict(rope=0), "null argument"), (dict(n_head=3), "3 q heads on 2"), (dict(n_head=0), "0 q heads"),
    (dict(qs=511), "511 and 256 floats"), (dict(ks=252), "512 and 252"), (dict(v=3 * M + 4), "16-byte"), (dict(n_pos=0), "0 positions"),
    (dict(out=M + 16), "overlaps the input rows"), (dict(q=M, qs=516, out=M), "overlaps the input rows"),
    (dict(out=2 * M), "overlaps the input rows"), (dict(out=1 << 20), "overlap the cache"), (dict(k=2 << 20), "overlap the cache"),
    (dict(rope=7 * M), "rows' places"), (dict(out=23 * M), "rows' places"), (dict(c=kv(type=0)), "type 0"),
    (dict(c=kv(v=(1 << 20) + 4096)), "planes overlap"), (dict(p=pages(slot=1 << 20)), "rows' places")])
def test_post(change, match):
    refused(post(**change), match)


def test_post_of_more_rows_than_a_launch_takes():
    refused(post(p=pages(n_row=2 ** 21), c=kv(n_kv=64, n_ctx=1, k=1 << 44, v=1 << 45), n_head=64, qs=64 * 128, ks=64 * 128,
                 q=1 << 46, k=1 << 47, v=1 << 48, out=1 << 49), "heads' rows")


@pytest.mark.parametrize("change,match", [
    (dict(q=0), "null argument"), (dict(out=0), "null argument"), (dict(n_head=5), "5 q heads on 2"), (dict(qs=508), "508 floats"),
    (dict(qs=514), "514 floats"), (dict(out=2 * M + 8), "16-byte"), (dict(out=M + 1024), "overlaps the queries"),
    (dict(out=2 << 20), "overlaps the cache"), (dict(out=22 * M), "overlaps the pages"), (dict(c=kv(n_ctx=15)), "15 rows in pages of 16"),
    (dict(c=kv(n_kv=0)), "0 KV heads"), (dict(c=kv(type=8)), "without scales")])
def test_attention(change, match):
    refused(attend(**change), match)


@pytest.mark.parametrize("change,match", [
    (dict(x=0), "null argument"), (dict(ids=0), "null argument"), (dict(lp=0), "null argument"), (dict(h=0), "null argument"),
    (dict(n=0), "0 rows"), (dict(n=2 ** 21 + 1), "2097153 rows"), (dict(vocab=0), "of 0 logits"), (dict(stride=999), "999 apart"),
    (dict(vocab=2 ** 28 + 1, stride=2 ** 28 + 1), "268435457 logits"), (dict(top=-1), "-1 alternatives"), (dict(top=33), "33 alternatives"),
    (dict(top=4, vocab=3), "4 alternatives of 3"), (dict(top_ids=0), "null alternatives"), (dict(top_lp=0), "null alternatives"),
    (dict(lp=3 * M + 2), "4-byte"), (dict(x=M + 1), "4-byte"), (dict(lp=4 * M + 8), "overlaps another"), (dict(top_lp=5 * M + 56), "overlaps another"),
    (dict(h=M + 4 * 2999), "overlaps another"), (dict(top_ids=2 * M + 8), "overlaps another")])
def test_logprobs(change, match):
    refused(score(**change), match)


@pytest.mark.parametrize("n_row,n_head,n_seq,page,max_pages,match", [
    (2 ** 21, 46, 1, 16, 5, "2097152 rows of 46 heads"), (2 ** 16, 256, 1, 16, 5, "65536 rows of 256 heads"),
    (2 ** 21, 16, 1024, 1024, 2 ** 21 - 1, "1024 reads of 2097152 rows of 16 heads over up to 2147482624 rows")])
def test_attention_of_more_than_is_counted(n_row, n_head, n_seq, page, max_pages, match):
    p = pages(n_seq, n_row, page, max_pages, start=1 << 50, past=1 << 51, table=1 << 52)
    refused(attend(p=p, c=kv(n_kv=1, n_ctx=2048), q=1 << 46, qs=n_head * 128, n_head=n_head, out=1 << 48), match)


def test_python_sizes():
    class Ref:
        ptr = M

    with pytest.raises(ValueError, match="pages of sizes"):
        htr.Pages.of(1, 0, 16, 1, Ref, Ref, Ref)
    with pytest.raises(ValueError, match="pages of sizes"):
        htr.Pages.of(2 ** 31, 1, 16, 1, Ref, Ref, Ref)


@pytest.mark.parametrize("stride", [2 ** 64 - 4, 2 ** 62, 2 ** 61 + 512, 2 ** 60])
def test_rows_that_end_past_any_memory(stride):
    """of a stride below 0, taken as 64 bits without a sign, or of any other whose rows lie past 2^62 bytes, the check of overlaps
    would count a few bytes, and the kernels would read in front of the rows"""
    refused(post(qs=stride), "floats apart")
    refused(post(ks=stride), "floats apart")
    refused(attend(qs=stride), "floats apart")
    refused(score(stride=stride), "apart")
    refused(score(stride=stride, n=2), "apart")
    refused(score(stride=stride, n=1), "null device")  # (one row: no stride)


def test_strides_of_rows_that_memory_could_hold():
    refused(post(q=1 << 58, qs=2 ** 40), "null device")
    refused(post(k=1 << 58, v=1 << 59, ks=2 ** 40), "null device")
    refused(attend(q=1 << 58, qs=2 ** 40), "null device")
    refused(score(x=1 << 58, stride=2 ** 40 + 1), "null device")


class Memory:
    """stands in for a device's buffers"""
    made = []

    def __init__(self, dev, nbytes):
        self.ptr = (len(self.made) + 1) << 40
        self.made.append(nbytes)

    def upload(self, a):
        return self

    def free(self):
        self.ptr = None


class NoDevice:
    h = None


@pytest.mark.parametrize("n_seq,n_row,page,max_pages", [
    (1025, 1, 16, 1), (0, 1, 16, 1), (-1, 1, 16, 1), (1, 2 ** 21 + 1, 16, 1), (1, -5, 16, 1), (1, 1, 8, 1), (1, 1, 48, 1), (1, 1, 2048, 1),
    (1, 1, 0, 1), (1, 1, -16, 1), (1, 1, 16, 0), (1, 1, 16, 2 ** 27), (1, 1, 16, -2), (1024, 1, 16, 2 ** 21), (2 ** 32 + 1, 1, 16, 1)])
def test_pages_of_sizes_that_no_call_takes_ask_for_no_memory(monkeypatch, n_seq, n_row, page, max_pages):
    """a table of 2^40 entries would be asked for before the first call refused it"""
    monkeypatch.setattr(htr, "Buffer", Memory)
    monkeypatch.setattr(Memory, "made", [])
    with pytest.raises(ValueError, match="pages of sizes"):
        htr.Pages(NoDevice, n_seq, n_row, page, max_pages)
    assert not Memory.made
    ref = type("Ref", (), {"ptr": M})
    with pytest.raises(ValueError, match="pages of sizes"):
        htr.Pages.of(n_seq, n_row, page, max_pages, ref, ref, ref)


@pytest.mark.parametrize("n_seq,n_row,page,max_pages", [(1, 1, 16, 1), (1024, 2 ** 21, 1024, 7), (15, 2 ** 21, 16, 2 ** 27 - 1),
                                                        (1, 1, 1024, 2 ** 21 - 1), (1024, 1, 16, 2 ** 21 - 1)])
def test_pages_of_the_largest_sizes(monkeypatch, n_seq, n_row, page, max_pages):
    """(what Pages takes the calls take: a null device is the next thing that is wrong)"""
    ref = type("Ref", (), {"ptr": M})
    at = [type("Ref", (), {"ptr": i << 50}) for i in range(1, 6)]
    p = htr.Pages.of(n_seq, n_row, page, max_pages, *at)
    with pytest.raises(htr.HtrError, match="null device"):
        htr.page_map(NoDevice, p, 1, ref, *[type("Ref", (), {"ptr": i << 56}) for i in range(1, 6)])


@pytest.mark.parametrize("more", [2 ** 32, -2 ** 32, 2 ** 63])
def test_sizes_past_32_bits_do_not_reach_the_library_as_others(more):
    """ctypes takes a size's low 32 bits (a stride's low 64): 2^32 + 3 rows would be answered as 3"""
    at = [type("Ref", (), {"ptr": M << i}) for i in range(12)]
    p, c = htr.Pages.of(3, 10, 16, 5, *at[7:12]), htr.KvCache.of(2, 640, at[5], at[6])
    d = NoDevice

    def page_map(n_page=40):
        htr.page_map(d, p, n_page, *at[:6])

    def post(n_pos=200, n_head=4, **strides):
        htr.qkv_post_pages(d, at[0], at[1], at[2], p, at[3], at[3], at[3], n_pos, n_head, 1e-6, c, at[4], **strides)

    def attend(n_head=4, **strides):
        htr.page_attention(d, at[0], p, c, n_head, 0.1, at[1], **strides)

    def score(n=3, n_vocab=1000, top=5, **strides):
        htr.token_logprobs(d, at[0], n, n_vocab, *at[1:4], top, *at[4:6], **strides)

    def rows(n=3, n_pos=200, pos0=7, n_head=4, row0=97, **strides):
        htr.qkv_post_rows(d, at[0], at[1], at[2], n, at[3], at[3], at[3], n_pos, pos0, n_head, 1e-6, c, row0, at[4], **strides)

    def copy(src_row=0, dst_row=90, n=5):
        htr.kv_copy(d, c, src_row, c, dst_row, n)

    def keep(row0=90):
        htr.kv_keep(d, c, row0, [0, 3])

    def tree(tree=3, n_past=97, n_head=4, **strides):
        htr.tree_attention(d, at[0], tree, n_past, c, n_head, 0.1, at[1], **strides)

    def window(n_q=3, pos0=97, window=16, n_sink=4, n_head=4, **strides):
        htr.window_attention(d, at[0], n_q, pos0, window, n_sink, c, n_head, 0.1, at[1], **strides)

    for call in (page_map, post, attend, score, rows, copy, keep, tree, window):
        with pytest.raises(htr.HtrError, match="null device"):
            call()
        for name, size in zip(call.__code__.co_varnames, call.__defaults__):
            with pytest.raises(ValueError, match="past 32 bits"):
                call(**{name: size + more})
    for call, strides in ((post, dict(q_stride=512, kv_stride=256)), (attend, dict(q_stride=512)), (score, dict(stride=1000)),
                          (rows, dict(q_stride=512, kv_stride=256)), (tree, dict(q_stride=512)), (window, dict(q_stride=512))):
        with pytest.raises(htr.HtrError, match="null device"):
            call(**strides)
        for name, stride in strides.items():
            for other in (stride + 2 ** 64, stride - 2 ** 64, -4):
                with pytest.raises(ValueError, match="floats apart"):
                    call(**{name: other})
