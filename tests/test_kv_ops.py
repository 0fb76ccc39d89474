"""The operators on a layer's KV cache without a GPU: the tree's masks and depths, and the refusals, which the entry points
give before they look at the device (a null one here, so that nothing can be launched)."""
import ctypes as C
import re

import numpy as np
import pytest

import htr


def test_tree_masks():
    #        0   1  2  3  4  5
    t = htr.Tree([-1, 0, 0, 1, -1, 3])
    assert t.masks.tolist() == [0b1, 0b11, 0b101, 0b1011, 0b10000, 0b101011]
    assert t.depths.tolist() == [0, 1, 1, 2, 0, 3]
    chain = htr.Tree(np.arange(64) - 1)
    assert int(chain.masks[63]) == 2 ** 64 - 1 and chain.depths.tolist() == list(range(64))
    u = htr.Tree.of_masks([3, 0], [0, 5])
    assert u.n == 2 and u.masks.tolist() == [3, 0] and u.depths.tolist() == [0, 5]


@pytest.mark.parametrize("parents,match", [([0], "node 0 has parent 0"), ([-1, 2, 0], "node 1 has parent 2"),
                                           ([-2], "parent -2"), ([], "0 nodes"), ([-1] * 65, "65 nodes")])
def test_tree_masks_refuse(parents, match):
    with pytest.raises(htr.HtrError, match=match):
        htr.Tree(parents)
    with pytest.raises(ValueError, match="2 depths for 1 masks"):
        htr.Tree.of_masks([1], [0, 1])


def _kv(type=1, n_kv=2, n_ctx=100, k=1 << 20, v=2 << 20, kd=0, vd=0):
    return htr.KvC(type, n_kv, n_ctx, k, v, kd, vd)


Q8 = dict(type=8, kd=3 << 20, vd=4 << 20)
BAD_CACHES = [(dict(type=0), "type 0"), (dict(n_kv=0), "0 KV heads"), (dict(n_kv=4097, n_ctx=1), "4097 KV heads"),
              (dict(n_ctx=0), "0 rows"), (dict(k=0), "null cache rows"), (dict(v=(1 << 20) + 8), "16-byte"),
              (dict(type=8), "without scales"), (dict(Q8, vd=(4 << 20) + 4), "8-byte")]


def _calls(kv):
    """each entry point with good arguments but a null device, as functions of the arguments that are changed"""
    L, ref = htr.lib(), None if kv is None else C.byref(kv)  # (byref keeps the struct alive)
    M = 16 << 20  # addresses that no call follows

    def post(q=M, qs=512, k=2 * M, v=3 * M, ks=256, n=3, qn=4 * M, kn=5 * M, rope=6 * M, n_pos=200, pos0=7, depth=None,
             n_head=4, row0=97, out=7 * M):
        d = None if depth is None else np.array(depth, np.int32).ctypes.data_as(C.c_void_p)
        return L.htr_qkv_post_rows(None, q, qs, k, v, ks, n, qn, kn, rope, n_pos, pos0, d, n_head, 1e-6, ref, row0, out)

    def copy(src_row=0, dst=None, dst_row=0, n=5):
        other = dst if dst is not None else _kv(type=8, k=5 << 20, v=6 << 20, kd=7 << 20, vd=8 << 20)
        return L.htr_kv_copy(None, ref, src_row, C.addressof(other), dst_row, n)

    def keep(row0=90, idx=(0, 3, 9), n=None):
        i = np.array(idx, np.int32)
        return L.htr_kv_keep(None, ref, row0, i.ctypes.data_as(C.c_void_p), len(idx) if n is None else n)

    def tree(q=M, qs=512, n=3, mask=None, past=97, n_head=4, out=2 * M):
        m = None if mask is None else np.array(mask, np.uint64).ctypes.data_as(C.c_void_p)
        return L.htr_tree_attention(None, q, qs, n, m, past, ref, n_head, 0.1, out)

    def window(q=M, qs=512, n=3, pos0=97, w=16, sink=4, n_head=4, out=2 * M):
        return L.htr_window_attention(None, q, qs, n, pos0, w, sink, ref, n_head, 0.1, out)

    return dict(post=post, copy=copy, keep=keep, tree=tree, window=window)


def _refused(rc, match):
    assert rc == -1 and match in htr.last_error(), htr.last_error()


@pytest.mark.parametrize("name", ["post", "copy", "keep", "tree", "window"])
def test_good_arguments_reach_the_device_and_bad_caches_do_not(name):
    for kv in (_kv(), _kv(**Q8)):
        other = {"dst": _kv(k=5 << 20, v=6 << 20)} if name == "copy" else {}
        _refused(_calls(kv)[name](**other), "null device")
    _refused(_calls(None)[name](), "null cache")
    for change, match in BAD_CACHES:
        _refused(_calls(_kv(**change))[name](), match)


@pytest.mark.parametrize("name,change,match", [
    ("post", dict(q=0), "null argument"), ("post", dict(out=0), "null argument"), ("post", dict(rope=0), "null argument"),
    ("post", dict(n_head=3), "3 q heads on 2"), ("post", dict(n_head=0), "0 q heads"),
    ("post", dict(qs=508), "508"), ("post", dict(ks=252), "252"), ("post", dict(qs=514), "multiples of 4"),
    ("post", dict(k=(32 << 20) + 8), "16-byte"), ("post", dict(n=0), "0 rows"), ("post", dict(row0=98), "3 rows from row 98"),
    ("post", dict(row0=-1), "row -1"), ("post", dict(pos0=198), "positions 198 … 200"), ("post", dict(pos0=-1), "positions -1"),
    ("post", dict(depth=[0, 64, 1]), "depth 64"), ("post", dict(depth=[0, -1, 1]), "depth -1"),
    ("post", dict(depth=[0, 63, 1], pos0=137), "positions 137 … 200"), ("post", dict(n_pos=0), "0-position"),
    ("post", dict(n=65, row0=0, depth=[0] * 65), "65 drafted rows"),
    ("post", dict(qs=516, out=16 << 20), "overlaps"), ("post", dict(out=(16 << 20) + 1024), "overlaps"),
    ("post", dict(out=32 << 20), "overlaps"), ("post", dict(out=1 << 20), "overlap the cache"),
    ("post", dict(v=(2 << 20) - 256), "overlap the cache"),
    ("post", dict(out=(64 << 20) + 256), "overlaps the norms"), ("post", dict(qn=(112 << 20) + 4096), "overlaps the norms"),
    ("post", dict(out=(96 << 20) + 64 * 1024), "overlaps the norms"), ("post", dict(rope=(1 << 20) - 512), "overlaps the norms"),
    ("copy", dict(src_row=96), "from row 96"), ("copy", dict(dst_row=-1), "row -1"), ("copy", dict(n=-1), "-1 rows"),
    ("copy", dict(dst=_kv(n_kv=1, k=5 << 20, v=6 << 20)), "2 KV heads into 1"), ("copy", dict(dst=_kv(), dst_row=4), "overlap"),
    ("copy", dict(dst=_kv(k=(1 << 20) + 256, v=6 << 20), dst_row=50), "overlap"),
    ("copy", dict(dst=_kv(k=2 << 20, v=1 << 20), dst_row=50), "overlap"),
    ("copy", dict(dst=_kv(**dict(Q8, k=5 << 20, v=6 << 20, vd=1 << 20)), dst_row=50), "overlap"),
    ("keep", dict(n=65, idx=[0] * 65), "65 rows"), ("keep", dict(n=-1), "-1 rows"), ("keep", dict(idx=[10]), "row 90 + 10"),
    ("keep", dict(idx=[-1]), "90 + -1"), ("keep", dict(row0=98), "3 rows from row 98"), ("keep", dict(row0=-1), "row -1"),
    ("tree", dict(q=0), "null argument"), ("tree", dict(n=0), "0 nodes"), ("tree", dict(n=65, past=0), "65 nodes"),
    ("tree", dict(past=98), "98 keys"), ("tree", dict(past=-1), "-1 keys"), ("tree", dict(n_head=5), "5 q heads"),
    ("tree", dict(qs=500), "500 floats"), ("tree", dict(qs=513), "513 floats"), ("tree", dict(out=(32 << 20) + 4), "16-byte"),
    ("tree", dict(mask=[1, 2, 8]), "node 2's mask 0x8"), ("tree", dict(out=(16 << 20) + 4096), "overlaps"),
    ("window", dict(out=0), "null argument"), ("window", dict(n=0), "0 queries"), ("window", dict(pos0=98), "position 98"),
    ("window", dict(pos0=-1), "position -1"), ("window", dict(w=0), "window of 0"), ("window", dict(sink=-1), "-1 first"),
    ("tree", dict(out=(2 << 20) + 64), "overlaps the cache"), ("window", dict(out=(1 << 20) - 2048), "overlaps the cache"),
    ("window", dict(n_head=-2), "-2 q heads"), ("window", dict(qs=0), "0 floats"), ("window", dict(out=16 << 20), "overlaps"),
])
def test_refusals(name, change, match):
    _refused(_calls(_kv())[name](**change), match)


@pytest.mark.parametrize("change", [dict(v=1 << 20), dict(v=(1 << 20) + 2 * 100 * 256 - 16), dict(Q8, vd=3 << 20),
                                    dict(Q8, kd=(2 << 20) + 128)])
def test_a_cache_that_is_written_to_has_planes_apart(change):
    kv = _kv(**change)
    for name in ("post", "keep"):
        _refused(_calls(kv)[name](), "planes overlap")
    _refused(_calls(_kv(k=32 << 20, v=33 << 20))["copy"](dst=kv), "planes overlap")
    for name in ("tree", "window"):
        _refused(_calls(kv)[name](), "null device")  # read only


def test_kv_keep_takes_any_integers_and_no_others():
    class Dev:
        h = None

    class B:
        ptr = 1 << 20

    class V:
        ptr = 2 << 20

    kv = htr.KvCache.of(2, 100, B, V)
    for rows in ([], [0, 3], (1,), range(4), np.array([2, 1]), np.array([5], np.int32)):
        with pytest.raises(htr.HtrError, match="null device"):
            htr.kv_keep(Dev, kv, 90, rows)
    with pytest.raises(OverflowError):
        htr.kv_keep(Dev, kv, 90, [1 << 32])
    with pytest.raises(TypeError):
        htr.kv_keep(Dev, kv, 90, [0.5])


def test_copy_between_rows_of_one_cache_and_in_place_rows_are_allowed():
    _refused(_calls(_kv())["copy"](dst=_kv(), dst_row=5), "null device")
    _refused(_calls(_kv(**Q8))["copy"](dst=_kv(**Q8), src_row=50, dst_row=45), "null device")
    _refused(_calls(_kv())["post"](out=16 << 20), "null device")
    _refused(_calls(_kv())["keep"](idx=[]), "null device")
    _refused(_calls(_kv())["window"](w=2 ** 31 - 1, sink=2 ** 31 - 1), "null device")


def test_cache_object_takes_scales_of_both():
    class B:
        ptr = 16

    with pytest.raises(ValueError, match="scales of both"):
        htr.KvCache.of(1, 1, B, B, B)


def test_no_lds_access_in_flight_at_a_barrier(tmp_path):
    """the attention's kernels fill LDS by loads that the compiler does not know and wait for their reads themselves: at each
    of their barriers, over all paths, no LDS access of the wave is in flight; and the loops that wait for a number of loads
    have no memory accesses but those loads, so that the number is theirs alone"""
    from test_kernel_waits import _assembly, _functions, _pending_at_barriers

    seen = 0
    for name, body in _functions(_assembly("kv_attention", tmp_path)):
        if "k_kv_attn" not in name or "join" in name:
            continue
        at = _pending_at_barriers(body)
        seen += len(at)
        assert not any(at.values()), (name, sorted(at.items()))
        if not re.search("attn_few|attn_split", name):
            continue  # waits for all of them
        last = max(i for i, s in enumerate(body) if "_load_lds_" in s)
        first = min(i for i, s in enumerate(body) if "v_mfma" in s)
        between = [s for s in body[first:last] if s.startswith(("global_", "buffer_", "flat_", "scratch_"))]
        assert between and all("_load_lds_" in s for s in between), (name, [s for s in between if "_load_lds_" not in s])
    assert seen >= 40


class _Memory:
    """stands in for a device's buffers: an address that no call follows"""
    made = []

    def __init__(self, dev, nbytes, kind):
        if len(self.made) == dev.room:
            raise htr.HtrError("no room")
        self.ptr = (len(self.made) + 1) << 20
        self.made.append(self)

    def free(self):
        self.ptr = None


class _NoDevice:
    h, room = None, 4


def test_a_cache_that_was_freed_is_refused(monkeypatch):
    """its addresses go with its memory: a call on it must not reach what another allocation has there by then"""
    monkeypatch.setattr(htr, "Buffer", _Memory)
    monkeypatch.setattr(_Memory, "made", [])
    out = _Memory(_NoDevice, 0, 0)
    for q8_0 in (False, True):
        _Memory.made.clear()
        kv = htr.KvCache(_NoDevice, 2, 50, q8_0)
        calls = [lambda: htr.kv_keep(_NoDevice, kv, 0, [1]), lambda: htr.kv_copy(_NoDevice, kv, 0, kv, 9, 1),
                 lambda: htr.tree_attention(_NoDevice, out, 1, 5, kv, 2, 1.0, type("B", (), {"ptr": 16 << 20})),
                 lambda: htr.window_attention(_NoDevice, out, 1, 5, 3, 0, kv, 2, 1.0, type("B", (), {"ptr": 16 << 20}))]
        for call in calls:
            with pytest.raises(htr.HtrError, match="null device"):
                call()
        kv.free()
        for call in calls:
            with pytest.raises(htr.HtrError, match="null cache rows"):
                call()
        kv.free()
    lent = htr.KvCache.of(2, 50, out, type("B", (), {"ptr": 9 << 20}))
    lent.free()  # the caller's buffers: nothing to free
    with pytest.raises(htr.HtrError, match="null device"):
        htr.kv_keep(_NoDevice, lent, 0, [1])


def test_a_cache_without_room_for_all_planes_frees_those_it_had(monkeypatch):
    monkeypatch.setattr(htr, "Buffer", _Memory)
    monkeypatch.setattr(_Memory, "made", [])
    with pytest.raises(htr.HtrError, match="no room"):
        htr.KvCache(type("D", (), {"h": None, "room": 3}), 2, 50, True)
    assert len(_Memory.made) == 3 and all(b.ptr is None for b in _Memory.made)


@pytest.mark.parametrize("n_kv,n_ctx", [(0, 5), (-1, 5), (4097, 5), (2, 0), (2, -3), (2, 2 ** 31)])
def test_a_cache_of_sizes_that_no_call_takes_asks_for_no_memory(monkeypatch, n_kv, n_ctx):
    """(a negative size would be asked for as nearly 2^64 bytes, which leaves the device dead; one past 32 bits would reach
    the library as another)"""
    monkeypatch.setattr(htr, "Buffer", _Memory)
    monkeypatch.setattr(_Memory, "made", [])
    with pytest.raises(ValueError, match="KV heads"):
        htr.KvCache(_NoDevice, n_kv, n_ctx)
    assert not _Memory.made
    with pytest.raises(ValueError, match="KV heads"):
        htr.KvCache.of(n_kv, n_ctx, type("B", (), {"ptr": 1 << 20}), type("B", (), {"ptr": 2 << 20}))


def test_more_rows_than_a_launch_takes_are_refused():
    """a grid's first dimension holds less than 2^32 threads: a launch of more fails and leaves the device dead, so that such a
    call is refused before, and the largest below is not"""
    T = 1 << 40
    big = dict(n_kv=4, n_ctx=2 ** 24, k=T, v=2 * T)
    post = dict(q=3 * T, k=4 * T, v=5 * T, n_head=8, qs=1024, ks=512, row0=0, pos0=0, n_pos=2 ** 25, out=6 * T)  # 16 heads a row
    _refused(_calls(_kv(**big))["post"](n=2 ** 24, **post), "16777216 rows of 8 + 8 heads in one call")
    _refused(_calls(_kv(**big))["post"](n=2 ** 24 - 1, **post), "null device")
    long = [_kv(n_kv=1, n_ctx=2 ** 30, k=i * T, v=(i + 1) * T) for i in (1, 3)]
    _refused(_calls(long[0])["copy"](dst=long[1], n=2 ** 29), "536870912 rows in one call")
    _refused(_calls(long[0])["copy"](dst=long[1], n=2 ** 29 - 32), "null device")
    wide = _kv(n_kv=2, n_ctx=2 ** 28, k=T, v=2 * T)
    _refused(_calls(wide)["window"](q=3 * T, out=4 * T, n=2 ** 28, pos0=0), "268435456 queries of 4 heads")
    _refused(_calls(wide)["window"](q=3 * T, out=4 * T, n=2 ** 28 - 32, pos0=0), "null device")


@pytest.mark.parametrize("stride", [2 ** 64 - 4, 2 ** 62, 2 ** 61 + 512, 2 ** 60])
def test_rows_that_end_past_any_memory_are_refused(stride):
    """of a stride below 0, taken as 64 bits without a sign, or of any other whose rows lie past 2^62 bytes, the check of overlaps
    would count a few bytes, and the kernels would read in front of the rows"""
    for kv in (_kv(), _kv(**Q8)):
        calls = _calls(kv)
        for name, change in (("post", dict(qs=stride)), ("post", dict(ks=stride)), ("tree", dict(qs=stride)), ("window", dict(qs=stride))):
            _refused(calls[name](**change), "floats apart")
            _refused(calls[name](**change, n=1), "null device")  # (one row: no stride)
        for name in ("post", "tree", "window"):
            _refused(calls[name](q=1 << 58, qs=2 ** 40), "null device")
