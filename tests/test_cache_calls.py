"""The paged cache's books and argument checks, on the CPU: calls beside those
of test_cache_host."""

from __future__ import annotations

import numpy as np
import pytest

import cache_ref as ref
from conftest import PKG
from test_cache_host import HostCache, _consistent

torch = pytest.importorskip("torch")
L = PKG._lib


def test_books_follow_rows_that_move_on_by_themselves():
    c = HostCache(n_pages=12)
    c.open(0, 130), c.open(1)
    c.step([0, 1], [126, 64])
    for _ in range(4):
        c.advance([0, 1])
    assert c.length(0) == 130 and c.length(1) == 68 and len(c.pages(1)) == 2
    _consistent(c)
    c.fork(0, [2])
    assert c.length(2) == 130 and c.pages(2)[:2] == c.pages(0)[:2] and c.pages(2)[2] != c.pages(0)[2]
    r = c.step([0, 1], [1, 1])
    assert r.pos0.tolist() == [130, 68]
    # pages that are shared become the slot's own before they are written; full ones stay shared
    c.calls.clear()
    c.release(2)
    shared = HostCache(n_pages=8, slots=[(0, [3], 10), (1, [3], 10)])
    shared._upload(0, 0), shared._upload(1, 0)
    shared.advance([1], 5)
    assert shared.calls == ["fmd_cache_copy_pages"] and shared.pages(0) == [3] and shared.pages(1) == [0]
    assert shared.length(1) == 15
    _consistent(c), _consistent(shared)
    for slots, n, status in (([0, 0], 1, L.FMD_EINVAL), ([3], 1, L.FMD_EINVAL), ([0], -1, L.FMD_EINVAL),
                             ([0], 400, L.FMD_EOVERFLOW)):
        with pytest.raises(PKG.FmdError) as e:
            c.advance(slots, n)
        assert e.value.status == status
    assert c.length(0) == 131
    _consistent(c)


def test_calls_without_rows_do_nothing():
    """An empty tensor's address is 0: calls that have no rows do not look at it."""
    import ctypes as C

    lib = PKG.load_library()
    cache = C.byref(L.Cache(4096, 4096, L.CACHE_BF16, 1, 4, 2, 128, 2, 4, 0))
    app = C.byref(L.CacheAppendArgs(k_row=256, k_head=128, v_row=256, v_head=128, dtype=L.DT_BF16))
    both = C.byref(L.CacheAppendArgs(k_row=256, k_head=128, v_row=256, v_head=128, q_row=512, q_head=128, q_out_row=512,
                                     q_out_head=128, dtype=L.DT_BF16, n_heads=4))
    att = C.byref(L.CacheAttendArgs(q_row=512, q_head=128, out_row=512, out_head=128, scale=0.1, dtype=L.DT_BF16,
                                    n_heads=4))
    for rows in (L.CacheRows(None, None, None, 0, 0, 0), L.CacheRows(4096, 4096, 4096, 3, 0, 0),
                 L.CacheRows(4096, 4096, 4096, 3, 0, 5)):
        r = C.byref(rows)
        assert lib.fmd_cache_append(cache, 0, r, app, None, None) == L.FMD_OK
        assert lib.fmd_cache_append(cache, 0, r, both, None, None) == L.FMD_OK
        assert lib.fmd_cache_read(cache, 0, r, None, None, None, None) == L.FMD_OK
        assert lib.fmd_cache_attend(cache, 0, r, att, None, 0, None, None) == L.FMD_OK
    # with rows they are looked at, and what does not depend on them is checked either way
    r, none = C.byref(L.CacheRows(4096, 4096, None, 1, 1, 1)), C.byref(L.CacheRows(4096, 4096, 4096, 3, 0, 0))
    assert lib.fmd_cache_append(cache, 0, r, app, None, None) == L.FMD_EINVAL
    assert lib.fmd_cache_read(cache, 0, r, None, None, None, None) == L.FMD_EINVAL
    assert lib.fmd_cache_attend(cache, 0, r, att, 4096, 1 << 40, None, None) == L.FMD_EINVAL
    assert lib.fmd_cache_append(cache, 1, none, app, None, None) == L.FMD_EINVAL
    assert lib.fmd_cache_attend(cache, 0, none, C.byref(L.CacheAttendArgs(dtype=9, n_heads=4, scale=0.1)), None, 0, None,
                                None) == L.FMD_EINVAL


def _sharing(n_pages=4, names=2, **kw):
    """Slots 0 .. names - 1 name one partial page."""
    c = HostCache(n_pages=n_pages, slots=[(i, [0], 10) for i in range(names)], **kw)
    for i in range(names):
        c._upload(i, 0)
    return c


def test_sharers_of_a_page_need_one_page_less_than_they_are():
    """The last of them keeps the page itself."""
    c = _sharing(n_pages=2)
    c.step([0, 1], [1, 1])
    assert c.pages(0) == [1] and c.pages(1) == [0] and c.free_pages == 0 and c.calls == ["fmd_cache_copy_pages"]
    _consistent(c)
    c = _sharing(n_pages=3, names=3)
    c.step([2, 0, 1], [3, 2, 1])
    assert sorted(c.pages(i)[0] for i in range(3)) == [0, 1, 2] and c._names == [1, 1, 1]
    _consistent(c)
    c = _sharing(n_pages=3, names=3)  # not all of them: each needs its copy
    c.step([0, 1], [1, 1])
    assert c.pages(2) == [0] and c.free_pages == 0
    c = _sharing(n_pages=2, names=3)
    with pytest.raises(PKG.FmdError) as e:
        c.step([0, 1], [1, 1])
    assert e.value.status == L.FMD_ENOMEM and c._names == [3, 0]
    _consistent(c)


def test_a_slot_without_new_positions_is_left_alone():
    c = _sharing(n_pages=1)  # no page for a copy
    r = c.step([0, 1], [0, 0])
    assert r.n_rows == 0 and c.pages(0) == c.pages(1) == [0] and c.calls == []
    c.advance([1], 0)
    _consistent(c)
    c = _sharing(n_pages=2)
    c.step([0, 1], [0, 1])
    assert c.pages(0) == [0] and c.pages(1) == [1] and (c.length(0), c.length(1)) == (10, 11)
    _consistent(c)


def test_slots_given_to_the_constructor_are_in_its_own_table():
    """Without the caller's page table the cache's own holds what `slots` names."""
    c = HostCache(slots=[(2, [3, 1], 100), (0, [5, -1, 3], 150)])
    assert c.page_table.tolist() == [[5, -1, 3, -1], [-1] * 4, [3, 1, -1, -1], [-1] * 4]
    _consistent(c)
    table = torch.tensor([[5, 6, 7, 0]] * 4, dtype=torch.int32)
    HostCache(page_table=table, slots=[(2, [5, 6], 100)])  # the caller's holds it already
    assert table.tolist() == [[5, 6, 7, 0]] * 4


def test_a_launch_that_fails_leaves_the_books_alone(monkeypatch):
    def refuse(fn, *args):
        raise PKG.FmdError(L.FMD_EIO, fn.__name__)

    def books(c):
        return [list(p) if p is not None else None for p in c._pages], list(c._length), list(c._names), sorted(c._free)

    c = _sharing(n_pages=6)
    c.open(2, 0)
    table, before, call = c.page_table.clone(), books(c), c._call
    monkeypatch.setattr(c, "_call", refuse)
    for f in (lambda: c.step([0, 2], [60, 5]), lambda: c.advance([1], 1), lambda: c.fork(0, [3])):
        with pytest.raises(PKG.FmdError):
            f()
        assert books(c) == before and torch.equal(c.page_table, table)
    monkeypatch.setattr(c, "_call", call)
    c.fork(0, [3])
    c.step([0, 2], [60, 5])
    assert c.length(0) == 70 and c.length(3) == 10 and c.pages(0) == [2, 3] and c.pages(2) == [4]


def test_the_strict_comparison_refuses_a_nan(monkeypatch):
    import test_gpu_cache as base

    held = [(np.ones((5, 1, 64)), np.ones((5, 1, 64)))]

    class Fake:
        head_dim = 64

        def attend(self, layer, rows, q, **kw):
            return self.out

        def check(self):
            pass

    monkeypatch.setattr(base, "_seq_rows", lambda *a: None)
    c, q = Fake(), torch.ones(2, 1, 64)
    call = lambda f: f(c, held, "bf16", "bf16", [2], [5], 1, q=q)
    c.out = torch.ones(2, 1, 64)
    call(base._check_attend), call(ref.finite(base._check_attend))
    for bad in (float("nan"), float("inf"), -float("inf")):
        c.out = torch.ones(2, 1, 64)
        c.out[1, 0, 3] = bad
        with pytest.raises(AssertionError):
            call(ref.finite(base._check_attend))


def test_a_capture_on_the_caches_device_is_seen_from_another(monkeypatch):
    """Whether a stream is capturing is asked of the current device, which need not be
    the cache's: a graph's workspace is its own either way."""
    class Cuda:
        at, capturing = 1, {0}

        def current_device(self):
            return self.at

        def device(self, index):
            cuda = self

            class Within:
                def __enter__(self):
                    self.was, cuda.at = cuda.at, index

                def __exit__(self, *a):
                    cuda.at = self.was

            return Within()

        def is_current_stream_capturing(self):
            return self.at in self.capturing

        def current_stream(self, index):
            return type("Stream", (), {"cuda_stream": 7 + index})

    c = HostCache(kv_heads=2)
    c.open(0)
    rows = c.step([0], [1])
    c._cuda, c._index = Cuda(), 0
    a, b = c._workspace(4, rows), c._workspace(4, rows)
    assert a is not b and not c._workspaces and c._cuda.at == 1
    c._cuda.capturing = {1}  # the other device's capture is none of the cache's
    a, b = c._workspace(4, rows), c._workspace(4, rows)
    assert a is b and list(c._workspaces) == [7]
    c._cuda.at = 0
    assert c._workspace(4, rows) is a


def test_sequences_of_one_row_need_max_rows_of_one():
    """Without row offsets every sequence has a row, so a `max_rows` of 0 cannot be
    right; attention would return without its outputs."""
    import ctypes as C

    lib = PKG.load_library()
    calls = []
    att = L.CacheAttendArgs(q=4096, out=8192, q_row=512, q_head=128, out_row=512, out_head=128, scale=0.1,
                            dtype=L.DT_BF16, n_heads=4)
    cache = L.Cache(4096, 4096, L.CACHE_BF16, 1, 4, 2, 128, 2, 4, 0)
    for row0, n_rows, max_rows in ((None, 1, 0), (4096, 0, 0), (4096, 1, 0)):
        r = L.CacheRows(4096, 4096, row0, 1, n_rows, max_rows)
        calls.append(lib.fmd_cache_attend(C.byref(cache), 0, C.byref(r), C.byref(att), 4096, 1 << 40, None, None))
    assert calls == [L.FMD_EINVAL, L.FMD_OK, L.FMD_OK]


def test_attention_counts_its_units_in_32_bits():
    """Units of 32 keys of all kv heads of a sequence are numbered in 32 bits: slots whose
    positions could pass that are refused, however long the sequences are."""
    import ctypes as C

    lib = PKG.load_library()
    r = C.byref(L.CacheRows(4096, 4096, None, 1, 1, 1))

    def attend(kv_heads, pages):
        cache = L.Cache(4096, 4096, L.CACHE_BF16, 1, 4, kv_heads, 128, 2, pages, 0)
        att = L.CacheAttendArgs(q=4096, out=1 << 30, q_row=kv_heads * 128, q_head=128, out_row=kv_heads * 128, out_head=128,
                                scale=0.1, dtype=L.DT_BF16, n_heads=kv_heads)
        return lib.fmd_cache_attend(C.byref(cache), 0, r, C.byref(att), 4096, 1 << 40, None, None)

    for kv_heads, pages in ((64, 2**24), (1024, 2**20), (32, 2**25 - 1)):
        assert attend(kv_heads, pages) == L.FMD_ENOTSUP, (kv_heads, pages)
    for kv_heads, pages in ((64, 2**24 - 9), (1024, 2**20 - 9), (1, 2**25 - 1), (8, 2**25 - 1)):
        assert attend(kv_heads, pages) == L.FMD_EINVAL, (kv_heads, pages)  # host memory is not a pool
