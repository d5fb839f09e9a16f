"""The paged cache's host side on the CPU: page bookkeeping, argument checks of
the Python class and of the C ABI, and the 64-bit reference of the cache tests."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import cache_ref as ref
from conftest import PKG

torch = pytest.importorskip("torch")
L = PKG._lib


class HostCache(PKG.PagedCache):
    """Bookkeeping on CPU tensors; operator calls are recorded, not made."""

    def __init__(self, **kw):
        self.calls = []
        base = dict(layers=2, kv_heads=2, head_dim=64, n_pages=8, max_slots=4, max_pages_per_slot=4, device="cpu")
        super().__init__(**{**base, **kw})

    def _call(self, fn, *args):
        self.calls.append(fn.__name__)


def _consistent(c):
    """Every page is free or named exactly as often as slots name it, and the
    table holds the slots' pages."""
    named = [0] * c.n_pages
    for s, pages in enumerate(c._pages):
        for k, p in enumerate(pages or ()):
            assert int(c.page_table[s, k]) == p
            if p >= 0:
                named[p] += 1
    assert named == c._names
    assert sorted(c._free) == [p for p in range(c.n_pages) if not named[p]]


def test_pages_are_taken_lowest_first_and_come_back():
    c = HostCache()
    c.open(0, 65)
    c.open(1)
    assert c.pages(0) == [0, 1] and c.pages(1) == [] and c.free_pages == 6
    r = c.step([1, 0], [130, 64])
    assert c.pages(1) == [2, 3, 4] and c.length(1) == 130 and c.length(0) == 64
    assert r.row0.tolist() == [0, 130, 194] and r.pos0.tolist() == [0, 0] and (r.n_rows, r.max_rows) == (194, 130)
    _consistent(c)
    c.release(0)
    c.open(3, 1)
    assert c.pages(3) == [0]
    c.step([3], [1])
    r = c.step([3, 1], [1, 1])
    assert r.row0 is None and r.pos0.tolist() == [1, 130] and r.slot.tolist() == [3, 1]
    r.advance()
    assert r.pos0.tolist() == [2, 131]


def test_a_failed_step_changes_nothing():
    c = HostCache()
    c.open(0)
    c.open(1)
    before = (list(c._free), list(c._length))
    for slots, counts, status in (([0, 1], [256, 257], L.FMD_EOVERFLOW), ([0, 1, 2], [1, 1, 1], L.FMD_EINVAL),
                                  ([0, 0], [1, 1], L.FMD_EINVAL), ([0], [-1], L.FMD_EINVAL),
                                  ([0], [1, 1], L.FMD_EINVAL)):
        with pytest.raises(PKG.FmdError) as e:
            c.step(slots, counts)
        assert e.value.status == status
    with pytest.raises(PKG.FmdError, match="free pages"):
        HostCache(n_pages=3).open(0, 4 * 64)
    c.open(2)
    with pytest.raises(PKG.FmdError, match="free pages") as e:
        c.step([0, 1, 2], [256, 256, 1])
    assert e.value.status == L.FMD_ENOMEM
    assert (list(c._free), [c._length[0], c._length[1]]) == (before[0], before[1][:2])
    _consistent(c)


def test_fork_shares_full_pages_and_release_counts_names():
    c = HostCache()
    c.open(0)
    c.step([0], [150])
    c.fork(0, [2, 3])
    assert c.calls == ["fmd_cache_fork"]
    assert c.pages(2) == [0, 1, 3] and c.pages(3) == [0, 1, 4] and c.length(3) == 150
    assert c._names[:5] == [3, 3, 1, 1, 1]
    c.release(0)
    assert c._names[:5] == [2, 2, 0, 1, 1] and 2 in c._free and 0 not in c._free
    with pytest.raises(PKG.FmdError) as e:
        c.fork(2, [3])
    assert e.value.status == L.FMD_EBUSY
    with pytest.raises(PKG.FmdError, match="twice"):
        c.fork(2, [0, 0])
    with pytest.raises(PKG.FmdError, match="not open"):
        c.fork(0, [1])
    c.release(2, 3)
    assert c.free_pages == 8
    c.open(0)
    c.step([0], [128])  # no partial page: nothing to copy, nothing taken
    c.fork(0, [1])
    assert c.pages(1) == c.pages(0) and c.free_pages == 6
    with pytest.raises(PKG.FmdError, match="listed twice"):
        c.release(0, 0)


def test_a_shared_page_is_copied_before_it_is_written():
    c = HostCache(slots=[(0, [5, 6], 70), (1, [5, 6], 70)], page_table=torch.full((4, 4), -1, dtype=torch.int32))
    c._upload(0, 0), c._upload(1, 0)
    c.step([0], [1])
    assert "fmd_cache_copy_pages" in c.calls
    assert c.pages(0) == [5, 0] and c.pages(1) == [5, 6]
    _consistent(c)
    c.calls.clear()
    c.step([1], [1])
    assert c.calls == [] and c.pages(1) == [5, 6]


def test_evict_frees_what_no_later_row_sees():
    for length, window, sinks, gone in ((256, 64, 0, [0, 1]), (256, 1, 0, [0, 1, 2, 3]), (255, 64, 0, [0, 1, 2][:3]),
                                        (256, 65, 0, [0, 1, 2]), (256, 64, 1, [1, 2]), (256, 64, 65, [2]),
                                        (10, 4, 0, []), (256, 1000, 0, [])):
        c = HostCache(max_pages_per_slot=5)
        c.open(0)
        c.step([0], [length])
        c.evict(0, window, sinks)
        pages = c.pages(0)
        # the next row is at `length`: it sees j > length - window and j < sinks
        for k in range(len(pages)):
            seen = any(j > length - window or j < sinks for j in range(64 * k, min(64 * k + 64, length)))
            later = any(j > length - window for j in range(64 * k, 64 * k + 64))
            assert (pages[k] >= 0) == (seen or later), (length, window, sinks, k)
        _consistent(c)
    c = HostCache()
    c.open(0)
    c.step([0], [70])
    with pytest.raises(PKG.FmdError, match="window"):
        c.evict(0, 0)


def test_a_page_evicted_ahead_of_its_rows_is_taken_again():
    c = HostCache()
    c.open(0, 256)
    c.step([0], [128])
    assert c.evict(0, 1) == 2  # the two full pages; those reserved ahead stay
    assert c.pages(0) == [-1, -1, 2, 3]
    c.step([0], [10])
    _consistent(c)


def test_compact_bookkeeping(monkeypatch):
    c = HostCache(n_pages=10)
    moved = []
    monkeypatch.setattr(c, "compact_tables", lambda t, n: moved.append(n.tolist()))
    c.open(0), c.open(1), c.open(2)
    c.step([0, 1, 2], [128, 128, 64])
    c.release(0)
    c.fork(2, [3])
    assert c.compact() == 3 and moved == [[0, 2, 1, 1]]
    assert c.pages(1) == [2, 0] and c.pages(2) == [1] and c.pages(3) == [1]
    assert sorted(c._free) == list(range(3, 10)) and c._names[:4] == [1, 2, 1, 0]


def test_constructor_refusals():
    for kw, status in ((dict(kind="int4"), L.FMD_EINVAL), (dict(head_dim=96), L.FMD_ENOTSUP),
                       (dict(layers=0), L.FMD_EINVAL), (dict(max_pages_per_slot=2**26), L.FMD_ENOTSUP),
                       (dict(pool=torch.zeros(3, dtype=torch.uint8)), L.FMD_EINVAL),
                       (dict(page_table=torch.zeros(4, 4)), L.FMD_EINVAL),
                       (dict(slots=[(0, [9], 1)]), L.FMD_EINVAL), (dict(slots=[(0, [1], 65)]), L.FMD_EINVAL),
                       (dict(slots=[(7, [1], 1)]), L.FMD_EINVAL)):
        with pytest.raises(PKG.FmdError) as e:
            HostCache(**kw)
        assert e.value.status == status, kw


def _aligned(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def test_operator_refusals():
    c = HostCache()
    c.open(0)
    rows = c.step([0], [3])
    k, q = _aligned(3, 2, 64), _aligned(3, 4, 64)
    big = _aligned(3, 2, 72)
    w = _aligned(64)
    cs = torch.zeros(8, 32)
    bad = [
        lambda: c.append(2, rows, k, k), lambda: c.append(0, rows, k[:2], k[:2]),
        lambda: c.append(0, rows, k.half(), k.half()), lambda: c.append(0, rows, k, k.half()),
        lambda: c.append(0, rows, k.float(), k), lambda: c.append(0, rows, _aligned(3, 3, 64), k),
        lambda: c.append(0, rows, big[..., 1:65], k), lambda: c.append(0, rows, _aligned(3, 64, 2).transpose(1, 2), k),
        lambda: c.append(0, rows, _aligned(3, 2, 68)[..., :64], k),
        lambda: c.append(0, rows, k, k, q_norm=w), lambda: c.append(0, rows, k, k, q=q, k_norm=w[:32]),
        lambda: c.append(0, rows, k, k, k_norm=w.float()), lambda: c.append(0, rows, k, k, cos=cs),
        lambda: c.append(0, rows, k, k, cos=cs[:, :6].contiguous(), sin=cs[:, :6].contiguous()),
        lambda: c.append(0, rows, k, k, cos=torch.zeros(8, 36), sin=torch.zeros(8, 36)),
        lambda: c.append(0, rows, k, k, cos=cs, sin=cs.half()), lambda: c.append(0, rows, k, k, q=q, q_out=k),
        lambda: c.attend(0, rows, q, window=-1), lambda: c.attend(0, rows, q, sinks=-1),
        lambda: c.attend(0, rows, _aligned(3, 3, 64)), lambda: c.attend(0, rows, _aligned(3, 12, 64)),
        lambda: c.attend(0, rows, q[:1]), lambda: c.attend(0, rows, q, out=k), lambda: c.attend(5, rows, q),
        lambda: c.read(0, rows, k_out=torch.zeros(3, 2, 32)), lambda: c.copy_pages([0, 1], [1, 2]),
        lambda: c.copy_pages([0, 1], [2, 2]), lambda: c.copy_pages([0], [8]), lambda: c.copy_pages([0], []),
        lambda: c.rows(torch.zeros(2), torch.zeros(2)),
        lambda: c.rows(torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)),
        lambda: c.rows(torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), max_rows=4),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(PKG.FmdError):
            f()
            pytest.fail(f"call {i} was accepted")
    assert c.calls == []


def _c_cache(**kw):
    base = dict(pool=4096, page_table=4096, format=L.CACHE_BF16, layers=1, n_pages=4, kv_heads=2, head_dim=128,
                max_slots=2, max_pages_per_slot=4, reserved=0)
    return L.Cache(**{**base, **kw})


def _c_rows(**kw):
    return L.CacheRows(**{**dict(slot=4096, pos0=4096, row0=None, n_seqs=1, n_rows=1, max_rows=1), **kw})


def _c_append(**kw):
    return L.CacheAppendArgs(**{**dict(k=4096, v=4096, k_row=256, k_head=128, v_row=256, v_head=128, dtype=L.DT_BF16),
                                **kw})


def _c_attend(**kw):
    return L.CacheAttendArgs(**{**dict(q=4096, out=8192, q_row=512, q_head=128, out_row=512, out_head=128, scale=0.1,
                                       dtype=L.DT_BF16, n_heads=4), **kw})


def test_c_entry_points_refuse_bad_arguments_before_touching_memory():
    """Pointers here are never valid: a call that gets past its checks would
    still be refused (not device memory), so the codes that differ from
    FMD_EINVAL pin the order, and none of these may return FMD_OK."""
    lib = PKG.load_library()

    def append(c=None, layer=0, r=None, a=None):
        return lib.fmd_cache_append(C.byref(c or _c_cache()), layer, C.byref(r or _c_rows()),
                                    C.byref(a or _c_append()), None, None)

    def attend(c=None, layer=0, r=None, a=None, ws=4096, nb=1 << 40):
        return lib.fmd_cache_attend(C.byref(c or _c_cache()), layer, C.byref(r or _c_rows()),
                                    C.byref(a or _c_attend()), ws, nb, None, None)

    inval = [dict(c=_c_cache(pool=None)), dict(c=_c_cache(pool=4100)), dict(c=_c_cache(page_table=None)),
             dict(c=_c_cache(format=3)), dict(c=_c_cache(layers=0)), dict(layer=1), dict(layer=-1),
             dict(r=_c_rows(n_seqs=-1)), dict(r=_c_rows(slot=None)), dict(r=_c_rows(n_seqs=2))]
    for kw in inval:
        assert append(**kw) == L.FMD_EINVAL and attend(**kw) == L.FMD_EINVAL, kw
    for kw in (dict(c=_c_cache(head_dim=96)), dict(c=_c_cache(max_pages_per_slot=2**26))):
        assert append(**kw) == L.FMD_ENOTSUP and attend(**kw) == L.FMD_ENOTSUP
    for kw in (dict(k=None), dict(v=4100), dict(dtype=L.DT_F32), dict(dtype=L.DT_F16), dict(n_heads=2),
               dict(q=4096, q_out=4096), dict(q=4096, n_heads=2), dict(k_row=4), dict(v_head=-8), dict(rot_dim=12),
               dict(rot_dim=136, cos_table=4096, sin_table=4096, table_rows=1), dict(rot_dim=64),
               dict(rot_dim=64, cos_table=4096, sin_table=4096), dict(k_norm=4096, eps=float("nan"))):
        assert append(a=_c_append(**kw)) == L.FMD_EINVAL, kw
    for kw in (dict(q=None), dict(out=8200), dict(dtype=9), dict(dtype=L.DT_F16), dict(n_heads=3), dict(n_heads=0),
               dict(window=-1), dict(sinks=-1), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")),
               dict(out_row=12)):
        assert attend(a=_c_attend(**kw)) == L.FMD_EINVAL, kw
    assert attend(a=_c_attend(n_heads=6)) == L.FMD_ENOTSUP and attend(a=_c_attend(n_heads=64)) == L.FMD_ENOTSUP
    # nothing to do is fine, whatever the pointers
    for kw in (dict(n_seqs=0, slot=None, pos0=None), dict(n_seqs=0, n_rows=0)):
        assert append(r=_c_rows(**kw)) == L.FMD_OK and attend(r=_c_rows(**kw)) == L.FMD_OK
    # host memory is not a pool
    assert append() == L.FMD_EINVAL and attend() == L.FMD_EINVAL
    ia = lambda *v: (C.c_int32 * len(v))(*v)
    cc = C.byref(_c_cache())
    assert lib.fmd_cache_copy_pages(cc, 1, ia(0), ia(4), None) == L.FMD_EINVAL
    assert lib.fmd_cache_copy_pages(cc, -1, ia(0), ia(1), None) == L.FMD_EINVAL
    assert lib.fmd_cache_copy_pages(cc, 0, None, None, None) == L.FMD_OK
    for src, dst, n, page, code in ((0, 0, 5, 1, L.FMD_EINVAL), (0, 2, 5, 1, L.FMD_EINVAL), (0, 1, -1, 1, L.FMD_EINVAL),
                                    (0, 1, 5, 4, L.FMD_EINVAL), (0, 1, 257, 1, L.FMD_EOVERFLOW)):
        assert lib.fmd_cache_fork(cc, 1, ia(src), ia(dst), ia(n), ia(page), None, None) == code
    assert lib.fmd_cache_compact(cc, 4096, 4096, 8, 4096, None, None) == L.FMD_EINVAL


def test_sizes():
    lib = PKG.load_library()
    assert [lib.fmd_cache_block_bytes(f, d) for f, d in ((1, 128), (2, 64), (4, 128), (4, 64), (3, 128), (4, 96))] == [
        16384, 8192, 4608, 2304, 0, 0]
    assert lib.fmd_cache_pool_bytes(C.byref(_c_cache(layers=3))) == 3 * 4 * 2 * 2 * 16384
    assert C.sizeof(L.Cache) == 48 and C.sizeof(L.CacheRows) == 40
    assert C.sizeof(L.CacheAppendArgs) == 152 and C.sizeof(L.CacheAttendArgs) == 72


def test_reference_quantiser_holds_its_promise():
    x = np.random.default_rng(0).standard_normal((50, 64)) * np.exp(np.random.default_rng(1).uniform(-4, 4, (50, 1)))
    x[3, :32] = 0
    v, d = ref.quantise(x)
    step = np.repeat(np.abs(d), 32, -1).reshape(x.shape)
    # a value lies within half a step of its code, a whole one where the codes end (+7.5 .. +8 steps of the other sign)
    assert (np.abs(v - x) <= step * (1 + 2.0 ** -7)).all()
    inside = np.abs(x) <= 7.4 * step
    assert (np.abs(v - x)[inside] <= step[inside] * (0.5 + 2.0 ** -7)).all() and (v[3, :32] == 0).all()


def test_reference_attention_of_one_key_is_its_value():
    rng = np.random.default_rng(2)
    q, k, v = rng.standard_normal((3, 2, 64)), rng.standard_normal((9, 1, 64)), rng.standard_normal((9, 1, 64))
    out, _ = ref.attend(q, k, v, [6, 7, 8], window=1)
    assert np.allclose(out[:, 1], v[6:9, 0])
    full, _ = ref.attend(q, k, v, [6, 7, 8])
    wide, _ = ref.attend(q, k, v, [6, 7, 8], window=9)
    sunk, _ = ref.attend(q, k, v, [6, 7, 8], window=1, sinks=9)
    assert np.allclose(full, wide) and np.allclose(full, sunk)


@pytest.mark.parametrize("fmt", [L.CACHE_BF16, L.CACHE_Q4])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_workspace_serves_smaller_calls(fmt, dim):
    """The workspace for up to n_seqs sequences of up to max_rows rows is large
    enough for every smaller call."""
    lib = PKG.load_library()
    c = C.byref(_c_cache(format=fmt, head_dim=dim))
    for heads in (2, 16, 32):
        sizes = [lib.fmd_cache_attend_workspace(c, heads, n, m) for n in (1, 64, 5000) for m in range(1, 40)]
        sizes += [lib.fmd_cache_attend_workspace(c, heads, 5000, m) for m in (512, 4096, 100000)]
        for n in range(3):
            part = sizes[n * 39:(n + 1) * 39]
            assert part == sorted(part) and part[0] > 0
        assert sizes[-1] >= max(sizes)


def test_c_entry_points_refuse_the_same_index_twice():
    lib = PKG.load_library()
    ia = lambda *v: (C.c_int32 * len(v))(*v)
    cc = C.byref(_c_cache(n_pages=16, max_slots=8))
    for src, dst in (((0, 1), (2, 2)), ((0, 1), (1, 2)), ((0, 1), (2, 1)), ((3,), (3,))):
        assert lib.fmd_cache_copy_pages(cc, len(src), ia(*src), ia(*dst), None) == L.FMD_EINVAL
    for src, dst, page in (((0, 0), (2, 2), (3, 4)), ((0, 1), (1, 2), (3, 4)), ((0, 1), (2, 0), (3, 4)),
                           ((0, 0), (1, 2), (3, 3))):
        assert lib.fmd_cache_fork(cc, 2, ia(*src), ia(*dst), ia(5, 70), ia(*page), None, None) == L.FMD_EINVAL
    # queries are read until the last output is written
    assert lib.fmd_cache_attend(cc, 0, C.byref(_c_rows()), C.byref(_c_attend(out=_c_attend().q)), 4096, 1 << 40, None,
                                None) == L.FMD_EINVAL
