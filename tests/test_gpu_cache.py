"""The paged-cache operators on the GPU against the 64-bit restatement
(`cache_ref`)."""

from __future__ import annotations

import numpy as np
import pytest

import cache_ref as ref
from conftest import PKG

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def _eps(dtype):
    return torch.finfo(DT[dtype]).eps


def _rand(rng, *shape, dtype="bf16", scale=1.0):
    return torch.from_numpy((rng.standard_normal(shape) * scale).astype(np.float32)).to(DT[dtype]).cuda()


def _np(t):
    return t.detach().double().cpu().numpy()


def _tables(positions, pairs, theta=1e4):
    ang = np.arange(positions)[:, None] / theta ** (np.arange(pairs) / pairs)
    return [torch.from_numpy(f(ang).astype(np.float32)).cuda() for f in (np.cos, np.sin)]


def _cache(kind, dim=128, kv_heads=2, layers=1, n_pages=40, max_slots=6, max_pages=32, **kw):
    return PKG.PagedCache(layers, kv_heads, dim, n_pages, max_slots, max_pages, kind=kind, **kw)


def _filled(kind, dtype, lengths, dim=128, kv_heads=2, seed=0, layer=0, layers=1, scale=1.0):
    """A cache whose slot i holds lengths[i] random positions in scattered pages,
    and what it holds as 64-bit (k, v) per slot."""
    rng = np.random.default_rng(seed)
    need = [-(-n // 64) for n in lengths]
    c = _cache(kind, dim, kv_heads, layers=layers, n_pages=sum(need) + 3, max_slots=len(lengths),
               max_pages=max(need) + 1)
    c.pool.random_(0, 256)  # what rows were not written hold anything, NaN included
    perm = rng.permutation(c.n_pages).tolist()
    slots = [(i, [perm.pop() for _ in range(k)], 0) for i, k in enumerate(need)]
    c = PKG.PagedCache(layers, kv_heads, dim, c.n_pages, c.max_slots, c.max_pages_per_slot, kind=kind, pool=c.pool,
                       page_table=c.page_table, slots=slots)
    for s, _, _ in slots:
        c._upload(s, 0)
    rows = c.step(range(len(lengths)), lengths)
    n = sum(lengths)
    k, v = _rand(rng, n, kv_heads, dim, dtype=dtype), _rand(rng, n, kv_heads, dim, dtype=dtype, scale=scale)
    c.append(layer, rows, k, v)
    c.check()
    held, at = [], 0
    for m in lengths:
        kk, vv = _np(k[at:at + m]), _np(v[at:at + m])
        held.append((ref.quantise(kk)[0], ref.quantise(vv)[0]) if kind == "q4" else (kk, vv))
        at += m
    return c, held


def _seq_rows(c, slots, counts, ends, max_rows=None):
    """Rows of the last counts[i] positions of each slot (they are cached)."""
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    row0 = np.concatenate([[0], np.cumsum(counts)])
    one = all(n == 1 for n in counts)
    return c.rows(t(slots), t([e - n for e, n in zip(ends, counts)]), None if one else t(row0),
                  max_rows=max_rows or max(counts), n_rows=int(row0[-1]))


def _check_attend(c, held, kind, dtype, counts, lengths, heads, window=0, sinks=0, scale=None, seed=5, q=None,
                  slots=None, **kw):
    slots = list(range(len(counts))) if slots is None else slots
    if q is None:
        q = _rand(np.random.default_rng(seed), sum(counts), heads, c.head_dim, dtype=dtype)
    out = c.attend(0, _seq_rows(c, slots, counts, lengths), q, window=window, sinks=sinks, scale=scale, **kw)
    c.check()
    at = 0
    for s, n, end in zip(slots, counts, lengths):
        k, v = held[s]
        want, mag = ref.attend(_np(q[at:at + n]), k, v, range(end - n, end), window, sinks, scale)
        got = _np(out[at:at + n])
        tol = ref.attend_tolerance(want, mag, _eps(dtype), kind == "q4")
        bad = np.abs(got - want) > tol
        assert not bad.any(), (s, n, end, np.argwhere(bad)[:4].tolist(), np.abs(got - want).max(), np.isnan(got).any())
        at += n
    return out


# ---- append ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim,rot,inter", [(128, 128, False), (128, 64, False), (128, 8, True), (128, 128, True),
                                           (64, 64, False), (64, 24, False), (64, 16, True), (64, 0, False),
                                           (128, 0, False)])
def test_append_norms_rotates_and_stores(dtype, dim, rot, inter):
    rng = np.random.default_rng(dim + rot)
    counts, kv_heads, heads = [1, 70, 0, 5], 3, 6
    c = _cache(dtype, dim, kv_heads, n_pages=12, layers=2)
    for s in range(4):
        c.open(s)
    c.step([0, 3], [63, 100])  # positions that are not written here
    rows = c.step([0, 1, 2, 3], counts)
    n = sum(counts)
    x = _rand(rng, n + 2, heads + 2 * kv_heads, dim, dtype=dtype, scale=3.0)
    q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    qw, kw = _rand(rng, dim, dtype=dtype), _rand(rng, dim, dtype=dtype)
    cos, sin = _tables(200, rot // 2) if rot else (None, None)
    q_out = torch.full((n + 2, heads, dim), 7.0, dtype=DT[dtype], device="cuda")
    before = c.pool.clone()
    got = c.append(1, rows, k, v, q=q, q_norm=qw, k_norm=kw, eps=1e-5, cos=cos, sin=sin, interleaved=inter,
                   q_out=q_out)
    c.check()
    pos = np.concatenate([np.arange(p, p + m) for p, m in zip((63, 0, 0, 100), counts)])
    cs = (_np(cos)[pos], _np(sin)[pos]) if rot else (None, None)
    for name, src, w, res in (("q", q, qw, _np(got[:n])), ("k", k, kw, None), ("v", v, None, None)):
        if res is None:
            kk, vv = c.read(1, rows, n_rows=n)
            res = _np(kk if name == "k" else vv)
        plain = name == "v"
        want = ref.norm_rotate(_np(src[:n]), None if plain else _np(w), 1e-5, *((None, None) if plain else cs), inter)
        tol = ref.append_tolerance(want, np.abs(want).max(-1, keepdims=True), _eps(dtype))
        assert (np.abs(res - want) <= tol).all(), name
    assert (got[n:] == 7).all()  # rows behind the last sequence
    # nothing but the rows' own positions was written: undo them and compare
    blk = c.pool.view(DT[dtype]).view(2, 12, 2, kv_heads, 64, dim)
    old = before.view(DT[dtype]).view(2, 12, 2, kv_heads, 64, dim)
    seq = np.repeat(np.arange(4), counts)
    for s, p in zip(seq, pos):
        page = c.pages(int(s))[p // 64]
        blk[1, page, :, :, p % 64] = old[1, page, :, :, p % 64]
    assert torch.equal(c.pool, before)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_append_4_bits_is_exact(dtype, dim):
    rng = np.random.default_rng(dim)
    c = _cache("q4", dim, 3, n_pages=8)
    c.open(1)
    c.open(4)
    rows = c.step([4, 1], [130, 67])
    n = 197
    k, v = _rand(rng, n, 3, dim, dtype=dtype), _rand(rng, n, 3, dim, dtype=dtype, scale=0.01)
    k[0] = 0                       # a block of zeros
    k[1, :, :32] = k[1, :, :32].abs().max()   # equal magnitudes: the first counts
    k[1, :, 1] = -k[1, :, 0]
    k[2] = torch.round(k[2] * 8) / 16  # many values half way between two codes
    v[3] = v[3] * 2.0 ** -12       # scales in the f16 subnormal range
    if dtype == "bf16":
        v[4, 0, 5], v[4, 1, 7] = 3e38, -1e6  # saturate
    c.append(0, rows, k, v)
    got_k, got_v = c.read(0, rows)
    c.check()
    assert np.array_equal(_np(got_k), ref.quantise(_np(k))[0])
    assert np.array_equal(_np(got_v), ref.quantise(_np(v))[0])
    # a NaN or an infinity makes its block of 32 NaN, and only that
    k[5, 1, 40] = float("nan")
    k[6, 2, 3] = float("-inf")
    c.append(0, rows, k, v)
    bad = np.isnan(_np(c.read(0, rows)[0]))
    want = np.zeros_like(bad)
    want[5, 1, 32:64] = want[6, 2, :32] = True
    assert np.array_equal(bad, want)


def test_append_4_bits_with_norm_and_rotation():
    rng = np.random.default_rng(3)
    for inter in (False, True):
        c = _cache("q4", 128, 2)
        c.open(0)
        rows = c.step([0], [90])
        x = _rand(rng, 90, 4, 128)
        kw = _rand(rng, 128)
        cos, sin = _tables(90, 64)
        c.append(0, rows, x[:, :2], x[:, 2:], k_norm=kw, cos=cos, sin=sin, interleaved=inter)
        c.check()
        want = ref.norm_rotate(_np(x[:, :2]), _np(kw), 1e-6, _np(cos), _np(sin), inter)
        step = np.repeat(np.abs(ref.quantise(want)[1]), 32, -1).reshape(want.shape)
        # a value on a border may take either code (as in the exact test otherwise)
        near = np.abs(_np(c.read(0, rows)[0]) - ref.quantise(want)[0])
        assert (near <= step * (1 + 2.0 ** -6)).all() and (near > step * 2.0 ** -6).mean() < 1e-3


def test_append_in_place_and_one_head():
    rng = np.random.default_rng(4)
    c = _cache("bf16", 64, 1, max_slots=2)
    c.open(0)
    rows = c.step([0], [9])
    q, k, v = (_rand(rng, 9, 1, 64) for _ in range(3))
    cos, sin = _tables(9, 32)
    want = ref.norm_rotate(_np(q), None, 0, _np(cos), _np(sin))
    out = c.append(0, rows, k, v, q=q, cos=cos, sin=sin, q_out=q)
    assert out is q
    assert (np.abs(_np(q) - want) <= ref.append_tolerance(want, np.abs(want).max(-1, keepdims=True), _eps("bf16"))).all()


# ---- attention --------------------------------------------------------------------------

LENGTHS = [1, 2, 63, 64, 65, 129, 700, 1029]


@pytest.mark.parametrize("kind,dtype", [("bf16", "bf16"), ("f16", "f16"), ("q4", "bf16"), ("q4", "f16")])
@pytest.mark.parametrize("dim,kv_heads,group", [(128, 2, 2), (64, 3, 1), (128, 1, 4), (64, 2, 8), (128, 1, 16),
                                                (64, 1, 16), (128, 3, 8)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (64, 0), (100, 4), (257, 70), (5000, 3)])
def test_attend_one_row_per_sequence(kind, dtype, dim, kv_heads, group, window, sinks):
    c, held = _filled(kind, dtype, LENGTHS, dim, kv_heads)
    _check_attend(c, held, kind, dtype, [1] * len(LENGTHS), LENGTHS, kv_heads * group, window, sinks)


@pytest.mark.parametrize("kind,dtype", [("bf16", "bf16"), ("f16", "f16"), ("q4", "bf16"), ("q4", "f16")])
@pytest.mark.parametrize("dim,kv_heads,group", [(128, 2, 2), (64, 1, 1), (128, 1, 4), (64, 2, 8), (128, 1, 16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 1), (65, 0), (100, 4), (257, 70)])
def test_attend_chunks(kind, dtype, dim, kv_heads, group, window, sinks):
    lengths, counts = [1, 65, 200, 300, 129, 131], [1, 65, 3, 131, 0, 64]
    c, held = _filled(kind, dtype, lengths, dim, kv_heads, seed=1)
    _check_attend(c, held, kind, dtype, counts, lengths, kv_heads * group, window, sinks)


@pytest.mark.parametrize("kind", ["bf16", "q4"])
@pytest.mark.parametrize("counts", [[2, 1, 7], [9, 8, 1], [16, 17, 33], [1, 0, 1]])
def test_attend_short_chunks(kind, counts):
    lengths = [400, 70, 129]
    c, held = _filled(kind, "bf16", lengths, seed=2)
    _check_attend(c, held, kind, "bf16", counts, lengths, 4, 90, 5)
    _check_attend(c, held, kind, "bf16", counts, lengths, 4)


@pytest.mark.parametrize("kind", ["f16", "q4"])
def test_attend_one_long_sequence(kind):
    c, held = _filled(kind, "f16", [20011], seed=3)
    _check_attend(c, held, kind, "f16", [1], [20011], 4)
    _check_attend(c, held, kind, "f16", [1], [20011], 4, 9000, 130)
    _check_attend(c, held, kind, "f16", [5], [20011], 4, 9000, 130)


@pytest.mark.parametrize("kind", ["bf16", "q4"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads", [1, 2, 16])
def test_attend_one_segment_over_the_whole_grid(kind, dim, heads):
    """One kv head: every block has a piece of the same segment."""
    c, held = _filled(kind, "bf16", [20011], dim, 1, seed=3)
    for count in (1, 3):
        _check_attend(c, held, kind, "bf16", [count], [20011], heads)


@pytest.mark.parametrize("kind", ["bf16", "q4"])
def test_attend_many_sequences_of_several_rows(kind):
    """So many (sequence, tile) pairs that items are dealt out whole."""
    counts = [40 - i % 9 for i in range(300)]
    lengths = [n + (37 * i) % 150 for i, n in enumerate(counts)]
    c, held = _filled(kind, "bf16", lengths, 64, 1, seed=4)
    counts[17] = 0
    q = _rand(np.random.default_rng(5), sum(counts), 16, 64)
    out = c.attend(0, _seq_rows(c, list(range(300)), counts, lengths, max_rows=65), q, window=33, sinks=2)
    c.check()
    assert torch.equal(out, c.attend(0, _seq_rows(c, list(range(300)), counts, lengths, max_rows=65), q, window=33,
                                     sinks=2))
    at = 0
    for s, (n, end) in enumerate(zip(counts, lengths)):
        if s % 7 == 3 and n:
            want, mag = ref.attend(_np(q[at:at + n]), *held[s], range(end - n, end), 33, 2)
            assert (np.abs(_np(out[at:at + n]) - want) <= ref.attend_tolerance(want, mag, _eps("bf16"), kind == "q4")).all()
        at += n


@pytest.mark.parametrize("kind", ["bf16", "q4"])
def test_attend_many_sequences(kind):
    lengths = [1 + (37 * i) % 150 for i in range(300)]
    c, held = _filled(kind, "bf16", lengths, 64, 1, seed=4)
    _check_attend(c, held, kind, "bf16", [1] * 300, lengths, 2, 33, 2)


@pytest.mark.parametrize("kind,dtype", [("bf16", "bf16"), ("f16", "f16"), ("q4", "bf16"), ("q4", "f16")])
@pytest.mark.parametrize("dim,group", [(64, 2), (128, 1)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 3), (300, 70)])
def test_attend_many_chunk_items_per_block(kind, dtype, dim, group, window, sinks):
    """More (tile, sequence, head) items than blocks: every block goes through
    several, of odd and even numbers of key tiles, some with one half empty."""
    counts = [900, 130, 1, 640, 257, 700, 64, 513]
    lengths = [n + 37 * i for i, n in enumerate(counts)]
    c, held = _filled(kind, dtype, lengths, dim, 8, seed=21)
    q = _rand(np.random.default_rng(5), sum(counts), 8 * group, dim, dtype=dtype)
    rows = _seq_rows(c, list(range(8)), counts, lengths)
    out = c.attend(0, rows, q, window=window, sinks=sinks)
    c.check()
    for _ in range(5):
        assert torch.equal(out, c.attend(0, rows, q, window=window, sinks=sinks))
    at = 0
    for s, (n, end) in enumerate(zip(counts, lengths)):
        for i in sorted({0, n // 2, max(0, n - 70), n - 1}):
            want, mag = ref.attend(_np(q[at + i:at + i + 1]), *held[s], [end - n + i], window, sinks)
            tol = ref.attend_tolerance(want, mag, _eps(dtype), kind == "q4")
            assert (np.abs(_np(out[at + i:at + i + 1]) - want) <= tol).all(), (s, i)
        at += n
    c.check()


@pytest.mark.parametrize("kind,dtype", [("bf16", "bf16"), ("f16", "f16"), ("q4", "bf16")])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("count", [1, 4])
def test_attend_many_tiles_per_block(kind, dtype, dim, count):
    """Enough pages that every ring goes round many times and a block's range
    covers whole sequences: 4 heads x about 2,800 pages."""
    lengths = [5000 - 31 * i for i in range(40)]
    c, held = _filled(kind, dtype, lengths, dim, 4, seed=17)
    q = _rand(np.random.default_rng(5), 40 * count, 8, dim, dtype=dtype)
    rows = _seq_rows(c, list(range(40)), [count] * 40, lengths)
    for window, sinks in ((0, 0), (3000, 100)):
        out = c.attend(0, rows, q, window=window, sinks=sinks)
        c.check()
        for s in (0, 7, 19, 20, 39):
            a = slice(s * count, (s + 1) * count)
            want, mag = ref.attend(_np(q[a]), *held[s], range(lengths[s] - count, lengths[s]), window, sinks)
            assert (np.abs(_np(out[a]) - want) <= ref.attend_tolerance(want, mag, _eps(dtype), kind == "q4")).all()
        # every sequence by itself: other cuts, the same sums up to roundings
        for s in range(40):
            a = slice(s * count, (s + 1) * count)
            one = c.attend(0, _seq_rows(c, [s], [count], [lengths[s]]), q[a], window=window, sinks=sinks)
            near = (_np(one) - _np(out[a])) / np.abs(_np(out[a])).max()
            assert np.abs(near).max() <= 4 * _eps(dtype)


@pytest.mark.parametrize("kind", ["bf16", "q4"])
@pytest.mark.parametrize("count", [1, 40])
def test_attend_strides_scale_and_rows_left_alone(kind, count):
    lengths = [150, 260, 90]
    c, held = _filled(kind, "bf16", lengths, seed=6)
    rng = np.random.default_rng(7)
    wide = _rand(rng, 4 * count, 9, 128)
    q = wide[:3 * count, 1:5]                       # strided rows
    back = _rand(rng, 4, 3 * count, 128)
    back.copy_(q.transpose(0, 1))
    big = torch.full((4, 4 * count, 136), 3.0, dtype=torch.bfloat16, device="cuda")
    out = big[:, :3 * count, :128].transpose(0, 1)  # heads outermost, padded rows
    _check_attend(c, held, kind, "bf16", [count] * 3, lengths, 4, 100, 3, scale=0.3, q=q, out=out)
    _check_attend(c, held, kind, "bf16", [count] * 3, lengths, 4, 100, 3, scale=0.3, q=back.transpose(0, 1))
    assert (big[:, 3 * count:] == 3).all() and (big[..., 128:] == 3).all()


@pytest.mark.parametrize("kind", ["bf16", "q4"])
@pytest.mark.parametrize("count", [1, 30])
def test_attend_padding_and_rows_behind(kind, count):
    lengths = [150, 260, 90]
    c, held = _filled(kind, "bf16", lengths, seed=6)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    q = _rand(np.random.default_rng(1), 4 * count + 2, 4, 128)
    out = torch.full_like(q, 5.0)
    row0 = None if count == 1 else t([0, count, 2 * count, 3 * count, 4 * count])
    rows = c.rows(t([1, -1, 0, -1]), t([260 - count, 0, 150 - count, -3]), row0, max_rows=count)
    c.attend(0, rows, q, window=70, sinks=2, out=out)
    c.check()
    for i, s in ((0, 1), (2, 0)):
        a = slice(i * count, (i + 1) * count)
        want, mag = ref.attend(_np(q[a]), *held[s], range(lengths[s] - count, lengths[s]), 70, 2)
        assert (np.abs(_np(out[a]) - want) <= ref.attend_tolerance(want, mag, _eps("bf16"), kind == "q4")).all()
    for a in (slice(count, 2 * count), slice(3 * count, None)):
        assert (out[a] == 5).all()
    # append leaves padding's and later rows' positions alone too
    k = _rand(np.random.default_rng(2), 4 * count + 2, 2, 128)
    before = c.pool.clone()
    c.append(0, c.rows(t([-1, -1]), t([0, 0]), None if count == 1 else t([0, count, 2 * count]), max_rows=count), k, k)
    assert torch.equal(before, c.pool)


@pytest.mark.parametrize("kind", ["bf16", "f16", "q4"])
@pytest.mark.parametrize("count", [1, 3, 40])
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_hidden_positions_have_no_influence(kind, count, poison):
    """Positions before the window, between sinks and window, and behind the
    newest row hold NaN or infinities."""
    dtype = "bf16" if kind == "q4" else kind
    length, window, sinks = 331, 100, 5
    c, held = _filled(kind, dtype, [length + 20], seed=8)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    first = length - count - window + 1  # the oldest position any row sees but the sinks
    for a, b in ((sinks, first), (length, length + 20)):
        bad = torch.full((b - a, 2, 128), poison, dtype=DT[dtype], device="cuda")
        c.append(0, c.rows(t([0]), t([a]), t([0, b - a]), max_rows=b - a), bad, bad)
    out = _check_attend(c, held, kind, dtype, [count], [length], 4, window, sinks)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("kind", ["bf16", "q4"])
def test_a_visible_nan_is_seen(kind):
    c, held = _filled(kind, "bf16", [100], seed=8)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    bad = torch.full((1, 2, 128), float("nan"), dtype=torch.bfloat16, device="cuda")
    c.append(0, c.rows(t([0]), t([50]), None), bad, bad)
    q = _rand(np.random.default_rng(0), 1, 4, 128)
    assert torch.isnan(c.attend(0, _seq_rows(c, [0], [1], [100]), q)).all()
    assert torch.isfinite(c.attend(0, _seq_rows(c, [0], [1], [100]), q, window=49)).all()


@pytest.mark.parametrize("kind,dtype", [("bf16", "bf16"), ("f16", "f16"), ("q4", "bf16"), ("q4", "f16")])
@pytest.mark.parametrize("count", [1, 50])
def test_attend_extreme_scores_and_values(kind, dtype, count):
    """One key wins by far (others underflow), large and tiny values, zero queries."""
    c, held = _filled(kind, dtype, [300], seed=9, scale=2.0 ** 12)
    q = _rand(np.random.default_rng(1), count, 4, 128, dtype=dtype)
    q[0] *= 0
    _check_attend(c, held, kind, dtype, [count], [300], 4, q=q)
    sharp = _rand(np.random.default_rng(1), count, 4, 128, dtype=dtype, scale=2.0 ** 7)
    out = c.attend(0, _seq_rows(c, [0], [count], [300]), sharp)
    for i in range(count):
        k, v = held[0]
        s = np.einsum("hd,jhd->hj", _np(sharp[i]), np.repeat(k[:300 - count + i + 1], 2, 1)) * 128 ** -0.5
        top = np.sort(s, -1)
        for h in range(4):
            if top[h, -1] - top[h, -2] > 40:  # one term: its value to the output's rounding (and 4 bits' product)
                want = v[s[h].argmax(), h // 2]
                assert (np.abs(_np(out[i, h]) - want) <= (2 ** -11 + _eps(dtype) / 2) * np.abs(want) + 1e-3).all()
    tiny, held = _filled(kind, dtype, [300], seed=10, scale=2.0 ** -9)
    _check_attend(tiny, held, kind, dtype, [count], [300], 4)


def test_attend_queries_of_any_magnitude_in_4_bits():
    """bf16 queries beyond the range of f16, with a scale that brings the scores back."""
    c, held = _filled("q4", "bf16", [200], seed=11)
    for count in (1, 40):
        for e in (-100, -30, 30, 100):
            q = _rand(np.random.default_rng(2), count, 4, 128) * 2.0 ** e
            _check_attend(c, held, "q4", "bf16", [count], [200], 4, scale=128 ** -0.5 * 2.0 ** -e, q=q)


@pytest.mark.parametrize("kind", ["bf16", "q4"])
def test_evicted_pages_are_not_looked_up(kind):
    lengths = [700, 515]
    c, held = _filled(kind, "bf16", lengths, seed=12)
    assert c.evict(0, 130, 5) == 7 and c.evict(1, 130, 5) == 5
    assert (c.page_table == -1).sum() >= 12
    _check_attend(c, held, kind, "bf16", [1, 1], lengths, 4, 130, 5)
    _check_attend(c, held, kind, "bf16", [1, 1], lengths, 4, 100, 5)
    # a page that is gone but wanted is reported, not read
    c.attend(0, _seq_rows(c, [0, 1], [1, 1], lengths), _rand(np.random.default_rng(0), 2, 4, 128))
    with pytest.raises(PKG.FmdError) as e:
        c.check()
    assert e.value.status == PKG._lib.FMD_EINVAL
    c.check()


@pytest.mark.parametrize("kind", ["bf16", "q4"])
@pytest.mark.parametrize("count", [1, 20])
def test_bad_slots_positions_and_pages_are_reported(kind, count):
    c, held = _filled(kind, "bf16", [200, 90], seed=13)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    q = _rand(np.random.default_rng(0), 2 * count, 4, 128)
    k = q[:, :2].contiguous()
    row0 = None if count == 1 else t([0, count, 2 * count])
    top = c.max_pages_per_slot * 64
    table = c.page_table.clone()
    for slot, pos, code in (([0, 2], [100, 0], "FMD_EINVAL"), ([0, -2], [100, 0], "FMD_EINVAL"),
                            ([0, 1], [100, top], "FMD_EOVERFLOW"), ([0, 1], [100, -count - 1], "FMD_EOVERFLOW"),
                            ([0, 1], [100, 2**31 - 1 - count], "FMD_EOVERFLOW")):
        before = c.pool.clone()
        out = torch.full_like(q, 5.0)
        rows = c.rows(t(slot), t(pos), row0, max_rows=count)
        c.attend(0, rows, q, out=out)
        with pytest.raises(PKG.FmdError) as e:
            c.check()
        assert e.value.status == getattr(PKG._lib, code)
        want, mag = ref.attend(_np(q[:count]), *held[0], range(100, 100 + count))
        assert (np.abs(_np(out[:count]) - want) <= ref.attend_tolerance(want, mag, _eps("bf16"), kind == "q4")).all()
        c.append(0, c.rows(t(slot[1:]), t(pos[1:]), None if count == 1 else t([0, count]), max_rows=count), k[:count],
                 k[:count])
        with pytest.raises(PKG.FmdError) as e:
            c.check()
        assert e.value.status == getattr(PKG._lib, code) and torch.equal(before, c.pool)
    for page in (-1, c.n_pages, 2**31 - 1):
        c.page_table[1, 0] = page
        c.attend(0, c.rows(t([0, 1]), t([100, 5]), row0, max_rows=count), q)
        with pytest.raises(PKG.FmdError):
            c.check()
        c.append(0, c.rows(t([1]), t([5]), None if count == 1 else t([0, count]), max_rows=count), k[:count], k[:count])
        with pytest.raises(PKG.FmdError):
            c.check()
    c.page_table.copy_(table)
    c.append(0, c.rows(t([0]), t([0]), None), k[:1], k[:1], cos=torch.ones(1, 64, device="cuda"),
             sin=torch.zeros(1, 64, device="cuda"))
    c.check()
    c.append(0, c.rows(t([0]), t([1]), None), k[:1], k[:1], cos=torch.ones(1, 64, device="cuda"),
             sin=torch.zeros(1, 64, device="cuda"))
    with pytest.raises(PKG.FmdError) as e:  # behind the rotation table
        c.check()
    assert e.value.status == PKG._lib.FMD_EOVERFLOW


@pytest.mark.parametrize("kind", ["bf16", "q4"])
def test_results_repeat_bit_for_bit(kind):
    lengths = [5000, 77, 1300]
    c, _ = _filled(kind, "bf16", lengths, seed=14)
    for counts in ([1, 1, 1], [100, 77, 3]):
        q = _rand(np.random.default_rng(0), sum(counts), 4, 128)
        rows = _seq_rows(c, [0, 1, 2], counts, lengths)
        first = c.attend(0, rows, q, window=3000, sinks=9).clone()
        for _ in range(5):
            assert torch.equal(first, c.attend(0, rows, q, window=3000, sinks=9))


# ---- pages --------------------------------------------------------------------------------


def _values(c, slot, layer):
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    n = c.length(slot)
    return c.read(layer, c.rows(t([slot]), t([0]), t([0, n]), max_rows=n), n_rows=n)


@pytest.mark.parametrize("kind", ["bf16", "f16", "q4"])
@pytest.mark.parametrize("dim,length", [(128, 150), (64, 1), (64, 191), (128, 128), (64, 65)])
def test_fork_copies_the_rows_behind_the_full_pages(kind, dim, length):
    c = _cache(kind, dim, 3, layers=3)
    c.open(0)
    rows = c.step([0], [length])
    rng = np.random.default_rng(0)
    dtype = "bf16" if kind == "q4" else kind
    for layer in range(3):
        c.append(layer, rows, _rand(rng, length, 3, dim, dtype=dtype), _rand(rng, length, 3, dim, dtype=dtype))
    before = c.pool.clone()
    c.fork(0, [2, 5])
    c.check()
    fresh = [c.pages(s)[-1] for s in (2, 5)] if length % 64 else []
    for s in (2, 5):
        for layer in range(3):
            for a, b in zip(_values(c, 0, layer), _values(c, s, layer)):
                assert torch.equal(a, b)
    # the fresh pages hold those rows and nothing else changed
    per = c.pool.numel() // (3 * c.n_pages)
    same = (c.pool.view(3, c.n_pages, per) == before.view(3, c.n_pages, per)).all(-1).all(0)
    assert [p for p in range(c.n_pages) if not same[p]] == sorted(fresh)
    if length % 64:
        blk = per // 6
        rowb = dim // 2 if kind == "q4" else 2 * dim
        tail = c.pool.view(3, c.n_pages, 6, blk)[:, fresh, :, (length % 64) * rowb:64 * rowb]
        assert torch.equal(tail, before.view(3, c.n_pages, 6, blk)[:, fresh, :, (length % 64) * rowb:64 * rowb])
    # the fork goes its own way
    step = c.step([2], [3])
    c.append(0, step, _rand(rng, 3, 3, dim, dtype=dtype), _rand(rng, 3, 3, dim, dtype=dtype))
    for layer in range(3):
        for a, b in zip(_values(c, 0, layer), _values(c, 5, layer)):
            assert torch.equal(a, b)


def test_fork_many_and_copy_many():
    c = _cache("bf16", 64, 1, n_pages=700, max_slots=300, max_pages=4)
    c.pool.random_(0, 256)
    c.open(0)
    c.step([0], [70])
    c.fork(0, list(range(1, 300)))
    pool = c.pool.view(700, -1)
    rows = 2 * 64 * 6
    for s in (1, 128, 129, 299):
        assert c.pages(s)[0] == c.pages(0)[0]
        for blk in (0, 64 * 128):
            assert torch.equal(pool[c.pages(s)[1]][blk:blk + rows], pool[c.pages(0)[1]][blk:blk + rows])
    assert torch.equal(c.page_table[299, :2].cpu(), torch.tensor(c.pages(299), dtype=torch.int32))
    src, dst = list(range(301)), list(range(350, 651))
    c.copy_pages(src, dst)
    assert torch.equal(pool[src], pool[dst])


@pytest.mark.parametrize("kind", ["bf16", "q4"])
@pytest.mark.parametrize("seed,n_pages", [(0, 40), (1, 33), (2, 1500), (3, 40000)])
def test_compact(kind, seed, n_pages):
    rng = np.random.default_rng(seed)
    layers, heads, dim = (2, 2, 128) if n_pages < 2000 else (1, 1, 64)
    c = PKG.PagedCache(layers, heads, dim, n_pages, 12, max(8, n_pages // 4), kind=kind)
    c.pool.random_(0, 256)
    perm = rng.permutation(n_pages).tolist()
    slots = []
    for s in range(0, 12, 2):
        pages = [perm.pop() for _ in range(int(rng.integers(0, n_pages // 12)))]
        if s == 4 and slots:  # shared pages and evicted ones
            pages = slots[0][1][:3] + [-1, -1] + pages
        slots.append((s, pages, 0))
    c = PKG.PagedCache(layers, heads, dim, n_pages, 12, max(8, n_pages // 4), kind=kind, pool=c.pool,
                       page_table=c.page_table, slots=slots)
    for s, _, _ in slots:
        c._upload(s, 0)
    before = c.pool.clone().view(layers, n_pages, -1)
    was = {s: c.pages(s) for s, _, _ in slots}
    used = sorted({p for pages in was.values() for p in pages if p >= 0})
    assert c.compact() == len(used)
    c.check()
    after = c.pool.view(layers, n_pages, -1)
    for s, pages in was.items():
        now = c.pages(s)
        assert torch.equal(c.page_table[s, :len(now)].cpu(), torch.tensor(now, dtype=torch.int32))
        assert all((a < 0) == (b < 0) for a, b in zip(pages, now)) and max(now, default=0) < max(1, len(used))
        keep = [(a, b) for a, b in zip(pages, now) if a >= 0]
        if keep:
            assert torch.equal(before[:, [a for a, _ in keep]], after[:, [b for _, b in keep]])
    assert c.compact() == len(used) and torch.equal(after, c.pool.view(layers, n_pages, -1))


def test_compact_reports_a_bad_page_and_goes_on():
    c = _cache("bf16", 64, 1, n_pages=10, max_slots=2, max_pages=4)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    table = t([[9, 99, -1, 5], [7, -7, 0, 0]])
    c.pool.random_(0, 256)
    want = c.pool.view(10, -1)[[9, 5, 7]].clone()
    n = c.compact_tables(table, t([4, 2]))
    with pytest.raises(PKG.FmdError):
        c.check()
    assert int(n) == 3
    got = table.cpu().tolist()
    assert got[0][1:3] == [99, -1] and got[1][1] == -7
    assert torch.equal(c.pool.view(10, -1)[[got[0][0], got[0][3], got[1][0]]], want)


# ---- together, streams, graphs ----------------------------------------------------------------


def _decode_model(c, held, rng, slots, steps, dtype, kind, window, sinks):
    """`steps` decode steps of several layers through the cache; every output
    against the reference."""
    cos, sin = _tables(4096, 64)
    for _ in range(steps):
        rows = c.step(slots, [1] * len(slots))
        for layer in range(c.layers):
            x = _rand(rng, len(slots), 8, 128, dtype=dtype)
            q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
            qr = c.append(layer, rows, k, v, q=q, cos=cos, sin=sin)
            out = c.attend(layer, rows, qr, window=window, sinks=sinks)
            kk, vv = (_np(t) for t in c.read(layer, rows))
            for i, s in enumerate(slots):
                hk, hv = held[layer][s]
                held[layer][s] = (np.concatenate([hk, kk[i:i + 1]]), np.concatenate([hv, vv[i:i + 1]]))
                want, mag = ref.attend(_np(qr[i:i + 1]), *held[layer][s], [c.length(s) - 1], window, sinks)
                tol = ref.attend_tolerance(want, mag, _eps(dtype), kind == "q4")
                assert (np.abs(_np(out[i:i + 1]) - want) <= tol).all()
    c.check()


@pytest.mark.parametrize("kind,dtype", [("bf16", "bf16"), ("q4", "bf16"), ("q4", "f16")])
def test_a_whole_session(kind, dtype):
    """Prefill, decode, fork, decode both, evict, release, compact, decode."""
    rng = np.random.default_rng(20)
    window, sinks = 150, 4
    c = _cache(kind, 128, 2, layers=2, n_pages=24, max_slots=4, max_pages=12)
    c.open(0)
    c.open(1)
    rows = c.step([1, 0], [201, 330])
    held = [{}, {}]
    for layer in range(2):
        x = _rand(rng, 531, 8, 128, dtype=dtype)
        c.append(layer, rows, x[:, 4:6], x[:, 6:])
        k, v = (_np(t) for t in c.read(layer, rows))
        held[layer] = {1: (k[:201], v[:201]), 0: (k[201:], v[201:])}
        out = c.attend(layer, rows, x[:, :4], window=window, sinks=sinks)
        for s, a, n in ((1, 0, 201), (0, 201, 330)):
            want, mag = ref.attend(_np(x[a:a + n, :4]), *held[layer][s], range(n), window, sinks)
            assert (np.abs(_np(out[a:a + n]) - want) <= ref.attend_tolerance(want, mag, _eps(dtype), kind == "q4")).all()
    _decode_model(c, held, rng, [0, 1], 3, dtype, kind, window, sinks)
    c.fork(0, [2, 3])
    for layer in range(2):
        held[layer][2] = held[layer][3] = held[layer][0]
    _decode_model(c, held, rng, [3, 0, 2], 4, dtype, kind, window, sinks)
    for s in (0, 2, 3):
        assert c.evict(s, window, sinks) > 0
    c.release(1, 2)
    assert c.compact() < 24
    _decode_model(c, held, rng, [0, 3], 66, dtype, kind, window, sinks)


@pytest.mark.parametrize("kind", ["bf16", "q4"])
def test_a_captured_decode_step_follows_the_positions(kind):
    c, held = _filled(kind, "bf16", [1200, 300], seed=15)
    c.reserve(0, 1220), c.reserve(1, 320)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    rows = c.rows(t([0, 1]), t([1200, 300]))
    q, k, v = (_rand(np.random.default_rng(i), 2, h, 128) for i, h in enumerate((4, 2, 2)))
    out = torch.zeros_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.attend(0, _seq_rows(c, [0, 1], [1, 1], [1200, 300]), q, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for w in (0, 500):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.append(0, rows, k, v)
            c.attend(0, rows, q, window=w, sinks=3, out=out)
        graphs.append((g, w))
    for step in range(6):
        g, w = graphs[step % 2]
        gen = np.random.default_rng(100 + step)
        for x in (q, k, v):
            x.copy_(_rand(gen, *x.shape))
        g.replay()
        c.check()
        pos = (1200 + step, 300 + step)
        for i in range(2):
            kk, vv = _np(k[i:i + 1]), _np(v[i:i + 1])
            if kind == "q4":
                kk, vv = ref.quantise(kk)[0], ref.quantise(vv)[0]
            held[i] = (np.concatenate([held[i][0], kk]), np.concatenate([held[i][1], vv]))
            want, mag = ref.attend(_np(q[i:i + 1]), *held[i], [pos[i]], w, 3)
            assert (np.abs(_np(out[i:i + 1]) - want) <= ref.attend_tolerance(want, mag, _eps("bf16"), kind == "q4")).all()
        rows.advance()


@pytest.mark.parametrize("kind", ["bf16", "q4"])
def test_two_streams_and_two_graphs_at_the_same_time(kind):
    c, _ = _filled(kind, "bf16", [9000, 8000], seed=16)
    q = [_rand(np.random.default_rng(i), 1, 4, 128) for i in range(2)]
    rows = [_seq_rows(c, [i], [1], [n]) for i, n in ((0, 9000), (1, 8000))]
    want = [c.attend(0, rows[i], q[i]).clone() for i in range(2)]
    outs = [[torch.zeros_like(q[i]) for _ in range(30)] for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for r in range(30):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                c.attend(0, rows[i], q[i], out=outs[i][r])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in outs[i])
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for r in range(30):
                c.attend(0, rows[i], q[i], out=outs[i][r])
        graphs.append(g)
    for i in range(2):
        for o in outs[i]:
            o.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in outs[i])


@pytest.mark.parametrize("kind", ["bf16", "q4"])
def test_one_workspace_for_calls_of_many_shapes(kind):
    """A workspace made for the largest call serves the smaller ones, in any order."""
    c, held = _filled(kind, "bf16", [700, 400, 90], seed=17)
    for heads, most in ((4, 5), (4, 8), (4, 9), (4, 300), (2, 16)):
        ws = c.workspace(heads, 3, most)
        for counts in ([1, 1, 1], [most, 2, 1], [3, 1, 4], [min(most, 90)] * 3, [1, 1, 1]):
            _check_attend(c, held, kind, "bf16", counts, [700, 400, 90], heads, workspace=ws)
        assert not bool(ws[:PKG._lib.CACHE_WORKSPACE_ZERO].any())


@pytest.mark.parametrize("kind", ["bf16", "q4"])
def test_a_hidden_weight_of_a_large_value_leaves_the_small_ones_alone(kind):
    """Values that differ by 2^24 between positions, the large ones with weights
    that are nearly 0: the small ones keep their digits."""
    rng = np.random.default_rng(18)
    n, dim, heads = 200, 64, 2
    c = _cache(kind, dim, 1, max_slots=1)
    c.open(0)
    rows = c.step([0], [n])
    k, v = _rand(rng, n, 1, dim, scale=0.1), _rand(rng, n, 1, dim, scale=2.0 ** -10)
    q = torch.ones(n, heads, dim, dtype=torch.bfloat16, device="cuda")
    v[::7] *= 2.0**24
    k[::7] = -4.0  # scores of -32 and about 0
    c.append(0, rows, k, v)
    kk, vv = (ref.quantise(_np(k))[0], ref.quantise(_np(v))[0]) if kind == "q4" else (_np(k), _np(v))
    _check_attend(c, [(kk, vv)], kind, "bf16", [1], [n], heads, q=q[:1])
    _check_attend(c, [(kk, vv)], kind, "bf16", [n - 20], [n], heads, q=q[:n - 20])


def test_calls_that_would_race_are_refused():
    import ctypes as C

    c = _cache("bf16", 64, 1, n_pages=8, max_slots=4, max_pages=2)
    ia = lambda *v: (C.c_int32 * len(v))(*v)
    before = c.pool.clone()
    lib, at = PKG.load_library(), C.byref(c._c)
    for src, dst in (((0, 1), (2, 2)), ((0, 1), (1, 2))):
        assert lib.fmd_cache_copy_pages(at, 2, ia(*src), ia(*dst), None) == PKG._lib.FMD_EINVAL
    for src, dst, page in (((0, 0), (2, 2), (3, 4)), ((0, 1), (1, 2), (3, 4)), ((0, 0), (1, 2), (3, 3))):
        assert lib.fmd_cache_fork(at, 2, ia(*src), ia(*dst), ia(5, 70), ia(*page), None, None) == PKG._lib.FMD_EINVAL
    c.open(0)
    rows = c.step([0], [1])
    q = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(PKG.FmdError):
        c.attend(0, rows, q, out=q)
    # one row or one head for all of an output, but not of an input
    c.open(1)
    rows = c.step([0, 1], [1, 1])
    q, kv = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros_like(before[:256]).view(torch.bfloat16)
    kv = kv[:64].expand(2, 1, 64)
    for out in (q[:1].clone().expand(2, 2, 64), q[:, :1].clone().expand(2, 2, 64)):
        with pytest.raises(PKG.FmdError):
            c.attend(0, rows, q, out=out)
        with pytest.raises(PKG.FmdError):
            c.append(0, rows, kv, kv, q=q, q_out=out)
    torch.cuda.synchronize()
    assert torch.equal(c.pool, before)
    kv = _rand(np.random.default_rng(0), 64).expand(2, 1, 64)
    assert torch.equal(c.append(0, rows, kv, kv, q=kv.expand(2, 2, 64)), kv.expand(2, 2, 64))
    c.check()
    for s in (0, 1):
        assert torch.equal(_values(c, s, 0)[0].to(torch.bfloat16)[-1], kv[0])


def test_large_offsets_in_a_long_pool():
    """A pool above 4 GB: pages whose byte and element offsets pass 32 bits."""
    heads, dim, n_pages = 8, 128, 20000
    c = PKG.PagedCache(1, heads, dim, n_pages, 2, 8, kind="bf16",
                       pool=torch.empty(n_pages * 2 * heads * 16384, dtype=torch.uint8, device="cuda"),
                       page_table=torch.full((2, 8), -1, dtype=torch.int32, device="cuda"),
                       slots=[(0, [19999, 3, 19998], 0)])
    c._upload(0, 0)
    rows = c.step([0], [150])
    rng = np.random.default_rng(0)
    k, v, q = _rand(rng, 150, heads, dim), _rand(rng, 150, heads, dim), _rand(rng, 150, 2 * heads, dim)
    c.append(0, rows, k, v)
    out = c.attend(0, rows, q)
    one = c.attend(0, _seq_rows(c, [0], [1], [150]), q[149:])
    c.check()
    want, mag = ref.attend(_np(q[140:]), _np(k), _np(v), range(140, 150))
    tol = ref.attend_tolerance(want, mag, _eps("bf16"), False)
    assert (np.abs(_np(out[140:]) - want) <= tol).all() and (np.abs(_np(one) - want[9:]) <= tol[9:]).all()
