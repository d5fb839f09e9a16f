"""Calls of the paged-cache operators as programs make them: from several host
threads, in graphs of several shapes, with empty batches and odd outputs."""

from __future__ import annotations

import ctypes as C
import threading

import numpy as np
import pytest

import cache_ref as ref
from conftest import PKG
from test_gpu_cache import _eps, _filled, _np, _rand, _seq_rows

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,dim", [("bf16", 128), ("q4", 128), ("f16", 64)])
def test_two_host_threads_with_different_shapes(kind, dim):
    """Each thread has a cache and a stream of its own; their calls differ in the
    query heads of a kv head, and so in the shared memory that they ask for."""
    dtype = "f16" if kind == "f16" else "bf16"
    jobs, failed = [], []
    for i, group in enumerate((1, 2, 4, 8)):
        c, _ = _filled(kind, dtype, [40 + i], dim=dim, seed=i)
        q = _rand(np.random.default_rng(i), 1, 2 * group, dim, dtype=dtype)
        rows = _seq_rows(c, [0], [1], [40 + i])
        out = torch.zeros_like(q)
        # the C entry with its arguments at hand, so that the threads are in it most of the time
        args = PKG._lib.CacheAttendArgs(q.data_ptr(), out.data_ptr(), *q.stride()[:2], *out.stride()[:2], dim ** -0.5,
                                        c._dtype(q, "q"), q.shape[1], 0, 0)
        ws = c.workspace(q.shape[1], 1)
        call = (c._ref, 0, c._rows_c(rows, 1), C.byref(args), ws.data_ptr(), ws.numel(), c._status_at)
        jobs.append((c, call, out, c.attend(0, rows, q).clone(), (q, args, ws, rows)))
    torch.cuda.synchronize()
    start = threading.Barrier(len(jobs))

    def work(c, call, out, want, keep):
        stream = torch.cuda.Stream()
        torch.cuda.set_device(0)
        start.wait()
        codes = {c.lib.fmd_cache_attend(*call, stream.cuda_stream) for _ in range(10000)}
        stream.synchronize()
        if codes != {PKG._lib.FMD_OK} or not torch.equal(out, want):
            failed.append((codes, keep[0].shape))

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for c, *_ in jobs:
        c.check()
    assert not failed, failed


@pytest.mark.parametrize("kind", ["bf16", "q4"])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_graph_of_calls_of_many_shapes(kind, dim):
    """Calls that ask for different amounts of shared memory, captured into one
    graph, with others made before it is replayed."""
    lengths = [200, 90]
    c, _ = _filled(kind, "bf16", lengths, dim=dim)
    shapes = [(heads, n) for heads in (2, 8, 16, 32) for n in (1, 2, 40)]
    calls = [(_seq_rows(c, [0, 1], [n, n], lengths),
              _rand(np.random.default_rng(heads + n), 2 * n, heads, dim)) for heads, n in shapes]
    want = [c.attend(0, rows, q).clone() for rows, q in calls]
    outs = [torch.zeros_like(q) for _, q in calls]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for (rows, q), out in zip(calls, outs):
            c.attend(0, rows, q, out=out)
    for rows, q in reversed(calls):
        c.attend(0, rows, q)
    for _ in range(2):
        g.replay()
    c.check()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("kind", ["bf16", "q4"])
def test_steps_and_forks_after_replayed_steps(kind):
    """A captured step is replayed; the cache's books, told by `advance`, then serve
    a fork and further steps, and nothing that was written is lost."""
    c = PKG.PagedCache(1, 2, 128, 12, 3, 4, kind=kind)
    c.open(0)
    rng = np.random.default_rng(3)
    held = [np.zeros((0, 2, 128)), np.zeros((0, 2, 128))]

    def keep(k, v):
        for i, x in enumerate((k, v)):
            x = _np(x)
            held[i] = np.concatenate([held[i], ref.quantise(x)[0] if kind == "q4" else x])

    def check(slot, n=1):
        end = c.length(slot)
        q = _rand(rng, n, 4, 128)
        out = c.attend(0, _seq_rows(c, [slot], [n], [end]), q)
        c.check()
        want, mag = ref.attend(_np(q), held[0][:end], held[1][:end], range(end - n, end))
        assert (np.abs(_np(out) - want) <= ref.attend_tolerance(want, mag, _eps("bf16"), kind == "q4")).all()

    rows = c.step([0], [60])
    k, v = _rand(rng, 60, 2, 128), _rand(rng, 60, 2, 128)
    c.append(0, rows, k, v)
    keep(k, v)
    k, v = _rand(rng, 1, 2, 128), _rand(rng, 1, 2, 128)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    moving = c.rows(t([0]), t([60]))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.append(0, moving, k, v)
        moving.advance()
    for _ in range(9):  # over the end of the first page
        k.copy_(_rand(rng, 1, 2, 128))
        v.copy_(_rand(rng, 1, 2, 128))
        c.advance([0])
        g.replay()
        keep(k, v)
    assert c.length(0) == 69
    check(0)
    check(0, 30)
    c.fork(0, [1])
    assert c.length(1) == 69
    check(1)
    rows = c.step([0], [2])
    assert rows.pos0.tolist() == [69]
    k, v = _rand(rng, 2, 2, 128), _rand(rng, 2, 2, 128)
    c.append(0, rows, k, v)
    keep(k, v)
    check(0)
    check(1)


@pytest.mark.parametrize("kind", ["bf16", "q4"])
@pytest.mark.parametrize("count", [1, 20])
def test_outputs_that_share_elements_are_refused_and_views_of_one_buffer_are_not(kind, count):
    lengths = [100, 60]
    c, held = _filled(kind, "bf16", lengths, kv_heads=2)
    n, d = 2 * count, 128
    rows = _seq_rows(c, [0, 1], [count] * 2, lengths)
    x = _rand(np.random.default_rng(0), n + 1, 16, d)
    q, k, v, out = x[:n, :4], x[:n, 4:6], x[:n, 6:8], x[:n, 8:12]
    big = torch.zeros(64 * n * d, dtype=torch.bfloat16, device="cuda")
    before, pool = x.clone(), c.pool.clone()
    bad = [x[:n, 2:6], x[:n, 3:7], big.as_strided((n, 4, d), (8 * d, d // 2, 1)), big.as_strided((n, 4, d), (8 * d, 8, 1)),
           x.flatten()[8:8 + n * 16 * d].view(n, 16, d)[:, :4]]
    if n > 2:
        bad += [big.as_strided((n, 4, d), (2 * d, d, 1)), big.as_strided((n, 4, d), (8, n * d, 1)), x[1:, :4]]
    for o in bad:
        with pytest.raises(PKG.FmdError) as e:
            c.append(0, rows, k, v, q=q, q_out=o)
        assert e.value.status == PKG._lib.FMD_EINVAL
    for o in bad + [q]:
        with pytest.raises(PKG.FmdError) as e:
            c.attend(0, rows, q, out=o)
        assert e.value.status == PKG._lib.FMD_EINVAL
    torch.cuda.synchronize()
    assert torch.equal(x, before) and torch.equal(c.pool, pool) and not bool(big.any())
    # views of one buffer beside one another, and heads outermost
    want = c.attend(0, rows, q.clone())
    c.attend(0, rows, q, out=out)
    turned = torch.zeros(4, n, d, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    c.attend(0, rows, q, out=turned)
    assert torch.equal(out, want) and torch.equal(turned, want)
    c.append(0, rows, k, v, q=q, q_out=out)
    c.append(0, rows, k, v, q=q, q_out=q)
    c.check()
    assert torch.equal(out, before[:n, :4]) and torch.equal(q, before[:n, :4])


@pytest.mark.parametrize("kind", ["bf16", "q4"])
def test_calls_without_rows_do_nothing(kind):
    c, _ = _filled(kind, "bf16", [70, 5])
    pool = c.pool.clone()
    for rows in (c.step([0, 1], [0, 0]), c.step([], [])):
        k, q = _rand(np.random.default_rng(0), 0, 2, 128), _rand(np.random.default_rng(0), 0, 4, 128)
        assert c.append(0, rows, k, k) is None
        assert c.append(0, rows, k, k, q=q).shape == q.shape
        assert c.attend(0, rows, q).shape == q.shape and c.attend(0, rows, q, window=3, out=q).shape == q.shape
        assert [t.shape for t in c.read(0, rows)] == [k.shape, k.shape]
    c.check()
    assert torch.equal(c.pool, pool) and c.length(0) == 70


def test_check_waits_for_every_stream():
    c, _ = _filled("bf16", "bf16", [100])
    q = _rand(np.random.default_rng(0), 1, 4, 128)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    bad = c.rows(t([17]), t([99]))
    out = torch.zeros_like(q)
    busy = torch.ones(8192, 8192, device="cuda")
    side, then = torch.cuda.Stream(), torch.zeros_like(busy)
    with torch.cuda.stream(side):  # what these allocate is there before the stream is busy
        torch.mm(busy, busy, out=then)
        c.attend(0, _seq_rows(c, [0], [1], [100]), q, out=out)
    c.check()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            torch.mm(busy, busy, out=then)
        c.attend(0, bad, q, out=out)
    with pytest.raises(PKG.FmdError) as e:
        c.check()
    assert e.value.status == PKG._lib.FMD_EINVAL
    c.check()


@pytest.mark.parametrize("e", [-133, -126, 110, 121, 125, 126, 127])
@pytest.mark.parametrize("count", [1, 40])
def test_queries_at_the_ends_of_bf16_over_4_bits(e, count):
    """Queries of up to 1.5 x 2^127 whose scores are finite: their scaling to f16 stays
    within f32 as well. One key meets them; the rest scores 0."""
    dim, n = 128, 100
    c = PKG.PagedCache(1, 1, dim, 3, 1, 2, kind="q4")
    c.open(0)
    rng = np.random.default_rng(4)
    k, v = torch.zeros(n, 1, dim, dtype=torch.bfloat16, device="cuda"), _rand(rng, n, 1, dim)
    k[20, 0, 0] = 2.0 ** -10
    c.append(0, c.step([0], [n]), k, v)
    q = torch.zeros(count, 2, dim, dtype=torch.bfloat16, device="cuda")
    q[:, :, 0] = 1.5 * 2.0 ** e
    out = c.attend(0, _seq_rows(c, [0], [count], [n]), q)
    c.check()
    kk, vv = ref.quantise(_np(k))[0], ref.quantise(_np(v))[0]
    want, mag = ref.attend(_np(q), kk, vv, range(n - count, n))
    assert (np.abs(_np(out) - want) <= ref.attend_tolerance(want, mag, _eps("bf16"), True)).all()


@pytest.mark.parametrize("kind", ["bf16", "q4"])
def test_max_rows_is_only_a_bound(kind):
    """A caller that does not know the longest sequence may say the largest number."""
    lengths = [90, 70, 300, 40] * 8
    c, held = _filled(kind, "bf16", lengths)
    counts = [40, 1, 33, 0] * 8
    q = _rand(np.random.default_rng(0), sum(counts), 4, 128)
    want = c.attend(0, _seq_rows(c, range(32), counts, lengths), q)
    for most in (1000, 2**31 - 1):
        assert torch.equal(c.attend(0, _seq_rows(c, range(32), counts, lengths, max_rows=most), q), want)
    c.check()


def test_read_outputs_that_overlap_are_refused():
    c, _ = _filled("bf16", "bf16", [30])
    rows = _seq_rows(c, [0], [30], [30])
    want = c.read(0, rows)
    n = 30 * 2 * 128
    both = torch.zeros(2 * n, device="cuda")
    view = lambda at: both[at:at + n].view(30, 2, 128)
    for a, b in ((view(0), view(0)), (view(0), view(4)), (view(n - 4), view(0))):
        with pytest.raises(PKG.FmdError) as e:
            c.read(0, rows, k_out=a, v_out=b)
        assert e.value.status == PKG._lib.FMD_EINVAL
    assert not bool(both.any())
    got = c.read(0, rows, k_out=view(n), v_out=view(0))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("kind,dtype", [("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("dim,group", [(128, 2), (64, 16)])
def test_decode_from_16_bits_loses_no_more_than_the_outputs_rounding(kind, dtype, dim, group):
    """Root-mean-square error against 64 bits, beside that of rounding the exact output
    once. Probabilities of one 16-bit term would add as much again; two terms leave
    2^-17 of each or less, and f32 sums and the exponential 2^-17 or so, a hundredth of
    f16's 2^-12 (mean): 1.1 allows ten times that."""
    n = 4000
    c, held = _filled(kind, dtype, [n], dim=dim, seed=21)
    q = _rand(np.random.default_rng(22), 1, 2 * group, dim, dtype=dtype)
    out = c.attend(0, _seq_rows(c, [0], [1], [n]), q)
    c.check()
    want, _ = ref.attend(_np(q), *held[0], [n - 1])
    once = _np(torch.from_numpy(want).to(q.dtype))
    rms = lambda x: np.sqrt((x * x).mean())
    assert rms(_np(out) - want) <= 1.1 * rms(once - want)
