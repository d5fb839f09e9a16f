"""The decoder on a 4-bit cache, with a window and sinks, and with forked and
compacted slots (`fmd_kv_options`, `fmd_slot_fork`, `fmd_kv_compact`), against
the CPU oracle with the same cache and mask."""

from __future__ import annotations

import importlib

import numpy as np
import pytest

import cache_ref
from conftest import PKG, gpu_teacher_forced, rel_err, tiny_config

syn = importlib.import_module("fmd_b200.synthetic")
pytestmark = pytest.mark.gpu

LOGIT_RTOL = 2e-2


@pytest.fixture(scope="module")
def tiny_w():
    return syn.make_weights(tiny_config(), seed=11, norm_jitter=0.2)


def _decoder(w, prec="bf16", slots=4, tokens=4096, rows=256, **kw):
    d = PKG.Qwen3Decoder(tiny_config(), prec, device=0)
    d.load_weights(w)
    d.reserve(slots, tokens, rows, **kw)
    return d


def _oracle(w, prec, kv, window, sinks, accumulate="f32"):
    """The oracle with the cache's 4 bits and the window in its mask."""
    import torch

    from oracle import qwen3_ref as ref

    class Windowed(ref.Qwen3Ref):
        def _causal(self, q_offset, q_len, kv_len):
            m = super()._causal(q_offset, q_len, kv_len)
            if window:
                row = (q_offset + torch.arange(q_len)).repeat(self.cfg.kv_repeat)[:, None]
                key = torch.arange(kv_len)
                m = m.masked_fill((key <= row - window) & (key >= sinks), float("-inf"))
            return m

        def new_caches(self, batch, capacity):
            caches = super().new_caches(batch, capacity)
            if kv == "q4":
                for c in caches:
                    plain = c.append
                    c.append = lambda k, v, plain=plain: plain(*(
                        torch.from_numpy(cache_ref.quantise(t.numpy())[0].astype(np.float32)) for t in (k, v)))
            return caches

    return Windowed(ref.TextConfig(**tiny_config().oracle_kwargs()), w, prec, max_len=8192, accumulate=accumulate)


@pytest.mark.parametrize("prec", ["bf16", "f16", "int8_bf16"])
@pytest.mark.parametrize("kv,window,sinks", [("act", 70, 4), ("q4", 0, 0), ("q4", 100, 5)])
def test_logits_match_the_oracle(prec, kv, window, sinks, tiny_w):
    """Two codes of a value on their border differ by a whole step, so the 4-bit
    oracle parts from an equally valid evaluation of itself (sums in 64 bits) by
    more than the 16-bit one does; that distance is measured, and three times it
    is granted on top of the bar for 16 bits."""
    cfg = tiny_config()
    rng = np.random.default_rng(0)
    prompt = rng.standard_normal((300, cfg.hidden_size), dtype=np.float32)  # two passes, chunks of 256 and 44
    tokens = rng.integers(0, cfg.vocab_size, 12)

    def run(m):
        caches = m.new_caches(1, 400)
        return [m.logits(m.prefill(prompt[None], caches))[0, 0].numpy()] + [
            m.decode_step(int(t), caches).numpy() for t in tokens]

    want = run(_oracle(tiny_w, prec, kv, window, sinks))
    floor = 0.0
    if kv == "q4":
        floor = max(rel_err(a, b) for a, b in zip(run(_oracle(tiny_w, prec, kv, window, sinks, "f64")), want))
    with _decoder(tiny_w, prec, kv=kv, window=window, sinks=sinks) as dec:
        dec.open_slot(0, 400)
        lg, ids = dec.prefill([0], [prompt])
        got = [lg[0]]
        for t in tokens:
            lg, _ = dec.decode_step([0], [int(t)])
            got.append(lg[0])
    for g, r in zip(got, want):
        assert rel_err(g, r) < LOGIT_RTOL + 3 * floor, (rel_err(g, r), floor)


@pytest.mark.parametrize("prec", ["bf16", "int8"])
def test_the_4_bit_cache_holds_the_quantised_rows(prec, tiny_w):
    """Layer 0's keys and values do not depend on attention: the 4-bit pool
    holds exactly what quantising the 16-bit pool's rows gives, through prefill
    passes and decode steps, rounded to the activation dtype on the way out."""
    import torch

    cfg = tiny_config()
    rng = np.random.default_rng(1)
    prompts = [rng.standard_normal((n, cfg.hidden_size), dtype=np.float32) for n in (130, 65)]
    held = []
    for kv in ("act", "q4"):
        with _decoder(tiny_w, prec, kv=kv) as dec:
            for s, p in ((2, prompts[0]), (1, prompts[1])):
                dec.open_slot(s, 200)
            dec.prefill([2, 1], prompts)
            dec.decode_step([1, 2], [5, 9])
            held.append([dec.debug_kv(s, 0, 0, n) for s, n in ((2, 131), (1, 66))])
            if kv == "q4":
                mem = dec.memory_bytes()["kv_pool"]
            else:
                full = dec.memory_bytes()["kv_pool"]
    dt = torch.bfloat16 if prec == "bf16" else torch.float16
    for act, q4 in zip(*held):
        for a, b in zip(act, q4):
            want = torch.from_numpy(cache_ref.quantise(a)[0]).to(dt).double().numpy()
            assert np.array_equal(b, want)
    # 4.5 of 16 bits, and one of the two layers in 16 bits as staging
    assert mem == full * 9 // 32 + full // 2


def _alone(w, kw, prompt, tokens):
    """Logits of one sequence by itself."""
    with _decoder(w, **kw) as dec:
        dec.open_slot(0, len(prompt) + len(tokens))
        lg, _ = dec.prefill([0], [prompt])
        return [lg[0]] + [dec.decode_step([0], [t])[0][0] for t in tokens]


@pytest.mark.parametrize("kw", [dict(), dict(kv="q4"), dict(window=50, sinks=3), dict(kv="q4", window=90)])
@pytest.mark.parametrize("length", [100, 64, 1])
def test_forks_go_their_own_ways(kw, length, tiny_w):
    cfg = tiny_config()
    prompt = np.random.default_rng(2).standard_normal((length, cfg.hidden_size), dtype=np.float32)
    ways = {0: [3, 4, 5, 6], 1: [3, 9, 9, 9], 3: [7, 1, 2, 3]}
    with _decoder(tiny_w, **kw) as dec:
        before = dec.memory_bytes()
        dec.open_slot(0, length + 80)
        dec.prefill([0], [prompt])
        dec.fork_slot(0, 1, length + 4)
        dec.fork_slot(1, 3, length + 70)  # a fork of a fork
        assert dec.slot_len(3) == length
        got = {s: [] for s in ways}
        for step in range(4):
            for s in ways:  # one at a time, as in the runs to compare with
                got[s].append(dec.decode_step([s], [ways[s][step]])[0][0])
        with pytest.raises(PKG.FmdError) as e:
            dec.fork_slot(0, 1, length + 4)
        assert e.value.status == PKG._lib.FMD_EBUSY
        assert dec.memory_bytes() == before
    for s, tokens in ways.items():
        want = _alone(tiny_w, kw, prompt, tokens)[1:]
        assert all(np.array_equal(a, b) for a, b in zip(got[s], want)), s


@pytest.mark.parametrize("kw", [dict(), dict(kv="q4"), dict(kv="q4", window=90, sinks=2)])
def test_release_of_forks_and_compaction_keep_the_others(kw, tiny_w):
    cfg = tiny_config()
    rng = np.random.default_rng(3)
    a, b = (rng.standard_normal((n, cfg.hidden_size), dtype=np.float32) for n in (150, 70))
    # 7 pages of positions and one more a slot: page exhaustion is within reach
    with _decoder(tiny_w, slots=4, tokens=7 * 64, **kw) as dec:
        dec.open_slot(2, 192)
        dec.prefill([2], [a])
        dec.open_slot(0, 128)
        dec.prefill([0], [b])
        dec.fork_slot(2, 1, 192)          # shares 2 pages, takes 1
        dec.release_slot(2)               # its partial page is free again, the shared ones are not
        assert dec.compact_kv() == 5
        first = dec.decode_step([1], [3])[0][0]
        dec.fork_slot(1, 2, 192)
        dec.fork_slot(1, 3, 192)
        assert dec.compact_kv() == 7
        second = [dec.decode_step([s], [4])[0][0] for s in (3, 1, 2)]
        other = dec.decode_step([0], [8])[0][0]
        dec.release_slot(1)
        dec.release_slot(3)
        with pytest.raises(PKG.FmdError) as e:
            dec.open_slot(1, 10 * 64)
        assert e.value.status == PKG._lib.FMD_ENOMEM
        dec.open_slot(1, 6 * 64)          # 11 pages, 2 + 3 in use
        dec.release_slot(1)
        dec.release_slot(0)
        dec.release_slot(2)
        assert dec.compact_kv() == 0
        dec.open_slot(0, 11 * 64)         # every page is back
    want = _alone(tiny_w, kw, a, [3, 4])
    assert np.array_equal(first, want[1]) and all(np.array_equal(x, want[2]) for x in second)
    assert np.array_equal(other, _alone(tiny_w, kw, b, [8])[1])


@pytest.mark.parametrize("kw", [dict(kv="q4"), dict(window=100, sinks=4), dict(kv="q4", window=100, sinks=4)])
def test_the_engine_runs_on_them(kw, tiny_w):
    """Continuous batching with chunked prefill and refilled slots: every pick
    is the operator path's on the same stream, up to near-ties of its logits
    (two batch compositions round differently; in 4 bits a border code may flip)."""
    cfg = tiny_config()
    rng = np.random.default_rng(7)
    lens = [30, 100, 64, 1, 250, 177]
    budget = [6, 4, 10, 3, 5, 8]
    prompts = [rng.standard_normal((n, cfg.hidden_size), dtype=np.float32) for n in lens]
    with _decoder(tiny_w, slots=6, tokens=2048, **kw) as dec:
        eng = PKG.Engine(dec)
        out, stats = eng.generate(lens, budget, -1, np.concatenate(prompts), max_batch=3, prefill_chunk=100)
        assert stats.requests == 6 and stats.prefill_tokens == sum(lens)
        again, _ = eng.generate(lens, budget, -1, np.concatenate(prompts), max_batch=3, prefill_chunk=100)
        assert [o.tokens for o in out] == [o.tokens for o in again]
        logits = gpu_teacher_forced(dec, prompts, [o.tokens for o in out])
    ties = 0
    for o, lg in zip(out, logits):
        for s, tok in enumerate(o.tokens):
            gap = lg[s].max() - lg[s][tok]
            assert gap <= LOGIT_RTOL * np.abs(lg[s]).max(), (s, tok, gap)
            ties += tok != int(np.argmax(lg[s]))
    assert ties <= 4


def test_options_are_checked(tiny_w):
    d = PKG.Qwen3Decoder(tiny_config(), "bf16", device=0)
    d.load_weights(tiny_w)
    L = PKG._lib
    for args in ((1, 0, 0), (0, -1, 0), (4, 5, -1)):
        assert d.lib.fmd_kv_options(d.handle, *args) == L.FMD_EINVAL
    with pytest.raises(PKG.FmdError, match="kv must be"):
        d.reserve(2, 256, 64, kv="q8")
    d.reserve(2, 256, 64, kv="q4")
    assert d.lib.fmd_kv_options(d.handle, 0, 0, 0) == L.FMD_EBUSY
    for args, status in (((0, 1, 10), L.FMD_EINVAL), ((-1, 1, 10), L.FMD_EINVAL), ((0, 2, 10), L.FMD_EINVAL)):
        with pytest.raises(PKG.FmdError) as e:
            d.fork_slot(*args)
        assert e.value.status == status
    d.open_slot(0, 70)
    d.prefill([0], [np.zeros((66, tiny_config().hidden_size), np.float32)])
    for args, status in (((0, 0, 80), L.FMD_EBUSY), ((0, 1, 65), L.FMD_EINVAL), ((0, 1, 1 << 20), L.FMD_EOVERFLOW),
                         ((0, 1, 64 * 7), L.FMD_ENOMEM)):
        with pytest.raises(PKG.FmdError) as e:
            d.fork_slot(*args)
        assert e.value.status == status, args
    d.fork_slot(0, 1, 66)
    d.close()
