"""A decoder on the cache operators after a reported device status: the status word
and the operators' counters are cleared on the steps' own stream, before the next step."""

from __future__ import annotations

import importlib
import re
from pathlib import Path

import numpy as np
import pytest

from conftest import PKG, tiny_config

syn = importlib.import_module("fmd_b200.synthetic")


def test_what_a_report_clears_is_cleared_on_the_steps_stream():
    """The steps' stream is a non-blocking one: the legacy stream's work is not ordered with it."""
    src = (Path(__file__).resolve().parents[1] / "fast-moss-diarization_b200" / "csrc" / "fmd_runtime.cu").read_text()
    body = src[src.index("int sync_check("):]
    body = body[:body.index("\n}\n")]
    assert "cudaStreamCreateWithFlags(&h->stream, cudaStreamNonBlocking)" in src
    assert not re.search(r"cudaMemset\(", body) and body.count("cudaMemsetAsync(") == 2


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(kv="q4"), dict(kv="q4", window=40, sinks=2), dict(window=40)])
def test_steps_after_a_reported_timeout_are_what_they_were(kw):
    cfg = tiny_config()
    w = syn.make_weights(cfg, seed=5, norm_jitter=0.2)
    prompt = np.random.default_rng(5).standard_normal((150, cfg.hidden_size), dtype=np.float32)
    runs = []
    for report in (False, True):
        with PKG.Qwen3Decoder(cfg, "bf16") as dec:
            dec.load_weights(w)
            dec.reserve(2, 512, 256, **kw)
            dec.open_slot(0, 200)
            got = [dec.prefill([0], [prompt])[0]]
            for t in range(6):
                if report:
                    with pytest.raises(PKG.FmdError) as e:
                        dec.debug_wait_timeout(100)
                    assert e.value.status == PKG._lib.FMD_ETIMEDOUT
                got.append(dec.decode_step([0], [t + 3])[0])
            runs.append(got)
    assert all(np.array_equal(a, b) for a, b in zip(*runs))
