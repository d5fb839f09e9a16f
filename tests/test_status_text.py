"""The words for a status that kernels set (`csrc/fmd_status.h`), compiled on the host."""

from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

from conftest import PKG

CSRC = Path(__file__).resolve().parents[1] / "fast-moss-diarization_b200" / "csrc"
L = PKG._lib
HARNESS = r"""
#include <cstdio>
#include "fmd_status.h"
int main() {
  int status, site;
  while (std::scanf("%d %d", &status, &site) == 2) std::printf("%s\n", fmd::device_status_text(status, site).c_str());
  std::printf("%s\n%s\n", fmd::refusal_text("").c_str(), fmd::refusal_text("out of memory").c_str());
}
"""


def test_every_status_is_named_for_what_it_is(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    (tmp_path / "s.cc").write_text(HARNESS)
    subprocess.run([cxx, "-O1", "-std=c++17", "-I", str(CSRC), str(tmp_path / "s.cc"), "-o", str(tmp_path / "s")], check=True)
    asked = [(L.FMD_EINVAL, 0), (L.FMD_EOVERFLOW, 0), (L.FMD_EIO, 0), (L.FMD_ETIMEDOUT, 10), (L.FMD_ETIMEDOUT, 99), (-7, 3)]
    out = subprocess.run([str(tmp_path / "s")], input="".join(f"{a} {b}\n" for a, b in asked), capture_output=True, text=True,
                         check=True).stdout.splitlines()
    for text, words in zip(out, ("slot or page", "position", "no finite logit", "wait gave up in k_cache_chunk",
                                 "wait gave up in ?", "unknown", "decode projection was not launched",
                                 "a cache operator was not launched: out of memory")):
        assert words in text
        assert ("wait gave up" in text) == ("wait gave up" in words)
    assert len(out) == len(asked) + 2


def test_every_site_has_a_name():
    """The names follow `TimeoutSite`."""
    sites = re.findall(r"kSite\w+ = (\d+)", (CSRC / "fmd_common.cuh").read_text())
    names = re.search(r"kSites\[\] = \{([^}]*)\}", (CSRC / "fmd_status.h").read_text()).group(1).count('"') // 2
    assert [int(s) for s in sites] == list(range(1, names))


def test_the_runtime_uses_them():
    src = (CSRC / "fmd_runtime.cu").read_text()
    assert "device_status_text(st[0], st[1])" in src and "refusal_text(h->cache_refused)" in src
