"""Which elements two strided row buffers share (`csrc/fmd_views.h`), compiled on
the host and held against the sets of elements themselves."""

from __future__ import annotations

import random
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "fast-moss-diarization_b200" / "csrc"
HARNESS = r"""
#include <cstdio>
#include "fmd_views.h"
// a line per pair of views "at row head rows heads dim" twice; prints whether the first overlaps itself
// and whether they meet
int main() {
  fmd::HeadRows v[2];
  for (;;) {
    for (auto& w : v) {
      unsigned long long at;
      long long f[5];
      if (std::scanf("%llu %lld %lld %lld %lld %lld", &at, f, f + 1, f + 2, f + 3, f + 4) != 6) return 0;
      w = fmd::HeadRows{at, f[0], f[1], f[2], f[3], f[4]};
    }
    std::printf("%d %d\n", v[0].overlaps(), fmd::meet(v[0], v[1]));
  }
}
"""


@pytest.fixture(scope="module")
def views(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    d = tmp_path_factory.mktemp("views")
    (d / "views.cc").write_text(HARNESS)
    subprocess.run([cxx, "-O1", "-std=c++17", "-I", str(CSRC), str(d / "views.cc"), "-o", str(d / "views")], check=True)

    def run(pairs):
        text = "".join(" ".join(map(str, a + b)) + "\n" for a, b in pairs)
        out = subprocess.run([str(d / "views")], input=text, capture_output=True, text=True, check=True).stdout
        return [tuple(x == "1" for x in line.split()) for line in out.splitlines()]

    return run


def _elements(v):
    at, row, head, rows, heads, dim = v
    return [at // 2 + i * row + j * head + d for i in range(rows) for j in range(heads) for d in range(dim)]


def test_layouts_that_programs_use(views):
    d = 64
    fused = lambda first, heads: (4096 + 2 * first * d, 12 * d, d, 5, heads, d)
    q, k, v = fused(0, 4), fused(4, 4), fused(8, 4)
    turned = (4096, d, 5 * d, 5, 4, d)           # heads outermost
    padded = (4096, d + 8, 5 * (d + 8), 5, 4, d)
    inner = lambda i: (4096 + 2 * i * d, 12 * d, 3 * d, 5, 4, d)  # q, k, v of a head side by side
    fine = [(q, k), (q, v), (k, v), (turned, (90000, *turned[1:])), (padded, (90000, *padded[1:])),
            (inner(0), inner(1)), (inner(2), inner(0))]
    assert views(fine) == [(False, False)] * len(fine)
    bad = [(q, q), (q, (q[0] + 16, *q[1:])), (q, (q[0] + 2 * 12 * d, *q[1:])), (k, fused(3, 2)), (inner(0), fused(3, 1))]
    assert views(bad) == [(False, True)] * len(bad)
    itself = [(4096, 12 * d, 8, 5, 4, d), (4096, d // 2, 5 * d, 5, 4, d), (4096, 2 * d, d, 5, 4, d), (4096, 0, d, 2, 1, d),
              (4096, d, 0, 1, 2, d)]
    assert [s for s, _ in views([(a, a) for a in itself])] == [True] * len(itself)
    one = [(4096, 0, d, 1, 4, d), (4096, 4 * d, 0, 5, 1, d), (4096, 0, 0, 1, 1, d)]
    assert [s for s, _ in views([(a, a) for a in one])] == [False] * len(one)


def test_against_the_elements(views):
    rng = random.Random(0)
    pairs = []
    for _ in range(4000):
        row, head = 8 * rng.randint(0, 30), 8 * rng.randint(0, 30)
        a = (4096, row, head, rng.randint(1, 6), rng.randint(1, 6), 16)
        row2 = row if rng.random() < 0.7 else 8 * rng.randint(0, 30)
        b = (4096 + 16 * rng.randint(-60, 60), row2, rng.choice([head, 8 * rng.randint(0, 30)]), a[3], rng.randint(1, 6), 16)
        pairs.append((a, b))
    exact = missed = 0
    for (a, b), (itself, shared) in zip(pairs, views(pairs)):
        ea, eb = _elements(a), _elements(b)
        assert itself == (len(set(ea)) < len(ea)), a
        real = bool(set(ea) & set(eb))
        if a[1] == b[1] or a[3] == 1:
            assert shared == real, (a, b)
            exact += 1
        else:  # never missed; refused where the ranges meet
            assert shared or not real, (a, b)
            missed += shared and not real
    assert exact > 2000 and missed < 800


def test_strides_beyond_64_bits_of_product(views):
    big = 2**62
    assert views([((4096, big, 64, 2**31 - 1, 4, 64), (4096, big, 64, 2**31 - 1, 4, 64))]) == [(False, True)]
