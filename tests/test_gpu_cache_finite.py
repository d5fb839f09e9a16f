"""The attention tests of test_gpu_cache once more, under a comparison that a NaN
does not pass."""

from __future__ import annotations

import inspect
import itertools

import pytest

import cache_ref as ref
import test_gpu_cache as base

pytestmark = pytest.mark.gpu


def _cases(test):
    """The keyword arguments of every case of a parametrised test."""
    axes = []
    for mark in getattr(test, "pytestmark", ()):
        if mark.name == "parametrize":
            names = [n.strip() for n in mark.args[0].split(",")]
            axes.append([dict(zip(names, v if len(names) > 1 else (v,))) for v in mark.args[1]])
    return [{k: v for part in case for k, v in part.items()} for case in itertools.product(*axes)]


TESTS = [f for name, f in vars(base).items() if name.startswith("test_") and "_check_attend(" in inspect.getsource(f)]


@pytest.mark.parametrize("test", TESTS, ids=lambda f: f.__name__[5:])
def test_outputs_are_finite(test, monkeypatch):
    monkeypatch.setattr(base, "_check_attend", ref.finite(base._check_attend))
    for case in _cases(test):
        test(**case)
