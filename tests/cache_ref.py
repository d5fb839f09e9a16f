"""Plain restatement of the paged-cache operators in 64 bits (numpy), for the
cache tests: storage, norms and rotation, windowed attention."""

from __future__ import annotations

import math

import numpy as np

PAGE = 64


def quantise(x):
    """(..., D) values -> (what the 4-bit cache holds of them, the scales)."""
    b = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 32)
    at = np.argmax(np.abs(b), -1)[..., None]
    m = np.clip(np.take_along_axis(b, at, -1), -65504.0, 65504.0)
    code = np.clip(np.floor(-8 * b / np.where(m == 0, 1.0, m) + 8.5), 0, 15)
    d = (m / -8).astype(np.float16).astype(np.float64)
    return ((code - 8) * d).reshape(x.shape), d[..., 0]


def norm_rotate(x, w=None, eps=1e-6, cos=None, sin=None, interleaved=False):
    """(rows, heads, D) in 64 bits; cos / sin: (rows, pairs)."""
    x = np.array(x, np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)
    if cos is not None:
        half = cos.shape[-1]
        a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
        c, s = np.asarray(cos, np.float64)[:, None], np.asarray(sin, np.float64)[:, None]
        u, v = x[..., a].copy(), x[..., b].copy()
        x[..., a], x[..., b] = u * c - v * s, v * c + u * s
    return x


def attend(q, k, v, pos, window=0, sinks=0, scale=None):
    """q (n, H, D) at positions pos, k / v (L, Hkv, D). Returns the output and
    sum_j p_j |v_j|, the magnitude that roundings of p and v scale with."""
    n, heads, dim = q.shape
    group = heads // k.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    out, mag = np.zeros(q.shape), np.zeros(q.shape)
    for i in range(n):
        j = np.arange(pos[i] + 1)
        if window:
            j = j[(j > pos[i] - window) | (j < sinks)]
        for h in range(heads):
            s = k[j, h // group] @ q[i, h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h] = p @ v[j, h // group]
            mag[i, h] = p @ np.abs(v[j, h // group])
    return out, mag


def append_tolerance(want, rows_max, eps):
    """One rounding to a type of machine epsilon `eps` (half a step, eps / 2 of
    the value; 2^-25 for f16 subnormals), and f32 arithmetic: a mean of up to
    128 squares, a product chain and a two-term sum, at most 2^-19 of the
    largest value of the row."""
    return eps / 2 * np.abs(want) + 2.0 ** -19 * rows_max + 2.0 ** -25


def attend_tolerance(want, mag, eps, q4):
    """The output's rounding (eps / 2 of the value), each probability's (eps / 2
    of its term; in 4 bits, where products run in f16, half a step of f16,
    2^-11: a step is 2^-10 of a value just above a power of two), in 4 bits also
    each value's product with its scale (2^-11 again), and f32 arithmetic: scores
    of magnitude up to 2^5 with 2^-20 of it wrong move p by 2^-15, sums and the
    hardware exponential by less: 2^-14 of the magnitude in all."""
    terms = 2 * 2.0 ** -11 if q4 else eps / 2
    return eps / 2 * np.abs(want) + (terms + 2.0 ** -14) * mag + 2.0 ** -25


def finite(check):
    """`check` (a comparison that returns the tensor it looked at), which a NaN or
    an infinity does not pass: |NaN - x| > tol is false."""
    def strict(*args, **kw):
        out = check(*args, **kw)
        values = out.detach().double().cpu().numpy()
        assert np.isfinite(values).all(), np.argwhere(~np.isfinite(values))[:4].tolist()
        return out

    return strict
