"""CPU oracle of the serving operators: E4M3 cache rows, decode over them, per-head norms with RoPE, 4-bit products.

TEST INFRASTRUCTURE ONLY, as ``oracle/gqa_oracle.py``.  Everything is float64 numpy written from the definitions:

* ``e4m3_row`` -- a row's values as the cache keeps them: the scale is the least power of two 2^e (e >= -126) with
  448 * 2^e >= the largest finite |x| (at most 1.875 * 2^127), each value the nearest multiple of the E4M3 step there
  (ties to even); infinities and NaN become NaN.
* ``decode`` -- softmax(scale * q K^T) V per query head, its natural-log sum, and the same average of |V|.
* ``norm_rope`` -- y = h / sqrt(mean(h^2) + eps) * w, pairs (2p, 2p + 1) rotated by position * base^(-2p / D).
* ``w4_matrix`` -- (c - 8) * scale of packed pairs of codes.

Pinned in ``tests/test_serving_oracle.py``.
"""
from __future__ import annotations

import numpy as np

TOP = 1.875 * 2.0**127


def e4m3_values() -> np.ndarray:
    """Value of every code 0..255 (bias 7, three fraction bits, no infinities; 0x7F and 0xFF are NaN)."""
    c = np.arange(256)
    sign, e, m = np.where(c & 128, -1.0, 1.0), (c >> 3) & 15, c & 7
    v = sign * np.where(e == 0, m * 2.0**-9, (1 + m / 8.0) * 2.0 ** (e - 7.0))
    v[(c & 127) == 127] = np.nan
    return v


def e4m3_row(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(codes' values, scale) of rows [..., D]."""
    x = np.asarray(x, dtype=np.float64)
    finite = np.isfinite(x)
    c = np.clip(np.where(finite, x, 0.0), -TOP, TOP)
    top = np.abs(c).max(-1)
    e = np.full(top.shape, -126)
    some = top > 0
    guess = np.floor(np.log2(np.where(some, top, 1.0) / 448.0)).astype(int)
    for d in (-1, 0, 1, 2):  # the least exponent that holds the row, whatever the logarithm rounded to
        cand = guess + 2 - (d + 1)
        e = np.where(some & (448.0 * 2.0 ** cand.astype(float) >= top), cand, e)
    e = np.maximum(e, -126)
    scale = 2.0 ** e.astype(float)
    v = c / scale[..., None]
    _, ve = np.frexp(v)
    step = 2.0 ** (np.maximum(ve - 1, -6) - 3.0)
    return np.where(finite, np.rint(v / step) * step, np.nan), scale


def stored(x: np.ndarray) -> np.ndarray:
    """Rows as the E4M3 cache gives them back."""
    v, s = e4m3_row(x)
    return v * s[..., None]


def decode(q, k, v, scale):
    """q [H_q, D] of one sequence against k, v [H_kv, L, D]: (o, lse, average of |V|)."""
    group = q.shape[0] // k.shape[0]
    if k.shape[1] == 0:
        return np.zeros(q.shape), np.full(q.shape[0], -np.inf), np.zeros(q.shape)
    s = scale * np.einsum("hd,hld->hl", q, np.repeat(k, group, 0))
    m = s.max(-1, keepdims=True)
    p = np.exp(s - m)
    total = p.sum(-1, keepdims=True)
    v = np.repeat(v, group, 0)
    o, a = (np.einsum("hl,hld->hd", p, t) / total for t in (v, np.abs(v)))
    return o, (m + np.log(total))[:, 0], a


def norm_rope(h, weight, eps, positions, base):
    """h [..., n, D] at positions [n]: (y, sum of the magnitudes that each y adds up); weight None: no norm, base 0: no
    rotation."""
    h = np.asarray(h, dtype=np.float64)
    if weight is not None:
        h = h / np.sqrt((h * h).mean(-1, keepdims=True) + eps) * weight
    if not base:
        return h, np.abs(h)
    d = h.shape[-1]
    angle = np.asarray(positions, dtype=np.float64)[:, None] * float(base) ** (-2.0 * np.arange(d // 2) / d)
    z = (h[..., 0::2] + 1j * h[..., 1::2]) * np.exp(1j * angle)
    a, b = np.abs(h[..., 0::2]), np.abs(h[..., 1::2])
    c, s = np.abs(np.cos(angle)), np.abs(np.sin(angle))
    y, mag = np.empty(h.shape), np.empty(h.shape)
    y[..., 0::2], y[..., 1::2] = z.real, z.imag
    mag[..., 0::2], mag[..., 1::2] = a * c + b * s, a * s + b * c
    return y, mag


def w4_matrix(codes, scales):
    """[rows, hidden] of codes [rows, hidden / 2] and scales [rows, hidden / group]."""
    c = np.empty((codes.shape[0], 2 * codes.shape[1]))
    c[:, 0::2], c[:, 1::2] = codes % 16, codes // 16
    return (c - 8) * np.repeat(scales, c.shape[1] // scales.shape[1], 1)
