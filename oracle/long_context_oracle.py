"""CPU oracle of the long-context operators: rotary forms, accumulated attention weight, eviction.

TEST INFRASTRUCTURE ONLY, as ``oracle/gqa_oracle.py``.  Everything is float64 numpy written from the definitions:

* ``frequencies`` -- angle per position of each pair, one pair at a time.
* ``norm_rotary`` -- y = h / sqrt(mean(h^2) + eps) * w, then the pairs turned as complex numbers.
* ``mass`` -- sum over query rows of exp(scale * q . k - lse) for the keys that each row sees.
* ``evict`` -- the rows that stay, by sorting.

Attention over a shared prefix is ``serving_oracle.decode`` over the rows put together.  Pinned in
``tests/test_long_context_oracle.py``.
"""
from __future__ import annotations

import math

import numpy as np


def frequencies(rotary_dim, base, scaling="plain", factor=1.0, original_len=0, low=0.0, high=0.0):
    """(angles per position [rotary_dim / 2], what multiplies cosine and sine)."""
    out = []
    ends = None
    if scaling == "ramp":
        at = [rotary_dim * math.log(original_len / (2 * math.pi * turns)) / (2 * math.log(base)) for turns in (high, low)]
        ends = max(0, math.floor(at[0])), min(rotary_dim - 1, math.ceil(at[1]))
    for p in range(rotary_dim // 2):
        f = float(base) ** (-2.0 * p / rotary_dim)
        if scaling == "linear":
            f /= factor
        elif scaling == "bands":
            turns = original_len * f / (2 * math.pi)
            if turns <= low:
                f /= factor
            elif turns < high:
                w = (turns - low) / (high - low)
                f = f * w + f / factor * (1 - w)
        elif scaling == "ramp":
            w = min(1.0, max(0.0, (p - ends[0]) / max(ends[1] - ends[0], 0.001)))
            f = f / factor * w + f * (1 - w)
        out.append(f)
    return np.array(out), 0.1 * math.log(factor) + 1 if scaling == "ramp" else 1.0


def norm_rotary(h, weight, eps, positions, freq, magnitude, halves):
    """h [..., n, D] at positions [n]: (y, sum of the magnitudes that each y adds up); weight None: no norm."""
    h = np.asarray(h, dtype=np.float64)
    if weight is not None:
        h = h / np.sqrt((h * h).mean(-1, keepdims=True) + eps) * weight
    n = len(freq)
    a, b = (np.arange(n), np.arange(n) + n) if halves else (2 * np.arange(n), 2 * np.arange(n) + 1)
    turn = magnitude * np.exp(1j * np.asarray(positions, dtype=np.float64)[:, None] * freq)
    z = (h[..., a] + 1j * h[..., b]) * turn
    c, s = np.abs(turn.real), np.abs(turn.imag)
    y, mag = h.copy(), np.abs(h)
    ha, hb = mag[..., a].copy(), mag[..., b].copy()
    y[..., a], y[..., b] = z.real, z.imag
    mag[..., a], mag[..., b] = ha * c + hb * s, ha * s + hb * c
    return y, mag


def mass(q, k, lse, scale, seen=None):
    """q [H_q, n, D], lse [H_q, n] against k [H_kv, L, D]: weight of every key [H_kv, L]; seen [n, L] (None: all).  Rows
    whose lse is not finite add nothing."""
    group = q.shape[0] // k.shape[0]
    out = np.zeros(k.shape[:2])
    for h in range(q.shape[0]):
        for i in range(q.shape[1]):
            if not np.isfinite(lse[h, i]):
                continue
            with np.errstate(invalid="ignore", over="ignore"):
                p = np.exp(scale * (k[h // group] @ q[h, i]) - lse[h, i])
            out[h // group] += p if seen is None else np.where(seen[i], p, 0.0)
    return out


def evict(mass_row, length, keep, sinks, recent):
    """Former rows of what one (sequence, kv head) keeps, in order."""
    if length <= keep:
        return np.arange(length)
    middle = list(range(sinks, length - recent))
    weight = [-math.inf if math.isnan(m) else m for m in mass_row]
    lowest = [math.isnan(m) for m in mass_row]
    middle.sort(key=lambda t: (-weight[t], lowest[t], t))
    best = sorted(middle[:keep - sinks - recent])
    return np.array(list(range(sinks)) + best + list(range(length - recent, length)), dtype=np.int64)
