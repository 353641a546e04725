"""Rotary forms: how a model turns its query and key heads (``gqa_rope`` of include/gqa.h).

``form`` makes one for ``AttentionAccelerator.qk_norm_rotary_device`` and its step form; ``frequencies`` gives the angle per
position of every pair that it turns.
"""
from __future__ import annotations

import ctypes

import numpy as np

from . import _lib

LAYOUTS = {"pairs": _lib.GQA_ROPE_PAIRS, "halves": _lib.GQA_ROPE_HALVES}
SCALINGS = {"plain": _lib.GQA_ROPE_PLAIN, "linear": _lib.GQA_ROPE_LINEAR, "bands": _lib.GQA_ROPE_BANDS, "ramp": _lib.GQA_ROPE_RAMP}
_ENDS = {"bands": (1.0, 4.0), "ramp": (1.0, 32.0)}  # turns over original_len: divided below, kept above


def form(layout: str = "halves", *, rotary_dim: int = 0, base: float = 10000.0, scaling: str = "plain", factor: float = 1.0,
         original_len: int = 0, low: float | None = None, high: float | None = None, magnitude: float = 0.0) -> "_lib.GqaRope":
    """The first ``rotary_dim`` dims of a head (0: all) turn in "pairs" (2p, 2p + 1) or "halves" (p, p + rotary_dim / 2);
    ``scaling`` stretches the frequencies for contexts longer than ``original_len`` by ``factor``: "linear" all of them,
    "bands" and "ramp" those that turn less than ``high`` (4, 32) times over it, entirely below ``low`` (1) times."""
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {sorted(LAYOUTS)}, got {layout!r}")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {sorted(SCALINGS)}, got {scaling!r}")
    ends = _ENDS.get(scaling, (0.0, 0.0))
    return _lib.GqaRope(LAYOUTS[layout], int(rotary_dim), SCALINGS[scaling], int(original_len), float(base), float(factor),
                        float(ends[0] if low is None else low), float(ends[1] if high is None else high), float(magnitude))


def frequencies(rope: "_lib.GqaRope", head_dim: int) -> tuple[np.ndarray, float]:
    """Angle per position of each pair that turns, and what multiplies cosine and sine (``gqa_rope_frequencies``)."""
    out, magnitude = (ctypes.c_double * (int(head_dim) // 2))(), ctypes.c_double(0.0)
    _lib.check(_lib.lib().gqa_rope_frequencies(ctypes.byref(rope), int(head_dim), out, ctypes.byref(magnitude)), "gqa_rope_frequencies")
    return np.array(out[: (rope.rotary_dim or int(head_dim)) // 2]), float(magnitude.value)
