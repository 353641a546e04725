"""4-bit weights with group scales on the host: quantisation and the packed sizes.

A matrix [rows, hidden] is codes c of 0..15 (two a byte, the even column in the low four bits) and one bf16 scale per row
and group of columns: w = (c - 8) * scale.  ``AttentionAccelerator.w4_pack_device`` lays them out for the products.
"""
from __future__ import annotations

import ctypes

import numpy as np

from . import _lib
from .attn_driver import bf16_u16_to_fp32

GROUPS = (32, 64, 128)


def packed_bytes(rows: int, hidden: int, group: int) -> tuple[int, int]:
    """Bytes of the packed codes and of the packed scales (``gqa_w4_bytes``)."""
    w, s = ctypes.c_int64(0), ctypes.c_int64(0)
    _lib.check(_lib.lib().gqa_w4_bytes(int(rows), int(hidden), int(group), ctypes.byref(w), ctypes.byref(s)), "gqa_w4_bytes")
    return int(w.value), int(s.value)


def quantize(w: np.ndarray, group: int) -> tuple[np.ndarray, np.ndarray]:
    """Codes [rows, hidden / 2] (uint8) and bf16 scale words [rows, hidden / group] of a matrix (floats, or bf16 words):
    per group the scale is its value of largest magnitude over -8, rounded to bf16, so that it takes code 0, and the
    others the nearest code (ties to the even one)."""
    w = bf16_u16_to_fp32(w) if np.asarray(w).dtype == np.uint16 else np.asarray(w, dtype=np.float32)
    if w.ndim != 2 or group not in GROUPS or w.shape[1] % group or not w.shape[1]:
        raise ValueError(f"expected [rows, hidden] with hidden a multiple of the group (one of {GROUPS}); got {w.shape}, {group}")
    if not np.all(np.isfinite(w)):
        raise ValueError("weights must be finite")
    g = w.reshape(w.shape[0], -1, group)
    top = np.take_along_axis(g, np.abs(g).argmax(-1)[..., None], -1)[..., 0]
    bits = (top / np.float32(-8)).astype(np.float32).view(np.uint32).astype(np.uint64)
    scales = ((bits + 0x7FFF + ((bits >> 16) & 1)) >> 16).astype(np.uint16)  # nearest even
    s = bf16_u16_to_fp32(scales)[..., None].astype(np.float64)
    c = np.divide(g, s, out=np.zeros(g.shape, np.float64), where=s != 0)
    c = (np.clip(np.rint(c), -8, 7) + 8).astype(np.uint8).reshape(w.shape)
    return np.ascontiguousarray(c[:, 0::2] | (c[:, 1::2] << 4)), scales
