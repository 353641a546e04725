"""Device buffers and engine pools for the tests of the serving operators."""
from __future__ import annotations

import ctypes

import numpy as np

from lara_amd import _lib

P = ctypes.c_void_p


def dev(words):
    """A numpy array on the GPU (uint16 words as int16)."""
    import torch

    a = np.ascontiguousarray(words)
    return torch.from_numpy(a.view(np.int16) if a.dtype == np.uint16 else a).cuda()


def words(t):
    """bf16 words of an int16 tensor, on the host."""
    return t.cpu().numpy().view(np.uint16)


def ptr(t):
    return P(t.data_ptr()) if t is not None else None


def call(name, *args):
    _lib.check(getattr(_lib.lib(), name)(*args), name)


class _Memory:
    def __init__(self, engine, address, shape):
        self.engine = engine
        self.__cuda_array_interface__ = {"shape": shape, "typestr": "|u1", "data": (address, False), "version": 2}


def kv8_pools(acc):
    """The active layer's codes and scale bytes of an E4M3 engine: (k, v, k_scale, v_scale) uint8 tensors."""
    import torch

    k, v, ks, vs, cap = P(), P(), P(), P(), ctypes.c_int32()
    call("gqa_cache_pointers", acc._ctx, ctypes.byref(k), ctypes.byref(v), ctypes.byref(cap))
    call("gqa_kv8_scales", acc._ctx, ctypes.byref(ks), ctypes.byref(vs))
    lead = acc.page_info()["n_pages"] if acc.paged else acc.batch
    shape = (lead, acc.n_kv_heads, cap.value)
    return [torch.as_tensor(_Memory(acc, p.value, s), device="cuda")
            for p, s in ((k, (*shape, acc.head_dim)), (v, (*shape, acc.head_dim)), (ks, shape), (vs, shape))]


def scatter_reserve(acc, lens, step):
    """Grow every sequence one page at a time, in turn, so that their pages interleave."""
    grown = [0] * len(lens)
    while any(g < t for g, t in zip(grown, lens)):
        for b, t in enumerate(lens):
            if grown[b] < t:
                grown[b] = min(t, grown[b] + step)
                acc.reserve(b, grown[b])
