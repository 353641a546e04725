"""Rotary forms (gqa_qk_norm_rotary_device, _step_device) against float64.

Bound of a value before its rounding, relative to the magnitudes M that it adds up (|a c| + |b s|): the norm's inverse root
and two products as in test_gpu_heads.py, below 2^-20.4; the angle, in turns: its fraction is rounded by at most 2^-26 of a
turn (2^-23.3 rad), its 64-bit product before that by 2^-53 of at most 2^28 turns (2^-22.3 rad), sine and cosine by 2^-22,
the magnitude, two products and a sum by 2^-22: below 2^-19 in all.  Then half a step of bf16 (2^-8 of the value), or of
the E4M3 row (2^-4 of it, or 2^-10 of the row's scale).
"""
import ctypes

import numpy as np
import pytest

from lara_amd import _lib, rope
from lara_amd.attn_driver import AttentionAccelerator
from oracle import gqa_oracle as orc
from oracle import long_context_oracle as lo
from oracle import serving_oracle as so
from tests._serving import call, dev, ptr, scatter_reserve, words

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

FP32 = 2.0**-19

SCALED = {"plain": dict(scaling="plain"), "linear": dict(scaling="linear", factor=4.0),
          "bands": dict(scaling="bands", factor=8.0, original_len=8192, low=1.0, high=4.0),
          "ramp": dict(scaling="ramp", factor=16.0, original_len=4096, low=1.0, high=32.0)}


def f64(w):
    return orc.bf16_u16_to_fp32(w).astype(np.float64)


def heads_in(rng, n, hq, hkv, d, pad=0):
    x = rng.standard_normal((n, hq + 2 * hkv, d)) * np.exp(rng.standard_normal((n, hq + 2 * hkv, 1)))
    out = np.full((n, (hq + 2 * hkv) * d + pad), 0x7FC0, np.uint16)
    out[:, :(hq + 2 * hkv) * d] = orc.bf16_rne(x.astype(np.float32)).reshape(n, -1)
    return out


def split(x, hq, hkv, d):
    h = f64(x[:, :(hq + 2 * hkv) * d]).reshape(x.shape[0], -1, d).transpose(1, 0, 2)
    return h[:hq], h[hq:hq + hkv], h[hq + hkv:]


def near_bf16(got, ref, mag):
    assert np.all(np.abs(f64(got) - ref) <= 2.0**-8 * np.abs(ref) + FP32 * mag + 2.0**-133)


def near_e4m3(got, ref, mag):
    _, scale = so.e4m3_row(ref)
    step = np.maximum(2.0**-4 * np.abs(ref), 2.0**-10 * scale[..., None])
    assert np.all(np.abs(f64(got) - ref) <= step + FP32 * mag)


def weights(rng, d):
    return orc.bf16_rne((1 + 0.2 * rng.standard_normal(d)).astype(np.float32))


@pytest.mark.parametrize("kv_format", ["bf16", "e4m3"])
@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("hq,hkv,d,part,scaling", [(8, 2, 64, 0, "ramp"), (8, 2, 64, 16, "linear"), (8, 2, 64, 8, "plain"), (8, 2, 64, 40, "bands"),
                                                   (32, 8, 128, 0, "bands"), (32, 8, 128, 64, "ramp"), (16, 8, 128, 32, "plain"),
                                                   (8, 2, 128, 120, "ramp")])
def test_prompt_rows(kv_format, layout, hq, hkv, d, part, scaling):
    """An odd count of tokens, positions of Q and K apart, rows behind the written ones as they were, pages, both norms."""
    rng = np.random.default_rng(hq * d + part)
    n, row0, q_pos, k_pos, pad = 37, 60, 1000003, 77, 8
    x = heads_in(rng, n, hq, hkv, d, pad)
    wq, wk = weights(rng, d), weights(rng, d)
    form = rope.form(layout, rotary_dim=part, base=5e5, **SCALED[scaling])
    with AttentionAccelerator(batch=2, n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=128, kv_format=kv_format,
                              page_size=64 if hq == 8 else None) as acc:
        if acc.paged:
            scatter_reserve(acc, [128, 128], 64)
        xd, wqd, wkd = dev(x), dev(wq), dev(wk)
        q = torch.full((hq + 1, n, d), 9, dtype=torch.int16, device="cuda")
        acc.qk_norm_rotary_device(xd.data_ptr(), x.shape[1], n, wqd.data_ptr(), wkd.data_ptr(), q.data_ptr(), form, b=1, q_pos_base=q_pos,
                                  kv_pos_base=k_pos, kv_row0=row0, eps=1e-6)
        kg, vg = acc.read_kv(1, 0, 128)
        other = acc.read_kv(0, 0, 128)
    f, m = lo.frequencies(part or d, 5e5, **SCALED[scaling])
    hq64, hk64, hv64 = split(x, hq, hkv, d)
    halves = layout == "halves"
    got = words(q)
    near_bf16(got[:hq], *lo.norm_rotary(hq64, f64(wq), 1e-6, q_pos + np.arange(n), f, m, halves))
    assert np.all(got[hq:] == 9)
    near = near_bf16 if kv_format == "bf16" else near_e4m3
    near(kg[:, row0:row0 + n], *lo.norm_rotary(hk64, f64(wk), 1e-6, k_pos + np.arange(n), f, m, halves))
    assert np.array_equal(f64(vg[:, row0:row0 + n]), hv64 if kv_format == "bf16" else so.stored(hv64))
    for t in (kg, vg):
        assert not t[:, :row0].any() and not t[:, row0 + n:].any()
    assert not other[0].any() and not other[1].any()


@pytest.mark.parametrize("kv_format", ["bf16", "e4m3"])
@pytest.mark.parametrize("layout,part,scaling,page", [("halves", 0, "ramp", None), ("halves", 32, "plain", 64), ("pairs", 64, "bands", 64),
                                                      ("halves", 128, "linear", None)])
def test_one_token_of_each_sequence(kv_format, layout, part, scaling, page):
    """Far positions, rows apart from them, sequences left out, an unmapped row; only one side normalised."""
    rng = np.random.default_rng(21)
    B, hq, hkv, d, L = 6, 8, 2, 128, 192
    x = heads_in(rng, B, hq, hkv, d)
    wq = weights(rng, d)
    pos = np.array([0, 5, -1, 2**29 + 12345, 190, 11], np.int32)
    row = np.array([0, 64, 3, 191, L, 130], np.int32)  # 4: outside; 5: not mapped on the paged engine
    form = rope.form(layout, rotary_dim=part, base=1e4, **SCALED[scaling])
    f, m = lo.frequencies(part or d, 1e4, **SCALED[scaling])
    halves = layout == "halves"
    with AttentionAccelerator(batch=B, n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=L, kv_format=kv_format,
                              page_size=page) as acc:
        if page:
            scatter_reserve(acc, [192, 192, 192, 192, 192, 64], 64)
        q = torch.full((B, hq, d), 9, dtype=torch.int16, device="cuda")
        xd, wd, pd, rd = dev(x), dev(wq), dev(pos), dev(row)
        acc.qk_norm_rotary_step_device(xd.data_ptr(), x.shape[1], wd.data_ptr(), None, pd.data_ptr(), q.data_ptr(), form,
                                       rows_ptr=rd.data_ptr(), eps=1e-5)
        torch.cuda.synchronize()
        rows_got = [acc.read_kv(b, 0, 64 if page and b == 5 else L) for b in range(B)]
    qg, h = words(q), split(x, hq, hkv, d)
    for b in range(B):
        out = pos[b] < 0 or row[b] >= L
        if out:
            assert np.all(qg[b] == 9)
        else:
            near_bf16(qg[b][:, None], *lo.norm_rotary(h[0][:, b:b + 1], f64(wq), 1e-5, pos[b:b + 1], f, m, halves))
        written = np.zeros(rows_got[b][0].shape[1], bool)
        if not out and row[b] < written.size:
            written[row[b]] = True
            want = lo.norm_rotary(h[1][:, b:b + 1], None, 0.0, pos[b:b + 1], f, m, halves)
            (near_bf16 if kv_format == "bf16" else near_e4m3)(rows_got[b][0][:, row[b]:row[b] + 1], *want)
            v = h[2][:, b:b + 1]
            assert np.array_equal(f64(rows_got[b][1][:, row[b]:row[b] + 1]), v if kv_format == "bf16" else so.stored(v))
        for t in rows_got[b]:
            assert not t[:, ~written].any()


def test_the_plain_form_is_near_the_other_entry_points():
    """Pairs over all of a head with plain frequencies are what qk_norm_rope_device computes, but for the angle's way: the two
    differ by a step of bf16 at most where a value lies next to a border."""
    rng = np.random.default_rng(5)
    hq, hkv, d, n = 8, 2, 64, 300
    x, wq, wk = heads_in(rng, n, hq, hkv, d), weights(rng, d), weights(rng, d)
    got = []
    for rotary in (False, True):
        with AttentionAccelerator(n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=n, max_q_len=64) as acc:
            xd, wqd, wkd = dev(x), dev(wq), dev(wk)
            q = torch.zeros((hq, n, d), dtype=torch.int16, device="cuda")
            args = (xd.data_ptr(), x.shape[1], n, wqd.data_ptr(), wkd.data_ptr(), q.data_ptr())
            if rotary:
                acc.qk_norm_rotary_device(*args, rope.form("pairs"), q_pos_base=9000, kv_pos_base=9000)
            else:
                acc.qk_norm_rope_device(*args, q_pos_base=9000, kv_pos_base=9000)
            got.append((f64(words(q)), *(f64(t) for t in acc.read_kv(0, 0, n))))
    _, mag = lo.norm_rotary(split(x, hq, hkv, d)[0], f64(wq), 1e-5, 9000 + np.arange(n), *lo.frequencies(d, 10000.0), False)
    assert np.all(np.abs(got[0][0] - got[1][0]) <= 2.0**-7 * np.abs(got[0][0]) + 2 * FP32 * mag)
    assert np.mean(got[0][0] != got[1][0]) < 0.01
    assert np.array_equal(got[0][2], got[1][2])


def test_magnitude_and_weights_of_none():
    rng = np.random.default_rng(6)
    hq, hkv, d, n = 4, 4, 64, 3
    x = heads_in(rng, n, hq, hkv, d)
    form = rope.form("halves", rotary_dim=32, magnitude=1.5)
    with AttentionAccelerator(n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=n) as acc:
        xd, q = dev(x), torch.zeros((hq, n, d), dtype=torch.int16, device="cuda")
        acc.qk_norm_rotary_device(xd.data_ptr(), x.shape[1], n, None, None, q.data_ptr(), form)
        torch.cuda.synchronize()
    f, _ = lo.frequencies(32, 10000.0)
    want, mag = lo.norm_rotary(split(x, hq, hkv, d)[0], None, 0.0, np.arange(n), f, 1.5, True)
    near_bf16(words(q), want, mag)
    assert np.array_equal(words(q)[..., 32:], x[:, :hq * d].reshape(n, hq, d).transpose(1, 0, 2)[..., 32:])


def test_refusals():
    rng = np.random.default_rng(7)
    hq, hkv, d, n = 8, 2, 64, 4
    width = (hq + 2 * hkv) * d
    x = dev(heads_in(rng, n, hq, hkv, d))
    q = torch.zeros((n * hq, d), dtype=torch.int16, device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    with AttentionAccelerator(batch=2, n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=64) as acc:
        def rc(form=rope.form(), **kw):
            a = dict(b=0, qkv=ptr(x), ld=width, n=n, wq=None, wk=None, eps=1e-5, q0=0, k0=0, row0=0, q=ptr(q), **{})
            a.update(kw)
            r = ctypes.byref(form) if form is not None else None
            return acc._lib.gqa_qk_norm_rotary_device(acc._ctx, a["b"], a["qkv"], a["ld"], a["n"], a["wq"], a["wk"], a["eps"], a["q0"], a["k0"],
                                                      a["row0"], r, a["q"], None)

        E = _lib
        for kw, want in [(dict(qkv=None), E.GQA_ERR_NULL), (dict(q=None), E.GQA_ERR_NULL), (dict(form=None), E.GQA_ERR_NULL),
                         (dict(b=2), E.GQA_ERR_STREAM_DEST), (dict(b=-1), E.GQA_ERR_STREAM_DEST), (dict(n=0), E.GQA_ERR_RANGE),
                         (dict(row0=61), E.GQA_ERR_RANGE), (dict(ld=width - 8), E.GQA_ERR_RANGE), (dict(ld=width + 4), E.GQA_ERR_RANGE),
                         (dict(eps=-1.0), E.GQA_ERR_RANGE), (dict(q0=2**30 - 3), E.GQA_ERR_RANGE), (dict(k0=-1), E.GQA_ERR_RANGE),
                         (dict(form=rope.form(rotary_dim=12)), E.GQA_ERR_RANGE), (dict(form=rope.form(rotary_dim=128)), E.GQA_ERR_RANGE),
                         (dict(form=rope.form(base=0.0)), E.GQA_ERR_RANGE), (dict(q=ptr(x)), E.GQA_ERR_RANGE),
                         (dict(q=ctypes.c_void_p(q.data_ptr() + 2)), E.GQA_ERR_RANGE)]:
            assert rc(**kw) == want, kw
        assert rc() == 0
        step = acc._lib.gqa_qk_norm_rotary_step_device
        f = ctypes.byref(rope.form())
        assert step(acc._ctx, ptr(x), width, None, None, 1e-5, None, None, f, ptr(q), None) == E.GQA_ERR_NULL
        assert step(acc._ctx, ptr(x), width, None, None, 1e-5, ctypes.c_void_p(pos.data_ptr() + 2), None, f, ptr(q), None) == E.GQA_ERR_RANGE
        assert step(acc._ctx, ptr(x), width, None, None, 1e-5, ptr(pos), None, None, ptr(q), None) == E.GQA_ERR_NULL
        assert step(acc._ctx, ptr(x), width, None, None, 1e-5, ptr(pos), None, f, ptr(q), None) == 0
        torch.cuda.synchronize()
