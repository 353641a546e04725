"""Per-head norms with RoPE and scatter (gqa_qk_norm_rope_device, _step_device) against float64.

Bound of a value before its rounding, relative to the magnitudes M that it adds up (|a cos| + |b sin|): the norm's inverse
root and two products are off by 2^-22 at most (a sum of squares of at most 16 sequential and tree additions: 2^-20, half
of it in the root, then four roundings of 2^-24), cosine, sine, two products and a sum 2^-22: below 2^-19 in all.  Then
half a step of bf16 (2^-8 of the value), or of the E4M3 row (2^-4 of it, or 2^-10 of the row's scale).
"""
import ctypes

import numpy as np
import pytest

from lara_amd import _lib
from lara_amd.attn_driver import AttentionAccelerator
from oracle import gqa_oracle as orc
from oracle import serving_oracle as so
from tests._gen import bf16_normal
from tests._serving import call, dev, ptr, scatter_reserve, words

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

FP32 = 2.0**-19


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


@pytest.mark.parametrize("hq,hkv,d,kv_format", [(*shape, fmt) for shape in ((8, 2, 64), (32, 8, 128), (4, 4, 64))
                                                for fmt in ("bf16", "e4m3")] + [(3, 1, 128, "e4m3")])
@pytest.mark.parametrize("norm,base", [(True, 10000.0), (True, 0.0), (False, 1e6)])
def test_tokens_of_one_sequence(hq, hkv, d, kv_format, norm, base):
    rng = np.random.default_rng(hq * d + int(base))
    n, row0, q_pos, k_pos, pad = 37, 60, 1000003, 77, 8
    x = heads_in(rng, n, hq, hkv, d, pad)
    wq, wk = (weights(rng, d) if norm else None for _ in range(2))
    with AttentionAccelerator(batch=2, n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=128, kv_format=kv_format,
                              page_size=64 if hq == 8 else None) as acc:
        if acc.paged:
            scatter_reserve(acc, [128, 128], 64)
        xd, q = dev(x), torch.zeros((hq, n, d), dtype=torch.int16, device="cuda")
        wd = [dev(w) if norm else None for w in (wq, wk)]
        acc.qk_norm_rope_device(xd.data_ptr(), x.shape[1], n, *(w.data_ptr() if norm else None for w in wd), q.data_ptr(), b=1,
                                q_pos_base=q_pos, kv_pos_base=k_pos, kv_row0=row0, eps=1e-6, rope_base=base)
        kg, vg = acc.read_kv(1, 0, 128)
        other = acc.read_kv(0, 0, 128)
    hq64, hk64, hv64 = split(x, hq, hkv, d)
    near_bf16(words(q), *so.norm_rope(hq64, f64(wq) if norm else None, 1e-6, q_pos + np.arange(n), base))
    near = near_bf16 if kv_format == "bf16" else near_e4m3
    near(kg[:, row0:row0 + n], *so.norm_rope(hk64, f64(wk) if norm else None, 1e-6, k_pos + np.arange(n), base))
    v_want = hv64 if kv_format == "bf16" else so.stored(hv64)
    assert np.array_equal(f64(vg[:, row0:row0 + n]), v_want)  # V goes as it is
    for t in (kg, vg):  # the other rows as they were
        assert not t[:, :row0].any() and not t[:, row0 + n:].any()
    assert not other[0].any() and not other[1].any()


@pytest.mark.parametrize("kv_format", ["bf16", "e4m3"])
@pytest.mark.parametrize("page", [None, 64])
def test_one_token_of_each_sequence(kv_format, page):
    """Far positions, rows apart from them, sequences left out, an unmapped row; only one side normalised."""
    rng = np.random.default_rng(21)
    B, hq, hkv, d, L = 6, 8, 2, 128, 192
    x = heads_in(rng, B, hq, hkv, d)
    wq = weights(rng, d)
    pos = np.array([0, 5, -1, 2**29 + 12345, 190, 11], np.int32)
    row = np.array([0, 64, 3, 191, L, 130], np.int32)  # 4: outside; 5: not mapped on the paged engine
    with AttentionAccelerator(batch=B, n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=L, kv_format=kv_format,
                              page_size=page) as acc:
        if page:
            scatter_reserve(acc, [192, 192, 192, 192, 192, 64], 64)
        q = torch.full((B, hq, d), 9, dtype=torch.int16, device="cuda")
        xd, wd, pd, rd = dev(x), dev(wq), dev(pos), dev(row)
        acc.qk_norm_rope_step_device(xd.data_ptr(), x.shape[1], wd.data_ptr(), None, pd.data_ptr(), q.data_ptr(),
                                     rows_ptr=rd.data_ptr(), eps=1e-5, rope_base=5e5)
        torch.cuda.synchronize()
        rows_got = [acc.read_kv(b, 0, 64 if page and b == 5 else L) for b in range(B)]
    qg, h = words(q), split(x, hq, hkv, d)
    for b in range(B):
        out = pos[b] < 0 or row[b] >= L
        if out:
            assert np.all(qg[b] == 9)
        else:
            want, mag = so.norm_rope(h[0][:, b:b + 1], f64(wq), 1e-5, pos[b:b + 1], 5e5)
            near_bf16(qg[b][:, None], want, mag)
        written = np.zeros(rows_got[b][0].shape[1], bool)
        if not out and row[b] < written.size:
            written[row[b]] = True
            want, mag = so.norm_rope(h[1][:, b:b + 1], None, 0.0, pos[b:b + 1], 5e5)
            (near_bf16 if kv_format == "bf16" else near_e4m3)(rows_got[b][0][:, row[b]:row[b] + 1], want, mag)
            v = h[2][:, b:b + 1]
            assert np.array_equal(f64(rows_got[b][1][:, row[b]:row[b] + 1]), v if kv_format == "bf16" else so.stored(v))
        for t in rows_got[b]:
            assert not t[:, ~written].any()


def test_rows_default_to_the_positions_and_long_prompts():
    rng = np.random.default_rng(22)
    hq, hkv, d, n = 8, 2, 64, 1500
    with AttentionAccelerator(batch=2, n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=n, max_q_len=64) as acc:
        x = heads_in(rng, n, hq, hkv, d)
        q = torch.zeros((hq, n, d), dtype=torch.int16, device="cuda")
        wq, wk = weights(rng, d), weights(rng, d)
        xd, wqd, wkd = dev(x), dev(wq), dev(wk)
        acc.qk_norm_rope_device(xd.data_ptr(), x.shape[1], n, wqd.data_ptr(), wkd.data_ptr(), q.data_ptr(), eps=0.0)
        torch.cuda.synchronize()
        h = split(x, hq, hkv, d)
        near_bf16(words(q), *so.norm_rope(h[0], f64(wq), 0.0, np.arange(n), 1e4))
        near_bf16(acc.read_kv(0, 0, n)[0], *so.norm_rope(h[1], f64(wk), 0.0, np.arange(n), 1e4))
        # the same tokens one by one, as steps of sequence 1: the same words
        for t in (0, 1, 63, 700):
            xs, ps = dev(np.stack([x[t], x[t]])), dev(np.array([-1, t], np.int32))
            qs = torch.zeros((2, hq, d), dtype=torch.int16, device="cuda")
            acc.qk_norm_rope_step_device(xs.data_ptr(), x.shape[1], wqd.data_ptr(), wkd.data_ptr(), ps.data_ptr(),
                                         qs.data_ptr(), eps=0.0)
            torch.cuda.synchronize()
            assert np.array_equal(words(qs)[1], words(q)[:, t])
            for a, b in zip(acc.read_kv(1, t, 1), acc.read_kv(0, t, 1)):
                assert np.array_equal(a, b)


def test_refusals():
    lib = _lib.lib()
    t = torch.zeros(1 << 16, dtype=torch.int16, device="cuda")
    u = torch.zeros(1 << 16, dtype=torch.int16, device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    with AttentionAccelerator(batch=2, n_q_heads=8, n_kv_heads=2, head_dim=64, max_seq_len=64, page_size=64, n_pages=1) as acc:
        acc.reserve(0, 64)
        c, width, R = acc._ctx, 12 * 64, _lib.GQA_ERR_RANGE
        odd = ctypes.c_void_p(t.data_ptr() + 2)

        def prompt(b=0, x=ptr(t), ld=width, n=4, wq=None, wk=None, eps=1e-5, qp=0, kp=0, row=0, base=1e4, q=ptr(u)):
            return lib.gqa_qk_norm_rope_device(c, b, x, ld, n, wq, wk, eps, qp, kp, row, base, q, None)

        def step(x=ptr(t), ld=width, eps=1e-5, p=ptr(pos), base=1e4, q=ptr(u)):
            return lib.gqa_qk_norm_rope_step_device(c, x, ld, None, None, eps, p, None, base, q, None)

        assert prompt(b=2) == _lib.GQA_ERR_STREAM_DEST
        assert prompt(x=None) == step(p=None) == step(q=None) == _lib.GQA_ERR_NULL
        for bad in (dict(ld=width - 8), dict(ld=width + 4), dict(n=0), dict(n=65), dict(row=61), dict(row=-1), dict(eps=-1.0),
                    dict(eps=float("nan")), dict(base=1.0), dict(base=-2.0), dict(base=float("inf")), dict(x=odd), dict(wq=odd),
                    dict(wk=odd), dict(q=odd), dict(qp=-1), dict(kp=1 << 30), dict(b=1), dict(q=ptr(t))):
            assert prompt(**bad) == R, bad
        for bad in (dict(ld=width - 8), dict(eps=-1.0), dict(base=0.5), dict(x=odd), dict(q=odd), dict(q=ptr(t))):
            assert step(**bad) == R, bad
        k, v, cap = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_int32()
        call("gqa_cache_pointers", c, ctypes.byref(k), ctypes.byref(v), ctypes.byref(cap))
        assert prompt(x=k) == R and prompt(x=v) == R  # the rows it writes
        assert prompt() == step() == _lib.GQA_OK
        torch.cuda.synchronize()


@pytest.mark.parametrize("d", [64, 128])
def test_rows_whose_squares_are_subnormal_or_zero(d):
    """Mean squares near 2^-128 (2^-21 of it a step of the sum: 2^-19 of a value with the bound above), eps 0; a row of zeros
    with an eps stays zero."""
    rng = np.random.default_rng(41)
    hq, hkv, n = 4, 2, 5
    scale = np.array([2.0**-64, 1.0, 2.0**-63, 2.0**-40, 2.0**-64])
    x = orc.bf16_rne((rng.standard_normal((n, (hq + 2 * hkv) * d)) * scale[:, None]).astype(np.float32))
    zero = np.zeros_like(x)
    with AttentionAccelerator(n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=64) as acc:
        one = dev(orc.bf16_rne(np.ones(d, np.float32)))
        for words_in, eps in ((x, 0.0), (zero, 1e-6)):
            xd, q = dev(words_in), torch.empty((hq, n, d), dtype=torch.int16, device="cuda")
            acc.qk_norm_rope_device(xd.data_ptr(), words_in.shape[1], n, one.data_ptr(), one.data_ptr(), q.data_ptr(), eps=eps, rope_base=0.0)
            torch.cuda.synchronize()
            qh, kh, _ = split(words_in, hq, hkv, d)
            k = acc.read_kv(0, 0, n)[0]
            for got, h in ((words(q), qh), (k, kh)):
                want = h / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
                assert np.all(np.abs(f64(got) - want) <= (2.0**-8 + 2 * FP32) * np.abs(want))


def test_refuses_outputs_in_the_cache_or_over_the_weights():
    t = torch.zeros(1 << 16, dtype=torch.int16, device="cuda")
    u = torch.zeros(1 << 16, dtype=torch.int16, device="cuda")
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    lib, R = _lib.lib(), _lib.GQA_ERR_RANGE
    with AttentionAccelerator(n_q_heads=8, n_kv_heads=2, head_dim=64, max_seq_len=64, kv_format="e4m3") as acc:
        c, width = acc._ctx, 12 * 64
        k, v, ks, vs = (ctypes.c_void_p() for _ in range(4))
        cap = ctypes.c_int32()
        call("gqa_cache_pointers", c, ctypes.byref(k), ctypes.byref(v), ctypes.byref(cap))
        call("gqa_kv8_scales", c, ctypes.byref(ks), ctypes.byref(vs))

        def prompt(x=ptr(t), ld=width, wq=None, q=ptr(u)):
            return lib.gqa_qk_norm_rope_device(c, 0, x, ld, 4, wq, None, 1e-5, 0, 0, 0, 1e4, q, None)

        for inside in (k, v, ks, vs):
            assert prompt(q=inside) == R and prompt(x=inside) == R
            assert lib.gqa_read_kv_device(c, 0, 0, 4, inside, ptr(t), None) == R
            assert lib.gqa_read_kv_device(c, 0, 0, 4, ptr(t), inside, None) == R
        assert lib.gqa_read_kv_device(c, 0, 0, 4, ptr(t), ptr(t), None) == R
        assert prompt(wq=ptr(u)) == R and prompt(ld=1 << 31) == R
        odd = ctypes.c_void_p(pos.data_ptr() + 2)
        for p, r in ((odd, None), (ptr(pos), odd)):
            assert lib.gqa_qk_norm_rope_step_device(c, ptr(t), width, None, None, 1e-5, p, r, 1e4, ptr(u), None) == R
        assert prompt() == _lib.GQA_OK
        torch.cuda.synchronize()
