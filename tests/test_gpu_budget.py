"""Accumulated attention weight (gqa_attention_mass_*) and eviction (gqa_evict_device).

Mass against float64.  A weight's relative error is that of its exponent: the score is a sum of D exact products, off by at
most D 2^-24 of S = scale * sum |q k| (every addition rounds once), the scale, the shift and their difference by 4 * 2^-24 of
|s| + |lse|; then exp2 (2^-22), and the sum over n query rows (n 2^-24 at most).  The old mass is rounded twice more.
Eviction moves and selects: everything is equal.
"""
import ctypes

import numpy as np
import pytest

from lara_amd import _lib
from lara_amd.attn_driver import AttentionAccelerator
from oracle import gqa_oracle as orc
from oracle import long_context_oracle as lo
from oracle import serving_oracle as so
from tests._gen import bf16_normal
from tests._serving import dev, kv8_pools, ptr, scatter_reserve

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def f64(w):
    return orc.bf16_u16_to_fp32(w).astype(np.float64)


def stored(k, kv_format):
    return f64(k) if kv_format == "bf16" else so.stored(f64(k))


def bound(new, q, k, lse, scale, old, decay):
    group = q.shape[0] // k.shape[0]
    s = scale * np.einsum("hnd,hld->hnl", np.abs(q), np.abs(np.repeat(k, group, 0))).max()
    finite = lse[np.isfinite(lse)]
    rel = (q.shape[-1] * s + 4 * (s + (np.abs(finite).max() if finite.size else 0)) + 4 + q.shape[1] * group) * 2.0**-24
    return rel * new + 2.0**-23 * (decay * np.abs(old) + new) + 1e-37


@pytest.mark.parametrize("kv_format", ["bf16", "e4m3"])
@pytest.mark.parametrize("page", [None, 64])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (32, 8, 128), (64, 4, 128), (4, 2, 128)])
def test_step_mass(kv_format, page, hq, hkv, d):
    """Lengths from none to several work-groups' keys, NaN behind them and in masses that decay 0 overwrites, rows without a
    finite lse, other rows' mass as it was."""
    rng = np.random.default_rng(hq + d)
    L = 1300
    lens = np.array([0, 1, 63, 64, 65, 700, 1300], np.int32)
    B = len(lens)
    k = bf16_normal(rng, (B, hkv, L, d))
    v = bf16_normal(rng, (B, hkv, L, d))
    q = bf16_normal(rng, (B, hq, d))
    with AttentionAccelerator(batch=B, n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=L, max_q_len=1, kv_format=kv_format,
                              page_size=page) as acc:
        if page:
            scatter_reserve(acc, [L] * B, 64)
        for b in range(B):
            bad = k[b].copy()
            bad[:, lens[b]:] = 0x7FC0  # stale rows
            acc.load_kv(bad, v[b], b=b)
        lse = np.full((B, hq), -np.inf, np.float32)
        for b in range(B):
            if lens[b]:
                lse[b] = so.decode(f64(q[b]), stored(k[b][:, :lens[b]], kv_format), f64(v[b][:, :lens[b]]), acc.scale)[1]
        lse[5, 1], lse[6, 0], lse[6, hq - 1] = np.nan, np.inf, -np.inf
        old = rng.random((B, hkv, L)).astype(np.float32)
        qd, ld, lsed = dev(q), dev(lens), dev(lse)
        for decay in (1.0, 0.75, 0.0):
            start = old if decay else np.full_like(old, np.nan)
            m = dev(start)
            acc.attention_mass_step_device(qd.data_ptr(), ld.data_ptr(), lsed.data_ptr(), m.data_ptr(), decay=decay)
            torch.cuda.synchronize()
            got = m.cpu().numpy()
            for b in range(B):
                n = lens[b]
                assert np.array_equal(got[b, :, n:], start[b, :, n:], equal_nan=True)
                if not n:
                    continue
                kk, l64 = stored(k[b][:, :n], kv_format), lse[b].astype(np.float64)[:, None]
                new = lo.mass(f64(q[b])[:, None], kk, l64, acc.scale)
                was = old[b, :, :n] if decay else 0.0
                tol = bound(new, f64(q[b])[:, None], kk, l64, acc.scale, was, decay)
                assert np.all(np.abs(got[b, :, :n] - (decay * was + new)) <= tol)


@pytest.mark.parametrize("kv_format", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq,hkv,d,q_len,kv_len,q0,causal,page", [(8, 2, 64, 1, 1, 0, True, None), (8, 2, 64, 33, 70, 37, True, 64),
                                                                 (32, 8, 128, 45, 333, 288, True, None), (8, 8, 128, 100, 90, 0, True, 64),
                                                                 (16, 1, 64, 13, 500, 0, False, None), (4, 2, 128, 150, 400, 100, True, None),
                                                                 (8, 2, 64, 64, 5000, 4936, True, 64), (16, 4, 64, 20, 70000, 69980, True, None),
                                                                 (12, 4, 128, 37, 200, 163, True, None)])
def test_block_mass(kv_format, hq, hkv, d, q_len, kv_len, q0, causal, page):
    """A prompt's rows: one, odd counts, rows past the keys and keys that no row sees, one work-group's keys and many."""
    if hq == 12 and kv_format == "bf16":
        pytest.skip("a bf16 engine has no groups of 3")
    rng = np.random.default_rng(q_len + kv_len)
    k, v = bf16_normal(rng, (hkv, kv_len, d)), bf16_normal(rng, (hkv, kv_len, d))
    q = bf16_normal(rng, (hq, q_len, d))
    kk = stored(k, kv_format)
    seen = np.arange(kv_len) <= q0 + np.arange(q_len)[:, None] if causal else np.ones((q_len, kv_len), bool)
    with AttentionAccelerator(batch=2, n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=kv_len + 3, max_q_len=q_len,
                              kv_format=kv_format, page_size=page) as acc:
        if page:
            scatter_reserve(acc, [kv_len + 3] * 2, 64)
        acc.load_kv(k, v, b=1)
        s = acc.scale * np.einsum("hnd,hld->hnl", f64(q), np.repeat(kk, hq // hkv, 0))
        s = np.where(seen, s, -np.inf)
        top = s.max(-1, keepdims=True)
        with np.errstate(divide="ignore"):
            lse = (top + np.log(np.exp(s - np.where(np.isinf(top), 0, top)).sum(-1, keepdims=True)))[..., 0].astype(np.float32)
        old = rng.random((2, hkv, kv_len + 3)).astype(np.float32)
        qd, lsed = dev(q), dev(lse)
        new = np.zeros((hkv, kv_len))
        for h in range(hq):
            with np.errstate(invalid="ignore"):
                p = np.where(seen, np.exp(s[h] - lse[h].astype(np.float64)[:, None]), 0.0)
            new[h // (hq // hkv)] += p[np.isfinite(lse[h])].sum(0)
        for decay in (1.0, 0.0):
            m = dev(old)
            acc.attention_mass_device(qd.data_ptr(), q_len, kv_len, lsed.data_ptr(), m.data_ptr(), b=1, q_pos_base=q0, causal=causal,
                                      decay=decay)
            torch.cuda.synchronize()
            got = m.cpu().numpy()
            assert np.array_equal(got[0], old[0]) and np.array_equal(got[1, :, kv_len:], old[1, :, kv_len:])
            was = decay * old[1, :, :kv_len]
            tol = bound(new, f64(q), kk, lse.astype(np.float64), acc.scale, was, 1.0)
            assert np.all(np.abs(got[1, :, :kv_len] - (was + new)) <= tol)


def test_block_mass_of_far_positions_and_the_same_twice():
    """Positions near 2^31 with a shifted key base, and two runs give the same words."""
    rng = np.random.default_rng(3)
    hq, hkv, d, n, L = 8, 2, 64, 70, 900
    k, v, q = bf16_normal(rng, (hkv, L, d)), bf16_normal(rng, (hkv, L, d)), bf16_normal(rng, (hq, n, d))
    lse = dev(np.full((hq, n), 3.0, np.float32))
    with AttentionAccelerator(n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=L, max_q_len=n) as acc:
        acc.load_kv(k, v)
        qd, out = dev(q), []
        base = 2**31 - 1 - L
        for kv0 in (0, base, base):
            m = torch.zeros((1, hkv, L), device="cuda")
            acc.attention_mass_device(qd.data_ptr(), n, L, lse.data_ptr(), m.data_ptr(), q_pos_base=kv0 + L - n - 100, kv_pos_base=kv0)
            out.append(m)
        torch.cuda.synchronize()
    assert torch.equal(out[0], out[1]) and torch.equal(out[1], out[2])
    assert not out[0][..., L - 100:].any() and out[0][..., :L - 100].gt(0).all()


def run_evict(acc, mass, lens, keep, sinks, recent, in_place):
    m, ln = dev(mass), dev(lens)
    nm, nl = (m, ln) if in_place else (torch.full_like(m, 7.0), torch.full_like(ln, 7))
    kept = torch.full((len(lens), acc.n_kv_heads, keep), 5, dtype=torch.int32, device="cuda")
    acc.evict_device(m.data_ptr(), ln.data_ptr(), keep, kept.data_ptr(), sinks=sinks, recent=recent,
                     new_mass_ptr=None if in_place else nm.data_ptr(), new_lens_ptr=None if in_place else nl.data_ptr())
    torch.cuda.synchronize()
    if not in_place:
        assert np.array_equal(m.cpu().numpy(), mass, equal_nan=True) and np.array_equal(ln.cpu().numpy(), lens)
    return kept.cpu().numpy(), nl.cpu().numpy(), nm.cpu().numpy()


def check_evict(rng, acc, lens, L, keep, sinks, recent, mass, in_place, kv_format):
    B, hkv, d = len(lens), acc.n_kv_heads, acc.head_dim
    k, v = bf16_normal(rng, (B, hkv, L, d)), bf16_normal(rng, (B, hkv, L, d), 3.0)
    for b in range(B):
        acc.load_kv(k[b], v[b], b=b)
    before = [acc.read_kv(b, 0, L) for b in range(B)]
    raw = [p.clone() for p in kv8_pools(acc)] if kv_format == "e4m3" else None
    kept, new_lens, new_mass = run_evict(acc, mass, lens, keep, sinks, recent, in_place)
    for b in range(B):
        n = min(max(int(lens[b]), 0), L)
        got = acc.read_kv(b, 0, L)
        assert new_lens[b] == min(n, keep)
        for h in range(hkv):
            at = lo.evict(mass[b, h, :n].tolist(), n, keep, sinks, recent)
            assert np.array_equal(kept[b, h, :len(at)], at) and np.all(kept[b, h, len(at):] == -1)
            for x, y in zip(before[b], got):
                want = x[h].copy()
                want[:len(at)] = x[h][at]
                assert np.array_equal(y[h], want)
            want = mass[b, h].copy() if in_place else np.full(L, 7.0, np.float32)
            want[:n] = 0.0
            want[:len(at)] = mass[b, h][at]
            assert np.array_equal(new_mass[b, h], want, equal_nan=True)
    if raw is not None and not acc.paged:  # the bytes themselves
        for pool, was in zip(kv8_pools(acc), raw):
            for b in range(B):
                n = new_lens[b]
                for h in range(hkv):
                    at = torch.from_numpy(kept[b, h, :n].astype(np.int64)).cuda()
                    assert torch.equal(pool[b, h, :n], was[b, h][at]) and torch.equal(pool[b, h, n:L], was[b, h, n:L])


@pytest.mark.parametrize("kv_format", ["bf16", "e4m3"])
@pytest.mark.parametrize("hkv,d,page", [(2, 64, None), (8, 128, 64), (1, 128, None), (4, 64, 128)])
@pytest.mark.parametrize("keep,sinks,recent", [(1, 0, 0), (100, 4, 32), (63, 0, 63), (64, 64, 0), (257, 1, 1), (600, 0, 0)])
def test_evict(kv_format, hkv, d, page, keep, sinks, recent):
    """Lengths below, at and above the budget, none at all, ties, infinities, NaN, negative masses."""
    rng = np.random.default_rng(hkv * d + keep)
    L = 700
    lens = np.array([0, 1, keep, min(L, keep + 1), 650, 700], np.int32)
    B = len(lens)
    mass = np.exp(2 * rng.standard_normal((B, hkv, L))).astype(np.float32)
    mass[rng.random(mass.shape) < 0.3] = 0.0
    mass[4] = rng.integers(-2, 3, mass[4].shape)  # mostly ties, -0.0 too
    mass[4][rng.random(mass[4].shape) < 0.2] = -0.0
    mass[5][rng.random(mass[5].shape) < 0.1] = np.nan
    mass[5][rng.random(mass[5].shape) < 0.05] = np.inf
    mass[5][rng.random(mass[5].shape) < 0.05] = -np.inf
    with AttentionAccelerator(batch=B, n_q_heads=4 * hkv, n_kv_heads=hkv, head_dim=d, max_seq_len=L, max_q_len=1, kv_format=kv_format,
                              page_size=page) as acc:
        if page:
            scatter_reserve(acc, [L] * B, page)
        for in_place in (False, True):
            check_evict(rng, acc, lens, L, keep, sinks, recent, mass, in_place, kv_format)


@pytest.mark.parametrize("L,keep", [(20000, 18001), (40000, 100), (16384, 16383), (16385, 9000)])
def test_evict_long_sequences(L, keep):
    """More masses than a work-group holds in registers; all equal, and in falling and rising order."""
    rng = np.random.default_rng(L)
    with AttentionAccelerator(batch=2, n_q_heads=4, n_kv_heads=1, head_dim=64, max_seq_len=L, max_q_len=1) as acc:
        lens = np.array([L, L - 3], np.int32)
        for mass in (rng.random((2, 1, L)), np.ones((2, 1, L)), np.stack([np.arange(L)[None], np.arange(L)[None, ::-1]])):
            check_evict(rng, acc, lens, L, keep, min(4, keep), 50, mass.astype(np.float32), True, "bf16")


def test_evict_of_one_layer_and_lengths_out_of_range():
    """Lengths are held to 0 .. max_seq_len, and a layered cache's other layers stay."""
    rng = np.random.default_rng(9)
    L, hkv, d = 130, 2, 64
    with AttentionAccelerator(batch=3, n_q_heads=8, n_kv_heads=hkv, head_dim=d, max_seq_len=L, max_q_len=1, page_size=64, n_layers=2) as acc:
        scatter_reserve(acc, [L] * 3, 64)
        other = bf16_normal(rng, (hkv, L, d))
        for b in range(3):
            acc.load_kv(other, other, b=b)
        acc.select_layer(1)
        mass = rng.random((3, hkv, L)).astype(np.float32)
        check_evict(rng, acc, np.array([-5, 2000, 100], np.int32), L, 77, 2, 3, mass, False, "bf16")
        acc.select_layer(0)
        for b in range(3):
            for t in acc.read_kv(b, 0, L):
                assert np.array_equal(t, other)


def test_evict_rows_of_unmapped_pages():
    """A length past the mapped rows: rows that are not there are zeros where they come to lie, and are not written."""
    rng = np.random.default_rng(10)
    L, hkv, d = 192, 2, 64
    with AttentionAccelerator(batch=2, n_q_heads=8, n_kv_heads=hkv, head_dim=d, max_seq_len=L, max_q_len=1, page_size=64) as acc:
        acc.reserve(0, 64)
        acc.reserve(1, 192)
        k = bf16_normal(rng, (2, hkv, L, d))
        acc.load_kv(k[0][:, :64], k[0][:, :64], b=0)
        acc.load_kv(k[1], k[1], b=1)
        mass = rng.random((2, hkv, L)).astype(np.float32)
        lens = np.array([150, 150], np.int32)
        kept, new_lens, _ = run_evict(acc, mass, lens, 100, 0, 40, True)
        got = [acc.read_kv(0, 0, 64), acc.read_kv(1, 0, L)]
    for b in range(2):
        for h in range(hkv):
            at = lo.evict(mass[b, h, :150].tolist(), 150, 100, 0, 40)
            assert np.array_equal(kept[b, h], at)
            rows = k[b, h].copy()
            if b == 0:
                rows[64:] = 0
            for t in got[b]:
                n = min(100, t.shape[1])
                assert np.array_equal(t[h, :n], rows[at[:n]])
                assert np.array_equal(t[h, n:], k[b, h, n:t.shape[1]])
    assert np.array_equal(new_lens, [100, 100])


@pytest.mark.parametrize("kv_format", ["bf16", "e4m3"])
@pytest.mark.parametrize("d", [64, 128])
def test_rows_whose_scores_are_nan_add_nothing(kv_format, d):
    """A key of NaN makes the lse of the rows that see it NaN: they add nothing, to any key; the others add what they do."""
    rng = np.random.default_rng(31)
    hq, hkv, L, n = 8, 2, 300, 40
    k, v = bf16_normal(rng, (2, hkv, L, d)), bf16_normal(rng, (2, hkv, L, d))
    k[1, 0, 280] = 0x7FC0
    q, qs = bf16_normal(rng, (hq, n, d)), bf16_normal(rng, (2, hq, d))
    qs[0, 3] = 0x7FC0  # a query head of NaN
    with AttentionAccelerator(batch=2, n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=L, max_q_len=n, kv_format=kv_format) as acc:
        for b in range(2):
            acc.load_kv(k[b], v[b], b=b)
        mass = torch.zeros((2, hkv, L), device="cuda")
        lens = dev(np.array([L, L], np.int32))
        lse = np.full((2, hq), 3.0, np.float32)
        lse[0, 3] = lse[1, :4] = np.nan
        qd, ld = dev(qs), dev(lse)
        torch.cuda.synchronize()
        acc.attention_mass_step_device(qd.data_ptr(), lens.data_ptr(), ld.data_ptr(), mass.data_ptr())
        torch.cuda.synchronize()
        got = mass.cpu().numpy()
        for b in range(2):
            kk, l64 = stored(k[b], kv_format), lse[b].astype(np.float64)[:, None]
            kk[np.isnan(kk)] = 0.0
            qq = f64(qs[b])[:, None]
            qq[np.isnan(qq)] = 0.0
            new = lo.mass(qq, kk, l64, acc.scale)
            assert np.all(np.abs(got[b] - new) <= bound(new, qq, kk, l64, acc.scale, 0.0, 1.0))
            assert b == 0 or not got[1, 0].any()
        # a block: the last 40 rows; the 20 from key 280 on see it
        for causal in (True, False):
            lse = np.full((hq, n), 2.0, np.float32)
            lse[:4, 20 if causal else 0:] = np.nan
            m, qd, ld = torch.zeros_like(mass), dev(q), dev(lse)
            torch.cuda.synchronize()
            acc.attention_mass_device(qd.data_ptr(), n, L, ld.data_ptr(), m.data_ptr(), b=1, q_pos_base=L - n, causal=causal)
            torch.cuda.synchronize()
            got = m[1].cpu().numpy()
            seen = np.arange(L) <= L - n + np.arange(n)[:, None] if causal else None
            kk, l64 = stored(k[1], kv_format), lse.astype(np.float64)
            kk[np.isnan(kk)] = 0.0
            new = lo.mass(f64(q), kk, l64, acc.scale, seen)
            assert np.all(np.abs(got - new) <= bound(new, f64(q), kk, l64, acc.scale, 0.0, 1.0))
