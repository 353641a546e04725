"""Decode over a shared prefix (gqa_decode_prefix_device, gqa_decode_append_prefix_device) against float64.

Bound of o: half a step of its rounding (2^-8 of it) and of the weights' (2^-8 of the average of |V|), and fp32: a weight's
exponent is off by D 2^-24 of S = scale * sum |q k| at most and by a few roundings of it (as in test_gpu_budget.py), sums and
joins by a part in 2^-24 for every key and partial.  Bound of lse: the same without the roundings to bf16.
"""
import ctypes

import numpy as np
import pytest

from lara_amd import _lib
from lara_amd.attn_driver import AttentionAccelerator
from oracle import gqa_oracle as orc
from oracle import serving_oracle as so
from tests._gen import bf16_normal, kv_with_outliers
from tests._serving import dev, ptr, scatter_reserve, words

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def f64(w):
    return orc.bf16_u16_to_fp32(w).astype(np.float64)


def stored(x, kv_format):
    return f64(x) if kv_format == "bf16" else so.stored(f64(x))


def near(o, lse, q, k, v, scale):
    """o [H_q, D] words and lse [H_q] of one sequence against all the rows that it attends."""
    want, want_lse, avg = so.decode(q, k, v, scale)
    if k.shape[1] == 0:
        assert not o.any() and np.all(lse == -np.inf)
        return
    s = scale * np.einsum("hd,hld->hl", np.abs(q), np.abs(np.repeat(k, q.shape[0] // k.shape[0], 0))).max()
    exponent = (q.shape[1] * s + 8 * s + 8 + k.shape[1]) * 2.0**-24
    assert np.all(np.abs(f64(o) - want) <= 2.0**-8 * np.abs(want) + (2.0**-8 + 4 * exponent) * avg + 1e-37)
    assert np.all(np.abs(lse - want_lse) <= 2 * exponent + 2.0**-22 * np.abs(want_lse))


TWO_LAUNCHES = 2112  # a context of this length: prefix and own rows in pieces, joined by a second launch


class Batch:
    """An engine whose last slot holds the prefix, and what every sequence's rows are."""

    def __init__(self, rng, hq, hkv, d, prefix, lens, kv_format="bf16", page=None, outliers=0.0, max_seq_len=None):
        self.B, self.prefix, self.kv_format = len(lens) + 1, prefix, kv_format
        self.lens = np.append(lens, 0).astype(np.int32)
        L = max_seq_len or max(prefix, *lens, TWO_LAUNCHES)
        self.acc = AttentionAccelerator(batch=self.B, n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=L, max_q_len=1,
                                        kv_format=kv_format, page_size=page)
        rows = [*lens, prefix]
        if page:
            scatter_reserve(self.acc, rows, page)
        self.k = [kv_with_outliers(rng, (hkv, n, d), fraction=outliers if n else 0.0, factor=8.0) for n in rows]
        self.v = [bf16_normal(rng, (hkv, n, d)) for n in rows]
        for b, n in enumerate(rows):
            if n:
                self.acc.load_kv(self.k[b], self.v[b], b=b)
        self.q, self.k_new, self.v_new = (bf16_normal(rng, (self.B, h, d)) for h in (hq, hkv, hkv))
        self.dev = [dev(t) for t in (self.q, self.k_new, self.v_new)]

    def run(self, shared=None, append=True, lens=None, positions=None, prefix=None, stream=None):
        """One step; shared None: the whole prefix for everyone.  Returns (o, lse) tensors."""
        lens = self.lens if lens is None else lens
        positions = lens - 1 if positions is None else positions
        o = torch.full(self.q.shape, 3, dtype=torch.int16, device="cuda")
        lse = torch.full(self.q.shape[:2], 3.0, device="cuda")
        self.keep = [dev(np.asarray(t, np.int32)) for t in (lens, positions)] + [dev(np.asarray(shared, np.int32)) if shared is not None else None]
        kw = dict(k_rows_ptr=self.dev[1].data_ptr(), v_rows_ptr=self.dev[2].data_ptr(), positions_ptr=self.keep[1].data_ptr()) if append else {}
        self.acc.decode_prefix_device(self.dev[0].data_ptr(), self.B - 1, self.prefix if prefix is None else prefix, self.keep[0].data_ptr(),
                                      o.data_ptr(), prefix_lens_ptr=self.keep[2].data_ptr() if shared is not None else None,
                                      lse_ptr=lse.data_ptr(), stream=stream, **kw)
        return o, lse

    def check(self, o, lse, shared=None, append=True, lens=None, positions=None):
        lens = self.lens if lens is None else lens
        positions = lens - 1 if positions is None else positions
        o, lse = words(o), lse.cpu().numpy()
        kp, vp = (stored(t, self.kv_format) for t in (self.k[-1], self.v[-1]))
        for b in range(self.B):
            p = self.prefix if shared is None else min(max(int(shared[b]), 0), self.prefix)
            p = 0 if b == self.B - 1 else p  # (the prefix's own sequence has its rows alone)
            n = int(lens[b])
            k, v = self.k[b][:, :n].copy(), self.v[b][:, :n].copy()
            if append and 0 <= positions[b] < n:
                k[:, positions[b]], v[:, positions[b]] = self.k_new[b], self.v_new[b]
            k, v = (np.concatenate((x[:, :p], stored(y, self.kv_format)), 1) for x, y in zip((kp, vp), (k, v)))
            near(o[b], lse[b], f64(self.q[b]), k, v, self.acc.scale)


@pytest.mark.parametrize("kv_format", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq,hkv,d,page", [(8, 2, 64, None), (32, 8, 128, None), (32, 2, 64, 64), (16, 8, 128, 128), (64, 8, 128, 64),
                                           (4, 4, 64, None), (6, 2, 128, None)])
@pytest.mark.parametrize("prefix", [0, 1, 64, 337])
def test_step(kv_format, hq, hkv, d, page, prefix):
    """Own lengths from none on, tiles that end inside a piece, rows appended and cached; every group's width."""
    if hq == 6 and kv_format == "bf16":
        pytest.skip("a bf16 engine has no groups of 3")
    rng = np.random.default_rng(hq * d + prefix)
    batch = Batch(rng, hq, hkv, d, prefix, [0, 1, 31, 32, 33, 64, 200], kv_format, page, outliers=0.02)
    with batch.acc:
        shared = np.array([prefix] * 7 + [0])
        batch.check(*batch.run(shared, append=False), shared, append=False)
        batch.check(*batch.run(shared), shared)
        for b in range(batch.B - 1):  # the appended row is in the cache
            if batch.lens[b]:
                k, v = batch.acc.read_kv(b, batch.lens[b] - 1, 1)
                assert np.array_equal(f64(k[:, 0]), stored(batch.k_new[b], kv_format)) and np.array_equal(f64(v[:, 0]), stored(batch.v_new[b], kv_format))


@pytest.mark.parametrize("kv_format", ["bf16", "e4m3"])
@pytest.mark.parametrize("B,hq,hkv,d,prefix", [(1, 8, 2, 64, 1000), (9, 8, 2, 64, 3001), (16, 32, 8, 128, 2100), (33, 16, 1, 128, 777),
                                               (40, 8, 2, 64, 5000), (130, 8, 2, 64, 700)])
def test_batches(kv_format, B, hq, hkv, d, prefix):
    """One to several row blocks a kv head, several pieces; sequences with a part of the prefix or none of it."""
    rng = np.random.default_rng(B + prefix)
    lens = rng.integers(0, 90, B)
    lens[B // 2] = 500
    batch = Batch(rng, hq, hkv, d, prefix, list(lens), kv_format)
    with batch.acc:
        for shared in (None, np.append(rng.integers(0, prefix + 1, B), 0), np.append(rng.choice([0, prefix, prefix + 9, -4], B), 0)):
            batch.check(*batch.run(shared), shared)


def test_words_do_not_depend_on_the_others():
    """A sequence's output is the same whatever the lengths of the batch's others beside it, where the pieces are."""
    rng = np.random.default_rng(12)
    batch = Batch(rng, 8, 2, 64, 500, [10, 80, 33])
    with batch.acc:
        a = batch.run(np.array([500, 500, 500, 0]))
        b = batch.run(np.array([500, 0, 7, 0]), lens=np.array([10, 0, 33, 0], np.int32))
        torch.cuda.synchronize()
        assert torch.equal(a[0][0], b[0][0]) and torch.equal(a[1][0], b[1][0])


def test_many_own_rows_and_more_sequences_than_a_wave():
    """Own rows whose pieces outgrow 64 keys, and a batch of several windows of 64 sequences."""
    rng = np.random.default_rng(13)
    lens = np.zeros(150, int)
    lens[[0, 63, 64, 100, 149]] = 1, 3000, 60000, 65, 40000
    batch = Batch(rng, 8, 4, 64, 100, list(lens), page=64, max_seq_len=60000)
    with batch.acc:
        shared = np.append(np.arange(150) % 101, 0)
        batch.check(*batch.run(shared), shared)


@pytest.mark.parametrize("kv_format", ["bf16", "e4m3"])
def test_rows_that_are_not_seen_do_not_reach(kv_format):
    """Infinities and NaN in K and V: in the prefix behind prefix_len and, inside it, in rows that some sequences see and
    others do not; behind own lengths."""
    rng = np.random.default_rng(14)
    nan, inf = 0x7FC0, 0x7F80
    batch = Batch(rng, 8, 2, 64, 300, [5, 40, 64, 100, 7])
    if kv_format == "e4m3":
        batch.acc.close()
        batch = Batch(rng, 8, 2, 64, 300, [5, 40, 64, 100, 7], "e4m3")
    with batch.acc:
        shared = np.array([100, 140, 139, 200, 0, 0])
        for at, word in ((139, nan), (150, inf), (250, nan)):
            batch.v[-1][:, at, 3] = word
            batch.k[-1][:, at, 5] = word
        batch.acc.load_kv(batch.k[-1], batch.v[-1], b=batch.B - 1)
        for b in range(5):
            n = batch.lens[b]
            bad = np.full((2, 300 - n, 64), nan, np.uint16)
            batch.acc.load_kv(bad, bad, b=b, start_pos=int(n))
        o, lse = batch.run(shared, prefix=200)
        torch.cuda.synchronize()
        seen = np.array([False, True, False, True, False, False])
        got, got_lse = words(o), lse.cpu().numpy()
        assert np.all(np.isnan(f64(got[seen])).all(-1)) and np.all(np.isnan(got_lse[seen]))  # (a score of NaN)
        clean_k, clean_v = batch.k[-1].copy(), batch.v[-1].copy()
        batch.k[-1][:, [139, 150, 250], 5] = batch.v[-1][:, [139, 150, 250], 3] = 0
        whole = o.clone()
        whole[torch.from_numpy(seen).cuda()] = 0
        for b in np.flatnonzero(~seen):
            p, n = int(shared[b]), int(batch.lens[b])
            k, v = batch.k[b][:, :n].copy(), batch.v[b][:, :n].copy()
            if n:
                k[:, -1], v[:, -1] = batch.k_new[b], batch.v_new[b]
            k, v = (np.concatenate((stored(x[:, :p], kv_format), stored(y, kv_format)), 1) for x, y in ((batch.k[-1], k), (batch.v[-1], v)))
            near(got[b], got_lse[b], f64(batch.q[b]), k, v, batch.acc.scale)
        # V alone: what is not finite stays in its dim, for those who see it
        batch.k[-1] = clean_k
        batch.k[-1][:, [139, 150, 250], 5] = 0
        batch.acc.load_kv(batch.k[-1], clean_v, b=batch.B - 1)
        o, lse = batch.run(shared, prefix=200)
        torch.cuda.synchronize()
        got = f64(words(o))
        assert np.isfinite(lse.cpu().numpy()[:5]).all()
        bad = np.zeros(got.shape, bool)
        if kv_format == "bf16":
            bad[seen, :, 3] = True
            assert np.array_equal(~np.isfinite(got), bad)
            assert np.all(np.isnan(got[3, :, 3]))  # NaN, and an infinity beside it
        else:  # (rows of the 8-bit cache hold NaN for both)
            bad[seen, :, 3] = True
            assert np.array_equal(np.isnan(got), bad)


def test_a_prefix_that_goes_on_and_rows_not_appended_to_it():
    """The prefix's own sequence decodes behind it; a position inside the prefix is not written; positions out of range are
    none; positions that are not the last row."""
    rng = np.random.default_rng(15)
    batch = Batch(rng, 8, 2, 128, 130, [20, 9, 64], max_seq_len=200)
    with batch.acc:
        hold = bf16_normal(rng, (2, 20, 128))
        batch.acc.load_kv(hold, hold, b=3, start_pos=130)
        batch.k[3], batch.v[3] = np.concatenate((batch.k[3], hold), 1), np.concatenate((batch.v[3], hold), 1)
        lens = np.array([20, 9, 64, 150], np.int32)
        shared = np.array([130, 130, 50, 130])
        pos = np.array([4, 200, 64, 149], np.int32)  # inside; out of range; written but not attended
        batch.check(*batch.run(shared, lens=lens, positions=pos), shared, lens=lens, positions=pos)
        assert np.array_equal(batch.acc.read_kv(2, 64, 1)[0][:, 0], batch.k_new[2])
        assert np.array_equal(batch.acc.read_kv(3, 149, 1)[1][:, 0], batch.v_new[3])
        before = batch.acc.read_kv(3, 0, 150)
        pos[3] = 129
        batch.k[3][:, 149], batch.v[3][:, 149] = batch.k_new[3], batch.v_new[3]
        batch.k[0][:, 4], batch.v[0][:, 4] = batch.k_new[0], batch.v_new[0]
        o, lse = batch.run(shared, lens=lens, positions=pos)
        batch.check(o, lse, shared, append=False, lens=lens)
        for a, b in zip(before, batch.acc.read_kv(3, 0, 150)):
            assert np.array_equal(a, b)


def test_equals_decode_without_a_prefix():
    """prefix_len 0 is decode: within the same bounds, and the same rows in the cache."""
    rng = np.random.default_rng(16)
    batch = Batch(rng, 32, 8, 128, 0, [300, 17, 1])
    with batch.acc:
        batch.check(*batch.run(), None)
        batch.check(*batch.run(np.array([5, -1, 2**31 - 1, 0])), None)


def test_unmapped_rows_are_zeros():
    """Own rows past the mapped pages count as rows of zeros, as in decode; a prefix past them is refused."""
    rng = np.random.default_rng(17)
    batch = Batch(rng, 8, 2, 64, 100, [64, 10], page=64, max_seq_len=256)
    with batch.acc:
        lens = np.array([100, 10, 0], np.int32)
        batch.k[0], batch.v[0] = (np.concatenate((t, np.zeros((2, 36, 64), np.uint16)), 1) for t in (batch.k[0], batch.v[0]))
        batch.check(*batch.run(append=False, lens=lens), append=False, lens=lens)
        with pytest.raises(_lib.GqaError) as e:
            batch.run(prefix=129)
        assert e.value.code == _lib.GQA_ERR_RANGE


def test_refusals():
    rng = np.random.default_rng(18)
    batch = Batch(rng, 8, 2, 64, 64, [10, 3], max_seq_len=64)
    lib, E = batch.acc._lib, _lib
    q, k, v = (ptr(t) for t in batch.dev)
    i32 = torch.zeros(8, dtype=torch.int32, device="cuda")
    o, lse = torch.zeros(batch.q.shape, dtype=torch.int16, device="cuda"), torch.zeros(batch.q.shape[:2], device="cuda")
    off = lambda t, n: ctypes.c_void_p(t.data_ptr() + n)  # noqa: E731
    kc, vc, cap = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_int32()
    lib.gqa_cache_pointers(batch.acc._ctx, ctypes.byref(kc), ctypes.byref(vc), ctypes.byref(cap))
    with batch.acc:
        def rc(**kw):
            a = dict(q=q, k=k, v=v, pos=ptr(i32), b=2, n=64, shared=ptr(i32), lens=ptr(i32), o=ptr(o), lse=ptr(lse))
            a.update(kw)
            return lib.gqa_decode_append_prefix_device(batch.acc._ctx, a["q"], a["k"], a["v"], a["pos"], a["b"], a["n"], a["shared"], a["lens"],
                                                       a["o"], a["lse"], None)

        for name in ("q", "k", "v", "pos", "lens", "o"):
            assert rc(**{name: None}) == E.GQA_ERR_NULL, name
        for name, t in (("q", batch.dev[0]), ("k", batch.dev[1]), ("v", batch.dev[2])):
            assert rc(**{name: off(t, 2)}) == E.GQA_ERR_RANGE, name
        for name, t in (("pos", i32), ("shared", i32), ("lens", i32), ("lse", lse)):
            assert rc(**{name: off(t, 2)}) == E.GQA_ERR_RANGE, name
        assert rc(o=off(o, 1)) == E.GQA_ERR_RANGE and rc(o=kc) == E.GQA_ERR_RANGE and rc(lse=vc) == E.GQA_ERR_RANGE
        assert rc(b=3) == E.GQA_ERR_STREAM_DEST and rc(b=-1) == E.GQA_ERR_STREAM_DEST
        assert rc(n=65) == E.GQA_ERR_RANGE and rc(n=-1) == E.GQA_ERR_RANGE
        assert lib.gqa_decode_prefix_device(None, q, 2, 64, None, ptr(i32), ptr(o), None, None) == E.GQA_ERR_NULL
        with pytest.raises(ValueError):
            batch.acc.decode_prefix_device(batch.dev[0].data_ptr(), 2, 64, i32.data_ptr(), o.data_ptr(), k_rows_ptr=batch.dev[1].data_ptr())
        assert rc(shared=None, lse=None) == 0
        torch.cuda.synchronize()


@pytest.mark.parametrize("B,prefix_b", [(1, 0), (6, 0), (6, 2), (70, 33)])
def test_any_sequence_can_hold_the_prefix(B, prefix_b):
    """The first, one in the middle, one behind a window of 32 rows; the only one, which has its own rows alone."""
    rng = np.random.default_rng(B + prefix_b)
    hq, hkv, d, n = 8, 2, 64, 150
    lens = rng.integers(0, 40, B).astype(np.int32)
    lens[prefix_b] = 170
    with AttentionAccelerator(batch=B, n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=200, max_q_len=1) as acc:
        k, v = (bf16_normal(rng, (B, hkv, 200, d)) for _ in range(2))
        for b in range(B):
            acc.load_kv(k[b], v[b], b=b)
        q = bf16_normal(rng, (B, hq, d))
        qd, ln = dev(q), dev(lens)
        o, lse = torch.zeros((B, hq, d), dtype=torch.int16, device="cuda"), torch.zeros((B, hq), device="cuda")
        torch.cuda.synchronize()
        acc.decode_prefix_device(qd.data_ptr(), prefix_b, n, ln.data_ptr(), o.data_ptr(), lse_ptr=lse.data_ptr())
        torch.cuda.synchronize()
        for b in range(B):
            p = 0 if b == prefix_b else n
            kk, vv = (np.concatenate((f64(t[prefix_b][:, :p]), f64(t[b][:, :lens[b]])), 1) for t in (k, v))
            near(words(o)[b], lse.cpu().numpy()[b], f64(q[b]), kk, vv, acc.scale)


@pytest.mark.parametrize("kv_format", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq,hkv,d,page", [(8, 2, 64, None), (32, 8, 128, None), (32, 2, 64, 64), (16, 8, 128, 128), (64, 8, 128, 64),
                                           (4, 4, 64, None), (6, 2, 128, None), (16, 1, 128, 64)])
@pytest.mark.parametrize("prefix", [0, 1, 64, 337])
def test_short_contexts_take_one_launch(kv_format, hq, hkv, d, page, prefix):
    """The same steps where a work-group takes all of a sequence's keys."""
    if hq == 6 and kv_format == "bf16":
        pytest.skip("a bf16 engine has no groups of 3")
    rng = np.random.default_rng(hq * d + prefix + 1)
    batch = Batch(rng, hq, hkv, d, prefix, [0, 1, 31, 32, 33, 64, 200], kv_format, page, outliers=0.02, max_seq_len=400)
    with batch.acc:
        shared = np.array([prefix] * 3 + [prefix // 2, 0, -3, prefix + 5, 0])
        batch.check(*batch.run(shared, append=False), shared, append=False)
        batch.check(*batch.run(shared), shared)
        batch.check(*batch.run(append=False, lens=np.zeros(8, np.int32)), append=False, lens=np.zeros(8, np.int32))
        for b in range(batch.B - 1):  # the appended row is in the cache
            if batch.lens[b]:
                k, v = batch.acc.read_kv(b, batch.lens[b] - 1, 1)
                assert np.array_equal(f64(k[:, 0]), stored(batch.k_new[b], kv_format)) and np.array_equal(f64(v[:, 0]), stored(batch.v_new[b], kv_format))


@pytest.mark.parametrize("L", [400, TWO_LAUNCHES])
@pytest.mark.parametrize("kv_format", ["bf16", "e4m3"])
def test_values_of_other_sequences_and_an_output_of_two_byte_alignment(kv_format, L):
    """Infinities and NaN of the prefix behind what a sequence sees, and of rows behind own lengths; o at an odd word."""
    rng = np.random.default_rng(19)
    nan = 0x7FC0
    batch = Batch(rng, 8, 2, 128, 100, [5, 40, 0], kv_format, max_seq_len=L)
    with batch.acc:
        shared = np.array([50, 70, 33, 0])
        bad = np.full((2, 30, 128), nan, np.uint16)
        batch.acc.load_kv(bad, bad, b=3, start_pos=70)
        for b in range(3):
            batch.acc.load_kv(bad, bad, b=b, start_pos=int(batch.lens[b]))
        held = torch.full((batch.q.size + 8,), 3, dtype=torch.int16, device="cuda")
        lens, sh = dev(batch.lens), dev(shared.astype(np.int32))
        torch.cuda.synchronize()
        for at in (0, 1, 3):
            held.fill_(3)
            torch.cuda.synchronize()
            batch.acc.decode_prefix_device(batch.dev[0].data_ptr(), 3, 100, lens.data_ptr(), held.data_ptr() + 2 * at, prefix_lens_ptr=sh.data_ptr())
            torch.cuda.synchronize()
            o = words(held[at:at + batch.q.size]).reshape(batch.q.shape)
            assert held[:at].eq(3).all() and held[at + batch.q.size:].eq(3).all()
            for b in range(3):
                k, v = (np.concatenate((stored(t[3][:, :shared[b]], kv_format), stored(t[b][:, :batch.lens[b]], kv_format)), 1) for t in (batch.k, batch.v))
                want, want_lse, _ = so.decode(f64(batch.q[b]), k, v, batch.acc.scale)
                near(o[b], want_lse, f64(batch.q[b]), k, v, batch.acc.scale)
