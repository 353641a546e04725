"""The E4M3 K/V cache on the GPU: rows as written and read back, decode and prefill over them.

Rows are compared exactly (value = code * 2^k, the oracle's nearest codes).  Attention is compared with float64 attention
over the stored rows.  Bound of an output element: its own rounding to bf16 (half a step, 2^-8 of it at most), the
weights' p * 2^k rounded to bf16 before the product (2^-8 of the average A of |V| under the weights), and fp32: a score is
a sum of D <= 128 products of |q k| summing to below 2^7 in the scaled log2 units here, off by at most 2^-24 * 2^7 * 2^4
for its at most 16 sequential additions, so p by 2^-13, which also covers exp2 and the sums: 2^-13 of A.  The
log-sum-exp is off by 2^-13 likewise, plus its own rounding.
"""
import ctypes

import numpy as np
import pytest

from lara_amd import _lib
from lara_amd.attn_driver import AttentionAccelerator
from oracle import gqa_oracle as orc
from oracle import serving_oracle as so
from tests._gen import bf16_normal
from tests._serving import call, dev, kv8_pools, ptr, scatter_reserve, words

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def f64(w):
    return orc.bf16_u16_to_fp32(w).astype(np.float64)


def engine(**kw):
    return AttentionAccelerator(kv_format="e4m3", **kw)


def rows(rng, shape, spread=1.0):
    """bf16 rows of several magnitudes."""
    x = rng.standard_normal(shape) * np.exp(spread * rng.standard_normal(shape[:-1] + (1,)))
    return orc.bf16_rne(x.astype(np.float32))


def close(o, lse, ref):
    want, want_lse, avg = ref
    bound = 2.0**-8 * np.abs(want) + (2.0**-8 + 2.0**-13) * avg
    assert np.all(np.abs(f64(o) - want) <= bound), float((np.abs(f64(o) - want) / np.maximum(bound, 1e-300)).max())
    if lse is not None:
        some = np.isfinite(want_lse)
        assert np.array_equal(np.isfinite(lse), some) and np.all(lse[~some] == -np.inf)
        assert np.all(np.abs(lse[some] - want_lse[some]) <= 2.0**-13 + 2.0**-22 * np.abs(want_lse[some]))


# ---- rows ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("d", [64, 128])
def test_every_bf16_word_is_stored_as_the_nearest_code(d):
    """All 65536 words, mixed into rows of near magnitudes and of all magnitudes, through both write paths; the codes and
    scale bytes themselves too."""
    rng = np.random.default_rng(d)
    near = np.arange(65536, dtype=np.uint16).reshape(-1, d)
    mixed = rng.permutation(65536).astype(np.uint16).reshape(-1, d)
    mixed[::2] &= 0xBFFF  # half of the rows without the largest magnitudes, infinities and NaN
    n = near.shape[0]
    with engine(n_q_heads=2, n_kv_heads=1, head_dim=d, max_seq_len=n) as acc:
        acc.load_kv(near[None], mixed[None])
        k, v = acc.read_kv(0, 0, n)
        pools = [p.cpu().numpy() for p in kv8_pools(acc)]
        for src, got, codes, scale in ((near, k, pools[0], pools[2]), (mixed, v, pools[1], pools[3])):
            with np.errstate(invalid="ignore"):
                want, want_scale = so.e4m3_row(f64(src))
            assert np.array_equal(so.e4m3_values()[codes[0, 0, :n]], want, equal_nan=True)
            assert np.array_equal(2.0 ** (scale[0, 0, :n].astype(float) - 127), want_scale)
            assert np.array_equal(f64(got[0]), want * want_scale[:, None], equal_nan=True)


@pytest.mark.parametrize("page", [None, 64])
def test_load_append_and_read_back(page):
    rng = np.random.default_rng(7)
    B, L = 3, 200
    with engine(batch=B, n_q_heads=4, n_kv_heads=2, head_dim=64, max_seq_len=L, page_size=page) as acc:
        if page:
            scatter_reserve(acc, [L] * B, page)
        k, v = rows(rng, (B, 2, L, 64), 3.0), rows(rng, (B, 2, L, 64), 3.0)
        for b in range(B):
            acc.load_kv(k[b, :, :150], v[b, :, :150], b=b)
        acc.load_kv(k[1, :, 63:66], v[1, :, 63:66], b=1, start_pos=63)  # across a page's end
        before = acc.read_kv(0, 0, L)
        kr, vr = rows(rng, (B, 2, 64)), rows(rng, (B, 2, 64))
        acc.append_kv(kr, vr, [-1, 150, L - 1])
        k[1, :, 150], v[1, :, 150], k[2, :, L - 1], v[2, :, L - 1] = kr[1], vr[1], kr[2], vr[2]
        written = np.zeros((B, L), bool)
        written[:, :150] = written[1, 150] = written[2, L - 1] = True
        for b in range(B):
            kg, vg = acc.read_kv(b, 0, L)
            for got, src in ((kg, k[b]), (vg, v[b])):
                want = np.where(written[b][:, None], so.stored(f64(src)), 0.0)
                assert np.array_equal(f64(got), want)
        after = acc.read_kv(0, 0, L)
        assert np.array_equal(before[0], after[0]) and np.array_equal(before[1], after[1])  # position -1 writes nothing
        # the device form, into rows of its own
        kd, vd = (torch.full((2, 70, 64), 7, dtype=torch.int16, device="cuda") for _ in range(2))
        acc.read_kv_device(2, 130, 70, kd.data_ptr(), vd.data_ptr())
        kg, vg = acc.read_kv(2, 130, 70)
        torch.cuda.synchronize()
        assert np.array_equal(words(kd), kg) and np.array_equal(words(vd), vg)


def test_read_kv_device_of_a_bf16_cache():
    rng = np.random.default_rng(8)
    for page in (None, 64):
        with AttentionAccelerator(batch=2, n_q_heads=4, n_kv_heads=2, head_dim=64, max_seq_len=130, page_size=page) as acc:
            if page:
                scatter_reserve(acc, [130, 130], 64)
            k, v = bf16_normal(rng, (2, 130, 64)), bf16_normal(rng, (2, 130, 64))
            acc.load_kv(k, v, b=1)
            kd, vd = (torch.zeros((2, 99, 64), dtype=torch.int16, device="cuda") for _ in range(2))
            acc.read_kv_device(1, 31, 99, kd.data_ptr(), vd.data_ptr())
            torch.cuda.synchronize()
            assert np.array_equal(words(kd), k[:, 31:]) and np.array_equal(words(vd), v[:, 31:])


def test_layers_and_recycled_pages_keep_apart():
    rng = np.random.default_rng(9)
    with engine(batch=2, n_q_heads=4, n_kv_heads=2, head_dim=64, max_seq_len=128, page_size=64, n_pages=2, n_layers=3) as acc:
        acc.reserve(0, 128)
        want = []
        for layer in range(3):
            acc.select_layer(layer)
            k, v = rows(rng, (2, 128, 64), 2.0), rows(rng, (2, 128, 64), 2.0)
            acc.load_kv(k, v)
            want.append((k, v))
        for layer in (1, 0, 2):
            acc.select_layer(layer)
            kg, vg = acc.read_kv(0, 0, 128)
            assert np.array_equal(f64(kg), so.stored(f64(want[layer][0])))
            assert np.array_equal(f64(vg), so.stored(f64(want[layer][1])))
        # a page that held NaN rows, handed to another sequence: rows past its length do not count
        acc.select_layer(0)
        acc.load_kv(np.full((2, 128, 64), 0x7FC0, np.uint16), np.full((2, 128, 64), 0x7FC0, np.uint16))
        acc.release(0)
        acc.reserve(1, 64)
        k, v, q = rows(rng, (2, 5, 64)), rows(rng, (2, 5, 64)), bf16_normal(rng, (2, 4, 64))
        acc.load_kv(k, v, b=1)
        o, lse = acc.decode_step(q, [0, 5], return_lse=True)
        close(o[1], lse[1], so.decode(f64(q[1]), so.stored(f64(k)), so.stored(f64(v)), acc.scale))
        assert not o[0].any() and np.all(lse[0] == -np.inf)


# ---- decode -------------------------------------------------------------------------------------------

SHAPES = [(4, 4, 64), (8, 2, 64), (12, 4, 128), (32, 8, 128), (16, 2, 128), (32, 2, 64), (16, 1, 128), (9, 3, 64)]


@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("page", [None, 64])
def test_decode_against_float64(hq, hkv, d, page):
    """Ragged batches: rows of length 0 and 1, rounds' and pages' ends, a row appended in the launch, idle slots."""
    rng = np.random.default_rng(hq * 1000 + hkv * 10 + d)
    lens = [0, 1, 31, 32, 33, 64, 65, 250, 257, 700]
    B, L = len(lens), 704
    with engine(batch=B, n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=L, page_size=page) as acc:
        if page:
            scatter_reserve(acc, [max(1, n) for n in lens], page)
        k, v = rows(rng, (B, hkv, L, d)), rows(rng, (B, hkv, L, d))
        for b, n in enumerate(lens):
            if n:
                acc.load_kv(k[b, :, :n], v[b, :, :n], b=b)
        q = bf16_normal(rng, (B, hq, d))
        o, lse = acc.decode_step(q, lens, return_lse=True)
        for b, n in enumerate(lens):
            close(o[b], lse[b], so.decode(f64(q[b]), so.stored(f64(k[b, :, :n])), so.stored(f64(v[b, :, :n])), acc.scale))
        # with rows appended by the launch: at the end, inside (rewritten), none
        pos = np.array([n - 1 for n in lens], np.int32)
        pos[7], pos[8] = 100, -1
        kr, vr = rows(rng, (B, hkv, d), 2.0), rows(rng, (B, hkv, d), 2.0)
        o, lse = acc.decode_step(q, lens, k_rows=kr, v_rows=vr, positions=pos, return_lse=True)
        for b, n in enumerate(lens):
            if pos[b] >= 0:
                k[b, :, pos[b]], v[b, :, pos[b]] = kr[b], vr[b]
            close(o[b], lse[b], so.decode(f64(q[b]), so.stored(f64(k[b, :, :n])), so.stored(f64(v[b, :, :n])), acc.scale))
            if n:
                kg, vg = acc.read_kv(b, 0, n)
                assert np.array_equal(f64(kg), so.stored(f64(k[b, :, :n])))
                assert np.array_equal(f64(vg), so.stored(f64(v[b, :, :n])))


@pytest.mark.parametrize("d,hq", [(128, 16), (64, 32)])
def test_decode_splits_meet(d, hq):
    """One sequence over many splits, merged in the launch and by a second one (the same words), and steps repeated: the
    counters are zero again after each.  A row at the end of a long cache, appended past the attended length too."""
    rng = np.random.default_rng(d)
    L = 3000
    with engine(n_q_heads=hq, n_kv_heads=2, head_dim=d, max_seq_len=L) as acc:
        k, v, q = rows(rng, (2, L, d)), rows(rng, (2, L, d)), bf16_normal(rng, (1, hq, d))
        acc.load_kv(k, v)
        ref = so.decode(f64(q[0]), so.stored(f64(k)), so.stored(f64(v)), acc.scale)
        for chunk in (0, 256, 320, 1024, 2048):
            call("gqa_set_option", acc._ctx, _lib.GQA_OPT_DECODE_CHUNK, chunk)
            seen = []
            for merge in (_lib.GQA_DECODE_MERGE_FUSED, _lib.GQA_DECODE_MERGE_LAUNCH, _lib.GQA_DECODE_MERGE_AUTO,
                          _lib.GQA_DECODE_MERGE_FUSED):
                call("gqa_set_option", acc._ctx, _lib.GQA_OPT_DECODE_MERGE, merge)
                o, lse = acc.decode_step(q, [L], return_lse=True)
                close(o[0], lse[0], ref)
                seen.append((o, lse))
            for o, lse in (seen[1], seen[3]):
                if chunk:
                    assert np.array_equal(o, seen[0][0]) and np.array_equal(lse, seen[0][1]), chunk
        kr, vr = rows(rng, (1, 2, d)), rows(rng, (1, 2, d))
        for n in (1000, L):  # the appended row outside and inside what is attended
            o, lse = acc.decode_step(q, [n], k_rows=kr, v_rows=vr, positions=[L - 1], return_lse=True)
            k[:, L - 1], v[:, L - 1] = kr[0], vr[0]
            close(o[0], lse[0], so.decode(f64(q[0]), so.stored(f64(k[:, :n])), so.stored(f64(v[:, :n])), acc.scale))


def test_decode_of_a_large_ragged_batch_takes_every_row_once():
    """More sequences than a wave has lanes, lengths by ticket, repeated: every output against float64."""
    rng = np.random.default_rng(12)
    B = 70
    lens = rng.integers(0, 300, B)
    lens[5] = 300
    with engine(batch=B, n_q_heads=4, n_kv_heads=1, head_dim=64, max_seq_len=300) as acc:
        k, v, q = rows(rng, (B, 1, 300, 64)), rows(rng, (B, 1, 300, 64)), bf16_normal(rng, (B, 4, 64))
        for b in range(B):
            acc.load_kv(k[b], v[b], b=b)
        first = None
        for _ in range(3):
            o, lse = acc.decode_step(q, lens, return_lse=True)
            if first is None:
                for b, n in enumerate(lens):
                    close(o[b], lse[b], so.decode(f64(q[b]), so.stored(f64(k[b, :, :n])), so.stored(f64(v[b, :, :n])), acc.scale))
                first = (o, lse)
            assert np.array_equal(o, first[0]) and np.array_equal(lse, first[1])


@pytest.mark.parametrize("hq,hkv,d,L", [(8, 4, 64, 2112), (4, 4, 64, 2112), (64, 4, 64, 2112), (20, 4, 128, 1088), (32, 4, 128, 1088)])
@pytest.mark.parametrize("page", [None, 64])
def test_decode_in_equal_runs_against_float64(hq, hkv, d, L, page):
    """Batches that share their keys out in equal runs: lengths around pieces' and rounds' ends, rows appended at the end,
    inside and past what is attended, idle slots; repeated steps give the same words."""
    rng = np.random.default_rng(hq * 100 + d)
    lens = [0, 1, 2, 63, 64, 65, 255, 256, 257, 320, 321, 384, 511, 513, 576, 577, 800, 1023, L - 1, L]
    B = len(lens)
    with engine(batch=B, n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=L, page_size=page) as acc:
        if page:
            scatter_reserve(acc, [max(1, n) for n in lens], page)
        k, v = rows(rng, (B, hkv, L, d)), rows(rng, (B, hkv, L, d))
        for b, n in enumerate(lens):
            if n:
                acc.load_kv(k[b, :, :n], v[b, :, :n], b=b)
        q = bf16_normal(rng, (B, hq, d))
        first = acc.decode_step(q, lens, return_lse=True)
        for b, n in enumerate(lens):
            close(first[0][b], first[1][b], so.decode(f64(q[b]), so.stored(f64(k[b, :, :n])), so.stored(f64(v[b, :, :n])), acc.scale))
        for _ in range(3):
            again = acc.decode_step(q, lens, return_lse=True)
            assert np.array_equal(again[0], first[0]) and np.array_equal(again[1], first[1])
        pos, attended = np.array([n - 1 for n in lens], np.int32), list(lens)
        pos[7], pos[8], pos[16] = 100, -1, 0
        attended[18] = 700  # (its row, the last of the cache, is stored but not attended)
        kr, vr = rows(rng, (B, hkv, d), 2.0), rows(rng, (B, hkv, d), 2.0)
        o, lse = acc.decode_step(q, attended, k_rows=kr, v_rows=vr, positions=pos, return_lse=True)
        for b, n in enumerate(attended):
            if pos[b] >= 0:
                k[b, :, pos[b]], v[b, :, pos[b]] = kr[b], vr[b]
            close(o[b], lse[b], so.decode(f64(q[b]), so.stored(f64(k[b, :, :n])), so.stored(f64(v[b, :, :n])), acc.scale))
            if lens[b]:
                kg, vg = acc.read_kv(b, 0, lens[b])
                assert np.array_equal(f64(kg), so.stored(f64(k[b, :, : lens[b]])))
                assert np.array_equal(f64(vg), so.stored(f64(v[b, :, : lens[b]])))


@pytest.mark.parametrize("full", [(), (3,), tuple(range(150))])
def test_decode_in_equal_runs_of_many_sequences(full):
    """More sequences than a work-group has lanes; next to no work, one long sequence, all of them long."""
    rng = np.random.default_rng(31)
    B, L, d = 150, 2624, 128
    lens = rng.integers(0, 40, B)
    lens[list(full)] = L if len(full) == 1 else rng.integers(200, 700, len(full))
    with engine(batch=B, n_q_heads=4, n_kv_heads=1, head_dim=d, max_seq_len=L) as acc:
        kv = {}
        for b in range(B):
            kv[b] = rows(rng, (1, int(lens[b]), d)), rows(rng, (1, int(lens[b]), d))
            if lens[b]:
                acc.load_kv(*kv[b], b=b)
        q = bf16_normal(rng, (B, 4, d))
        # (the host's step plans for the longest length given, the device's for the cache: both are taken)
        o, lse = acc.decode_step(q, lens, return_lse=True)
        qd, ld = dev(q), dev(lens.astype(np.int32))
        od, lsed = torch.empty((B, 4, d), dtype=torch.int16, device="cuda"), torch.empty((B, 4), device="cuda")
        call("gqa_decode_device", acc._ctx, ptr(qd), ptr(ld), ptr(od), ptr(lsed), None)
        torch.cuda.synchronize()
        for b, n in enumerate(lens):
            ref = so.decode(f64(q[b]), so.stored(f64(kv[b][0])), so.stored(f64(kv[b][1])), acc.scale)
            close(o[b], lse[b], ref)
            close(words(od)[b], lsed.cpu().numpy()[b], ref)


@pytest.mark.parametrize("batch,L", [(18, 1 << 18), (2, 2400000)])
@pytest.mark.parametrize("page", [None, 64])
def test_rows_past_4_gib_of_a_cache(batch, L, page):
    """K and V of over 2^32 bytes each: rows of the last sequence, written, read, appended and attended to."""
    rng = np.random.default_rng(32)
    hq, hkv, d, n = 16, 8, 128, 1500
    with engine(batch=batch, n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=L, page_size=page) as acc:
        if page:
            for b in range(batch):
                acc.reserve(b, L if b < batch - 1 else n + 1)
        b = batch - 1
        k, v = rows(rng, (hkv, n + 1, d)), rows(rng, (hkv, n + 1, d))
        acc.load_kv(k[:, :n], v[:, :n], b=b)
        lens, pos = np.zeros(batch, np.int32), np.full(batch, -1, np.int32)
        lens[b], pos[b] = n + 1, n
        q = bf16_normal(rng, (batch, hq, d))
        kr, vr = rows(rng, (batch, hkv, d)), rows(rng, (batch, hkv, d))
        kr[b], vr[b] = k[:, n], v[:, n]
        t = [dev(x) for x in (q, kr, vr, pos, lens)]
        o, lse = torch.empty((batch, hq, d), dtype=torch.int16, device="cuda"), torch.empty((batch, hq), device="cuda")
        call("gqa_decode_append_device", acc._ctx, *[ptr(x) for x in t], ptr(o), ptr(lse), None)
        torch.cuda.synchronize()
        close(words(o)[b], lse[b].cpu().numpy(), so.decode(f64(q[b]), so.stored(f64(k)), so.stored(f64(v)), acc.scale))
        kg, vg = acc.read_kv(b, 0, n + 1)
        assert np.array_equal(f64(kg), so.stored(f64(k))) and np.array_equal(f64(vg), so.stored(f64(v)))
        assert not np.any(acc.read_kv(0, 0, 300)[0])  # (what the low 32 bits of their places would have hit)


@pytest.mark.parametrize("page", [None, 64])
def test_two_engines_on_two_streams_at_once(page):
    rng = np.random.default_rng(33)
    B, L = 24, 1600
    kw = dict(batch=B, n_q_heads=16, n_kv_heads=4, head_dim=128, max_seq_len=L, page_size=page)
    with engine(**kw) as x, engine(**kw) as y:
        sides = []
        for eng in (x, y):
            lens = rng.integers(1, L, B)
            if page:
                scatter_reserve(eng, list(lens), page)
            for b in range(B):
                eng.load_kv(rows(rng, (4, lens[b], 128)), rows(rng, (4, lens[b], 128)), b=b)
            q, n = dev(bf16_normal(rng, (B, 16, 128))), dev(lens.astype(np.int32))
            o = [torch.zeros((B, 16, 128), dtype=torch.int16, device="cuda") for _ in range(9)]
            call("gqa_decode_device", eng._ctx, ptr(q), ptr(n), ptr(o[8]), None, None)
            sides.append((eng, q, n, o, torch.cuda.Stream()))
        torch.cuda.synchronize()
        for i in range(8):
            for eng, q, n, o, stream in sides:
                call("gqa_decode_device", eng._ctx, ptr(q), ptr(n), ptr(o[i]), None, ctypes.c_void_p(stream.cuda_stream))
        torch.cuda.synchronize()
        for _, _, _, o, _ in sides:
            assert torch.count_nonzero(o[8]) and all(torch.equal(t, o[8]) for t in o[:8])


def test_equal_runs_in_a_captured_graph():
    """Lengths, positions and rows that change between replays; every replay against the eager step."""
    rng = np.random.default_rng(34)
    B, hkv, L, d = 20, 4, 1600, 128
    kw = dict(batch=B, n_q_heads=16, n_kv_heads=hkv, head_dim=d, max_seq_len=L)
    with engine(**kw) as a, engine(**kw) as e:
        start = rng.integers(0, 1500, B)
        for b in range(B):
            if start[b]:
                k, v = rows(rng, (hkv, start[b], d)), rows(rng, (hkv, start[b], d))
                a.load_kv(k, v, b=b)
                e.load_kv(k, v, b=b)
        lens = dev(start.astype(np.int32))
        buf = [dict(q=torch.zeros((B, 16, d), dtype=torch.int16, device="cuda"), k=torch.zeros((B, hkv, d), dtype=torch.int16, device="cuda"),
                    v=torch.zeros((B, hkv, d), dtype=torch.int16, device="cuda"), pos=lens - 1, lens=lens.clone(),
                    o=torch.zeros((B, 16, d), dtype=torch.int16, device="cuda"), lse=torch.zeros((B, 16), device="cuda")) for _ in range(2)]

        def args(t):
            return [ptr(t[n]) for n in ("q", "k", "v", "pos", "lens", "o", "lse")]

        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            call("gqa_decode_append_device", a._ctx, *args(buf[0]), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        for step in range(6):
            for name, t in (("q", bf16_normal(rng, (B, 16, d))), ("k", rows(rng, (B, hkv, d))), ("v", rows(rng, (B, hkv, d)))):
                for t_buf in buf:
                    t_buf[name].copy_(dev(t))
            idle = int(rng.integers(0, B))
            for t_buf in buf:
                t_buf["pos"] += 1
                t_buf["lens"] += 1
                t_buf["lens"][idle] = 0
                t_buf["pos"][idle] = -1
            _ = torch.randn(256, 256, device="cuda") @ torch.randn(256, 256, device="cuda")
            torch.cuda.synchronize()
            graph.replay()
            call("gqa_decode_append_device", e._ctx, *args(buf[1]), None)
            torch.cuda.synchronize()
            assert torch.equal(buf[0]["o"], buf[1]["o"]) and torch.equal(buf[0]["lse"], buf[1]["lse"])
            assert torch.all(torch.isneginf(buf[0]["lse"][idle])) and not torch.any(buf[0]["o"][idle])


def test_decode_extremes():
    """A dominating key, equal keys, values of very different scales, NaN in rows that are not attended, a key whose scale
    byte is the smallest."""
    rng = np.random.default_rng(13)
    L, d = 100, 128
    with engine(n_q_heads=4, n_kv_heads=1, head_dim=d, max_seq_len=L) as acc:
        k, v, q = rows(rng, (1, L, d)), rows(rng, (1, L, d), 8.0), bf16_normal(rng, (1, 4, d))
        k[0, 17] = orc.bf16_rne((40 * f64(q[0, 0])).astype(np.float32))
        k[0, 30:40] = k[0, 30]
        k[0, 50] = orc.bf16_rne(np.full(d, 1e-38, np.float32))
        k[0, 90:], v[0, 90:] = 0x7FC0, 0x7F80
        acc.load_kv(k, v)
        o, lse = acc.decode_step(q, [90], return_lse=True)
        ref = so.decode(f64(q[0]), so.stored(f64(k[:, :90])), so.stored(f64(v[:, :90])), acc.scale)
        want, want_lse, avg = ref
        # (head 0's score of key 17 is about 40 * 128 / sqrt(128): 2^9 in log2 units, four times the scores of the bound above)
        assert np.all(np.abs(f64(o[0]) - want) <= 2.0**-8 * np.abs(want) + (2.0**-8 + 2.0**-10) * avg)
        assert np.all(np.abs(lse[0] - want_lse) <= 2.0**-10 + 2.0**-22 * np.abs(want_lse))


# ---- prefill and the layer stage ------------------------------------------------------------------------

@pytest.mark.parametrize("hq,hkv,d,page", [(8, 2, 64, None), (32, 8, 128, 64), (8, 8, 128, None)])
def test_prefill_chunks_equal_a_bf16_engine_on_the_stored_rows(hq, hkv, d, page):
    """Each chunk's rows quantised, attended as stored: the words of a bf16 engine that holds the stored rows."""
    rng = np.random.default_rng(hq + d)
    L, step = 300, 100
    kw = dict(n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=L, max_q_len=step)
    with engine(page_size=page, **kw) as acc, AttentionAccelerator(**kw) as ref:
        if page:
            acc.reserve(0, L)
        k, v, q = rows(rng, (hkv, L, d)), rows(rng, (hkv, L, d)), bf16_normal(rng, (hq, L, d))
        ks, vs = (orc.bf16_rne(so.stored(f64(t)).astype(np.float32)) for t in (k, v))
        ref.load_kv(ks, vs)
        for at in range(0, L, step):
            o, lse = acc.prefill_chunk(q[:, at:at + step], q_pos_base=at, k_rows=k[:, at:at + step], v_rows=v[:, at:at + step],
                                       return_lse=True)
            want, want_lse = ref.prefill_chunk(q[:, at:at + step], q_pos_base=at, return_lse=True)
            assert np.array_equal(o, want) and np.array_equal(lse, want_lse)
        assert all(np.array_equal(a, b) for a, b in zip(acc.read_kv(0, 0, L), (ks, vs)))
        o = acc.prefill_chunk(q[:, :37], q_pos_base=0, kv_len=211, causal=False)
        assert np.array_equal(o, ref.prefill_chunk(q[:, :37], q_pos_base=0, kv_len=211, causal=False))
        o = acc.run_attention(q[:, :step], k[:, :step], v[:, :step])
        assert np.array_equal(o, ref.run_attention(q[:, :step], ks[:, :step], vs[:, :step]))


@pytest.mark.parametrize("tokens", [1, 40])
def test_layer_stage_quantises_its_rows(tokens):
    rng = np.random.default_rng(tokens)
    hidden, kw = 1024, dict(n_q_heads=8, n_kv_heads=2, head_dim=64, max_seq_len=100, max_q_len=64)
    x = dev(bf16_normal(rng, (tokens, hidden)))
    w = [dev(bf16_normal(rng, (n, hidden), hidden**-0.5)) for n in (512, 128, 128)]
    gamma = dev(bf16_normal(rng, (hidden,)))
    q = [torch.zeros((8, tokens, 64), dtype=torch.int16, device="cuda") for _ in range(2)]
    with engine(**kw) as acc, AttentionAccelerator(**kw) as ref:
        for eng, out in ((acc, q[0]), (ref, q[1])):
            eng.layer_qkv_device(x.data_ptr(), tokens, hidden, *(t.data_ptr() for t in w), gamma.data_ptr(), out.data_ptr(),
                                 q_pos_base=20, kv_pos_base=20, kv_row0=20)
        for got, want in zip(acc.read_kv(0, 0, 100), ref.read_kv(0, 0, 100)):
            assert np.array_equal(f64(got), so.stored(f64(want)))
        torch.cuda.synchronize()
        assert torch.equal(q[0], q[1])


def test_workspace_passes_between_streams():
    """Prefill calls of several lengths on streams that take turns share the bf16 workspace: each result is that of a
    call alone."""
    rng = np.random.default_rng(15)
    L, n = 1500, 32
    with engine(batch=2, n_q_heads=8, n_kv_heads=2, head_dim=64, max_seq_len=L, max_q_len=n) as acc:
        for b in range(2):
            acc.load_kv(rows(rng, (2, L, 64)), rows(rng, (2, L, 64)), b=b)
        q = dev(bf16_normal(rng, (8, n, 64)))
        cases = [(b, kv) for kv in (1500, 700, 1500) for b in (0, 1)]
        out = [torch.zeros((8, n, 64), dtype=torch.int16, device="cuda") for _ in cases]
        want = []
        for (b, kv), o in zip(cases, out):
            call("gqa_prefill_device", acc._ctx, b, ptr(q), n, kv - n, kv, 0, 1, ptr(o), None, None)
            torch.cuda.synchronize()
            want.append(o.clone())
        streams = [torch.cuda.Stream() for _ in range(3)]
        for o in out:
            o.zero_()
        torch.cuda.synchronize()
        for i, ((b, kv), o) in enumerate(zip(cases, out)):
            call("gqa_prefill_device", acc._ctx, b, ptr(q), n, kv - n, kv, 0, 1, ptr(o), None, ctypes.c_void_p(streams[i % 3].cuda_stream))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


# ---- graphs and refusals ----------------------------------------------------------------------------------

def test_decode_step_in_a_captured_graph_and_a_prepared_step():
    rng = np.random.default_rng(16)
    B, L = 2, 1024
    lens = torch.tensor([300, 900], dtype=torch.int32, device="cuda")
    kw = dict(batch=B, n_q_heads=32, n_kv_heads=8, head_dim=128, max_seq_len=L)
    k, v = rows(rng, (B, 8, 900, 128)), rows(rng, (B, 8, 900, 128))
    with engine(**kw) as a, engine(**kw) as p, engine(**kw) as e:
        engines = (a, p, e)
        for eng in engines:
            for b in range(B):
                eng.load_kv(k[b], v[b], b=b)
        buf = [dict(q=torch.zeros((B, 32, 128), dtype=torch.int16, device="cuda"),
                    k=torch.zeros((B, 8, 128), dtype=torch.int16, device="cuda"),
                    v=torch.zeros((B, 8, 128), dtype=torch.int16, device="cuda"), pos=lens - 1, lens=lens.clone(),
                    o=torch.zeros((B, 32, 128), dtype=torch.int16, device="cuda"), lse=torch.zeros((B, 32), device="cuda"))
               for _ in engines]

        def args(t):
            return [ptr(t[n]) for n in ("q", "k", "v", "pos", "lens", "o", "lse")]

        prepared = ctypes.c_void_p()
        call("gqa_graph_capture_decode_append", p._ctx, *args(buf[1]), ctypes.byref(prepared))
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            call("gqa_decode_append_device", a._ctx, *args(buf[0]), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        try:
            for step in range(4):
                print(f"[kv8 graph] replay {step}", flush=True)
                for name, t in (("q", bf16_normal(rng, (B, 32, 128))), ("k", rows(rng, (B, 8, 128))), ("v", rows(rng, (B, 8, 128)))):
                    for t_buf in buf:
                        t_buf[name].copy_(dev(t))
                for t_buf in buf:
                    t_buf["pos"] += 1
                    t_buf["lens"] += 1
                _ = torch.randn(256, 256, device="cuda") @ torch.randn(256, 256, device="cuda")
                torch.cuda.synchronize()
                graph.replay()
                call("gqa_graph_launch", prepared, None)
                call("gqa_decode_append_device", e._ctx, *args(buf[2]), None)
                torch.cuda.synchronize()
                for t_buf in buf[:2]:
                    assert torch.equal(t_buf["o"], buf[2]["o"]) and torch.equal(t_buf["lse"], buf[2]["lse"])
                for b in range(B):
                    got = [eng.read_kv(b, 0, int(lens[b]) + step + 1) for eng in engines]
                    assert all(np.array_equal(g[i], got[2][i]) for g in got for i in (0, 1))
        finally:
            _lib.lib().gqa_graph_destroy(prepared)


def test_refusals():
    lib = _lib.lib()
    t = torch.zeros(1 << 16, dtype=torch.int16, device="cuda")
    at, odd = ptr(t), ctypes.c_void_p(t.data_ptr() + 2)
    with engine(batch=2, n_q_heads=8, n_kv_heads=2, head_dim=64, max_seq_len=100, page_size=64, n_pages=2) as acc:
        c = acc._ctx
        assert lib.gqa_set_option(c, _lib.GQA_OPT_NUMERICS, _lib.GQA_NUMERICS_KV260) == _lib.GQA_ERR_UNSUPPORTED
        acc.reserve(0, 64)
        assert lib.gqa_load_kv_device(c, 0, 0, 65, at, at, None) == _lib.GQA_ERR_RANGE  # the second page is not mapped
        assert lib.gqa_load_kv_device(c, 0, 0, 4, odd, at, None) == _lib.GQA_ERR_RANGE
        assert lib.gqa_load_kv_device(c, 2, 0, 4, at, at, None) == _lib.GQA_ERR_STREAM_DEST
        assert lib.gqa_read_kv_device(c, 0, 0, 65, at, at, None) == _lib.GQA_ERR_RANGE
        assert lib.gqa_read_kv_device(c, 0, 90, 11, at, at, None) == _lib.GQA_ERR_RANGE
        assert lib.gqa_read_kv_device(c, 0, -1, 1, at, at, None) == _lib.GQA_ERR_RANGE
        assert lib.gqa_read_kv_device(c, 0, 0, 4, at, odd, None) == _lib.GQA_ERR_RANGE
        assert lib.gqa_read_kv_device(c, 0, 0, 0, at, at, None) == _lib.GQA_OK
        assert lib.gqa_append_kv_device(c, odd, at, ptr(t), None) == _lib.GQA_ERR_RANGE
        with pytest.raises(_lib.GqaError):
            acc.read_kv(1, 0, 1)
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        q = torch.zeros((8, 4, 64), dtype=torch.int16, device="cuda")
        seen = []
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):  # the workspace cannot be ordered with a graph's replays
            seen.append(lib.gqa_prefill_device(c, 0, ptr(q), 4, 0, 4, 0, 1, ptr(q), None, ctypes.c_void_p(stream.cuda_stream)))
            q.zero_()
        assert seen == [_lib.GQA_ERR_UNSUPPORTED]
    with AttentionAccelerator(n_q_heads=8, n_kv_heads=2, head_dim=64, max_seq_len=64) as acc:
        assert lib.gqa_kv8_scales(acc._ctx, None, None) == _lib.GQA_ERR_UNSUPPORTED
    with engine(n_q_heads=12, n_kv_heads=4, head_dim=64, max_seq_len=64) as acc:  # 3 heads a group: decode, but no prefill
        q = bf16_normal(np.random.default_rng(0), (12, 4, 64))
        with pytest.raises(_lib.GqaError) as e:
            acc.prefill_chunk(q, q_pos_base=0)
        assert e.value.code == _lib.GQA_ERR_UNSUPPORTED


def test_decode_refuses_more_keys_than_its_runs_count():
    """A paged context sized for 2^39 keys with one page of rows: the device form plans for all of them and is refused, the
    host form plans for the lengths."""
    rng = np.random.default_rng(43)
    B, hkv, d, page = 512, 8, 64, 1 << 12
    with engine(batch=B, n_q_heads=8, n_kv_heads=hkv, head_dim=d, max_seq_len=1 << 27, max_q_len=16, page_size=page,
                n_pages=1) as acc:
        acc.reserve(3, 40)
        k, v, q = rows(rng, (hkv, 40, d)), rows(rng, (hkv, 40, d)), bf16_normal(rng, (B, 8, d))
        acc.load_kv(k, v, b=3)
        lens = np.zeros(B, np.int32)
        lens[3] = 40
        t, n, o = dev(q), dev(lens), torch.zeros((B, 8, d), dtype=torch.int16, device="cuda")
        assert _lib.lib().gqa_decode_device(acc._ctx, ptr(t), ptr(n), ptr(o), None, None) == _lib.GQA_ERR_UNSUPPORTED
        got, lse = acc.decode_step(q, lens, return_lse=True)
        close(got[3], lse[3], so.decode(f64(q[3]), so.stored(f64(k)), so.stored(f64(v)), acc.scale))


def test_unmapped_pages_read_as_zeros_on_the_device():
    """Device lengths past the mapped rows: keys and values of zero, nothing written."""
    rng = np.random.default_rng(17)
    with engine(batch=2, n_q_heads=4, n_kv_heads=2, head_dim=128, max_seq_len=256, page_size=64, n_pages=3) as acc:
        acc.reserve(0, 128)
        acc.reserve(1, 64)
        k, v = rows(rng, (2, 2, 128, 128)), rows(rng, (2, 2, 128, 128))
        acc.load_kv(k[0], v[0], b=0)
        acc.load_kv(k[1, :, :64], v[1, :, :64], b=1)
        q = bf16_normal(rng, (2, 4, 128))
        before = [p.clone() for p in kv8_pools(acc)]
        o = torch.zeros((2, 4, 128), dtype=torch.int16, device="cuda")
        lse = torch.zeros((2, 4), device="cuda")
        lens = torch.tensor([200, 100], dtype=torch.int32, device="cuda")
        pos = torch.tensor([199, 70], dtype=torch.int32, device="cuda")  # unmapped rows
        new = dev(rows(rng, (2, 2, 128)))
        qd = dev(q)
        call("gqa_decode_append_device", acc._ctx, ptr(qd), ptr(new), ptr(new), ptr(pos), ptr(lens), ptr(o), ptr(lse), None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(before, kv8_pools(acc)))
        nw = words(new)
        for b, (n, have) in enumerate(((200, 128), (100, 64))):
            kk, vv = np.zeros((2, n, 128)), np.zeros((2, n, 128))
            kk[:, :have], vv[:, :have] = so.stored(f64(k[b, :, :have])), so.stored(f64(v[b, :, :have]))
            kk[:, pos[b].item()] = vv[:, pos[b].item()] = so.stored(f64(nw[b]))
            close(words(o)[b], lse[b].cpu().numpy(), so.decode(f64(q[b]), kk, vv, acc.scale))
