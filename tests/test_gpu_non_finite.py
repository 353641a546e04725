"""NaN and infinities in what attention reads: they come out where the definition has them, and nowhere else.

A score that is NaN makes its row's sum NaN, so the row's output and log-sum-exp are NaN -- not the zeros and -inf of a row
without keys.  A value that is NaN makes its own dimension NaN.  Every other word is that of the same call on clean rows:
the plan does not depend on values.
"""
import numpy as np
import pytest

from lara_amd import _lib
from lara_amd.attn_driver import AttentionAccelerator
from oracle import gqa_oracle as orc
from tests._gen import bf16_normal
from tests._serving import call

pytestmark = pytest.mark.gpu

NAN, INF = 0x7FC0, 0x7F80

# name: (H_q, H_kv, D, lengths, decode chunk, merge)
DECODE_PLANS = {
    "whole": (8, 2, 64, [0, 1, 300, 300], 0, _lib.GQA_DECODE_MERGE_AUTO),
    "merged in the launch": (32, 2, 128, [0, 1, 700, 1500], 256, _lib.GQA_DECODE_MERGE_FUSED),
    "merge launch": (8, 2, 64, [0, 1, 700, 1500], 256, _lib.GQA_DECODE_MERGE_LAUNCH),
    "many sequences": (16, 4, 64, [0, 1, 2112, 700] + [2112, 300] * 9, 0, _lib.GQA_DECODE_MERGE_AUTO),
}


def decode_non_finite(kv_format, plan):
    hq, hkv, d, lens, chunk, merge = DECODE_PLANS[plan]
    rng = np.random.default_rng(hq + d)
    B, L, group = len(lens), max(lens), hq // hkv
    q, k, v = bf16_normal(rng, (B, hq, d)), bf16_normal(rng, (B, hkv, L, d)), bf16_normal(rng, (B, hkv, L, d))
    values = ((1, 1, 0, 0), (2, 0, 200, d - 1), (3, 1, lens[3] - 1, 17))
    for at in values:
        v[at] = 0  # (not the largest of their rows, whose E4M3 scale stays the same without them)
    with AttentionAccelerator(batch=B, n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=L, kv_format=kv_format) as acc:
        call("gqa_set_option", acc._ctx, _lib.GQA_OPT_DECODE_CHUNK, chunk)
        call("gqa_set_option", acc._ctx, _lib.GQA_OPT_DECODE_MERGE, merge)

        def step(q, k, v):
            for b, n in enumerate(lens):
                if n:
                    acc.load_kv(k[b, :, :n], v[b, :, :n], b=b)
            o, lse = acc.decode_step(q, lens, return_lse=True)
            assert not o[0].any() and np.all(lse[0] == -np.inf)  # the idle slot, whatever the others hold
            return orc.bf16_u16_to_fp32(o), lse

        clean, clean_lse = step(q, k, v)

        def check(o, lse, o_nan, lse_nan):
            assert np.array_equal(np.isnan(o), o_nan) and np.array_equal(np.isnan(lse), lse_nan)
            assert np.array_equal(o[~o_nan], clean[~o_nan]) and np.array_equal(lse[~lse_nan], clean_lse[~lse_nan])

        # one query head of NaN in sequences of one key, of some and of many
        bad = q.copy()
        want = np.zeros((B, hq), bool)
        for b, h in ((1, 0), (2, hq - 1), (3, group)):
            bad[b, h, 5] = NAN
            want[b, h] = True
        check(*step(bad, k, v), np.repeat(want[..., None], d, -1), want)
        # keys: the only one, one among many, the last one, 256 that make up a whole piece; of one kv head each
        want = np.zeros((B, hq), bool)
        bad = k.copy()
        for b, h, keys in ((1, 0, slice(0, 1)), (2, 0, slice(37, 38)), (2, 1, slice(lens[2] - 1, lens[2])),
                           (3, 1, slice(256, 512) if lens[3] > 512 else slice(0, lens[3]))):
            bad[b, h, keys, 7] = NAN if b < 3 or kv_format == "bf16" else INF  # (an E4M3 row keeps an infinity as NaN)
            want[b, h * group:(h + 1) * group] = True
        check(*step(q, bad, v), np.repeat(want[..., None], d, -1), want)
        # values: one dimension of one row
        bad = v.copy()
        want = np.zeros((B, hq, d), bool)
        for b, h, key, dim in values:
            bad[b, h, key, dim] = NAN
            want[b, h * group:(h + 1) * group, dim] = True
        check(*step(q, k, bad), want, np.zeros((B, hq), bool))


@pytest.mark.parametrize("plan", DECODE_PLANS)
def test_e4m3_decode(plan):
    decode_non_finite("e4m3", plan)


@pytest.mark.parametrize("plan", DECODE_PLANS)
def test_bf16_decode(plan):
    decode_non_finite("bf16", plan)


PREFILL_KERNELS = {"rows": _lib.GQA_PREFILL_KERNEL_ROWS, "shared": _lib.GQA_PREFILL_KERNEL_SHARED,
                   "paired": _lib.GQA_PREFILL_KERNEL_PAIRED, "segments": _lib.GQA_PREFILL_KERNEL_SHARED}


@pytest.mark.parametrize("kv_format", ["bf16", "e4m3"])
@pytest.mark.parametrize("kernel", PREFILL_KERNELS)
def test_prefill(kernel, kv_format):
    """Causal blocks: some query rows of NaN (one of them without keys), then a key of NaN, which the rows before it do not
    see."""
    rng = np.random.default_rng(29)
    hq, hkv, d, n, history, kv_pos = 8, 2, 64, 70, 90, 100
    kv_len = history + n
    q, k, v = (bf16_normal(rng, (h, m, d)) for h, m in ((hq, n), (hkv, kv_len), (hkv, kv_len)))
    with AttentionAccelerator(n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=kv_len, max_q_len=n,
                              kv_format=kv_format) as acc:
        call("gqa_set_option", acc._ctx, _lib.GQA_OPT_PREFILL_KERNEL, PREFILL_KERNELS[kernel])
        if kernel == "segments":
            call("gqa_set_option", acc._ctx, _lib.GQA_OPT_PREFILL_WGS, 64)

        def block(q, k, q_pos_base):
            acc.load_kv(k, v)
            o, lse = acc.prefill_chunk(q, q_pos_base=q_pos_base, kv_len=kv_len, kv_pos_base=kv_pos, causal=True, return_lse=True)
            return orc.bf16_u16_to_fp32(o), lse

        def check(got, clean, want):
            want_o = np.repeat(want[..., None], d, -1)
            assert np.array_equal(np.isnan(got[0]), want_o) and np.array_equal(np.isnan(got[1]), want)
            assert np.array_equal(got[0][~want_o], clean[0][~want_o]) and np.array_equal(got[1][~want], clean[1][~want])

        bad = q.copy()
        want = np.zeros((hq, n), bool)
        bad[0, 0, 3] = bad[2, 31, 0] = bad[5, 64, 63] = bad[7, n - 1, 9] = NAN
        want[2, 31] = want[5, 64] = want[7, n - 1] = True
        q_pos = kv_pos - 1  # row 0 is before the first key: no scores, so no NaN either
        clean = block(q, k, q_pos)
        assert not clean[0][:, 0].any() and np.all(clean[1][:, 0] == -np.inf)
        check(block(bad, k, q_pos), clean, want)
        q_pos = kv_pos + history  # the rows follow the keys
        want[0, 0] = True
        check(block(bad, k, q_pos), block(q, k, q_pos), want)
        bad = k.copy()
        bad[1, history + 40, 11] = NAN
        want = np.zeros((hq, n), bool)
        want[hq // hkv:, 40:] = True
        check(block(q, bad, q_pos), block(q, k, q_pos), want)
