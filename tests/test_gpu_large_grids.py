"""Launches of more than 2^20 work-groups, whose grids have a second dimension: each against the same work in smaller calls,
or in float64."""
import ctypes

import numpy as np
import pytest

from lara_amd import _lib
from lara_amd.attn_driver import AttentionAccelerator
from oracle import gqa_oracle as orc
from oracle import serving_oracle as so
from tests._gen import bf16_normal
from tests._serving import call, dev, ptr

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

PART = 1 << 20


def normal(shape, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, device="cuda", generator=gen, dtype=torch.bfloat16)


def test_e4m3_rows_written_and_read_back():
    hkv, d, n = 2, 128, (1 << 23) + 4999
    assert hkv * n * (d // 8) > 256 << 20
    k, v = normal((hkv, n, d), 1), normal((hkv, n, d), 2)
    with AttentionAccelerator(batch=2, n_q_heads=hkv, n_kv_heads=hkv, head_dim=d, max_seq_len=n, max_q_len=1, kv_format="e4m3") as acc:
        call("gqa_load_kv_device", acc._ctx, 0, 0, n, ptr(k), ptr(v), None)
        for at in range(0, n, PART):
            m = min(PART, n - at)
            ks, vs = k[:, at:at + m].contiguous(), v[:, at:at + m].contiguous()
            call("gqa_load_kv_device", acc._ctx, 1, at, m, ptr(ks), ptr(vs), None)
            torch.cuda.synchronize()
        k.fill_(float("nan")), v.fill_(float("nan"))
        torch.cuda.synchronize()
        acc.read_kv_device(0, 0, n, k.data_ptr(), v.data_ptr())
        for at in range(0, n, PART):
            m = min(PART, n - at)
            parts = [torch.empty((hkv, m, d), dtype=torch.bfloat16, device="cuda") for _ in range(4)]
            torch.cuda.synchronize()
            for b in range(2):
                acc.read_kv_device(b, at, m, parts[2 * b].data_ptr(), parts[2 * b + 1].data_ptr())
            torch.cuda.synchronize()
            assert torch.equal(parts[0], parts[2]) and torch.equal(parts[1], parts[3]), at  # written by one call and by many
            assert torch.equal(k[:, at:at + m], parts[2]) and torch.equal(v[:, at:at + m], parts[3]), at  # and read by one


@pytest.mark.parametrize("d,kv_format", [(64, "e4m3"), (128, "bf16")])
def test_heads_of_a_long_prompt(d, kv_format):
    n = (1 << 20) * (128 // d) + 3
    x, wq, wk = normal((n, 3 * d), 3), normal((d,), 4), normal((d,), 5)
    q = torch.full((n, d), float("nan"), dtype=torch.bfloat16, device="cuda")
    with AttentionAccelerator(batch=2, n_q_heads=1, n_kv_heads=1, head_dim=d, max_seq_len=n, max_q_len=1, kv_format=kv_format) as acc:
        acc.qk_norm_rope_device(x.data_ptr(), 3 * d, n, wq.data_ptr(), wk.data_ptr(), q.data_ptr(), b=0)
        step = PART // 2 - 7
        for at in range(0, n, step):
            m = min(step, n - at)
            part = torch.empty((m, d), dtype=torch.bfloat16, device="cuda")
            torch.cuda.synchronize()
            acc.qk_norm_rope_device(x[at:].data_ptr(), 3 * d, m, wq.data_ptr(), wk.data_ptr(), part.data_ptr(), b=1, q_pos_base=at,
                                    kv_pos_base=at, kv_row0=at)
            torch.cuda.synchronize()
            assert torch.equal(q[at:at + m], part), at
        rows = [torch.empty((1, n, d), dtype=torch.bfloat16, device="cuda") for _ in range(4)]
        torch.cuda.synchronize()
        for b in range(2):
            acc.read_kv_device(b, 0, n, rows[2 * b].data_ptr(), rows[2 * b + 1].data_ptr())
        torch.cuda.synchronize()
        assert torch.equal(rows[0], rows[2]) and torch.equal(rows[1], rows[3])


def test_e4m3_decode_merges_many_sequences():
    """Runs cut inside sequences all over the batch; bounds as in the E4M3 cache's own tests."""
    rng = np.random.default_rng(6)
    B, hq, hkv, d, L, unique = 1 << 15, 64, 4, 64, 600, 64
    k, v, q = bf16_normal(rng, (hkv, L, d)), bf16_normal(rng, (hkv, L, d)), bf16_normal(rng, (unique, hq, d))
    f64 = lambda w: orc.bf16_u16_to_fp32(w).astype(np.float64)
    want, want_lse, bound = [], [], []
    with AttentionAccelerator(batch=B, n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=L, max_q_len=1, kv_format="e4m3") as acc:
        for s in range(unique):
            o, lse, avg = so.decode(f64(q[s]), so.stored(f64(k)), so.stored(f64(v)), acc.scale)
            want.append(o), want_lse.append(lse), bound.append(2.0**-8 * np.abs(o) + (2.0**-8 + 2.0**-13) * avg)
        want, want_lse, bound = (torch.tensor(np.array(t), device="cuda") for t in (want, want_lse, bound))
        kd, vd, qd = dev(k), dev(v), dev(q).repeat(B // unique, 1, 1)
        for b in range(B):
            call("gqa_load_kv_device", acc._ctx, b, 0, L, ptr(kd), ptr(vd), None)
        lens = torch.full((B,), L, dtype=torch.int32, device="cuda")
        o = torch.full((B, hq, d), float("nan"), dtype=torch.bfloat16, device="cuda")
        lse = torch.full((B, hq), float("nan"), device="cuda")
        torch.cuda.synchronize()
        call("gqa_set_option", acc._ctx, _lib.GQA_OPT_PROFILE, 1)
        call("gqa_decode_device", acc._ctx, ptr(qd), ptr(lens), ptr(o), ptr(lse), None)
        torch.cuda.synchronize()
        counts = (ctypes.c_int32 * _lib.GQA_TIMER_COUNT)()
        call("gqa_kernel_launch_counts", acc._ctx, counts, _lib.GQA_TIMER_COUNT)
        assert counts[_lib.GQA_TIMER_COMBINE] == 1  # cut into runs: B * hq work-groups join them
    for at in range(0, B, 2048):
        got, got_lse = o[at:at + 2048].view(-1, unique, hq, d).double(), lse[at:at + 2048].view(-1, unique, hq).double()
        assert torch.all((got - want).abs() <= bound), at
        assert torch.all((got_lse - want_lse).abs() <= 2.0**-13 + 2.0**-22 * want_lse.abs()), at
