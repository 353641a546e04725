"""The sequence that holds a shared prefix, in a program's steps and evictions: its prefix rows stay what they are, word for word,
and every other sequence's attention over them stays right (float64, with the bounds of the operators' own tests).

A slot that only holds the prefix has position -1 and length 0; one that goes on itself writes its rows behind the prefix and is
given to evictions with a length of 0.
"""
import numpy as np
import pytest

from oracle import long_context_oracle as lo
from tests._serving import words
from tests.test_gpu_long_context import Serving, a_stream, current, f64  # noqa: F401  (a_stream: every test's)
from tests.test_gpu_prefix import near

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("goes_on", [False, True])
@pytest.mark.parametrize("kv_format,page,L", [("bf16", None, 256), ("bf16", 64, 2176), ("e4m3", 64, 256), ("e4m3", None, 2176)])
def test_the_prefix_stays_through_steps_and_evictions(kv_format, page, L, goes_on):
    s = Serving(21, kv_format, page, prefix=60, prompts=(0, 33, 45), L=L)  # (a prefix of more rows than evictions keep)
    slot = s.B - 1
    with s.acc:
        s.prompt(slot, s.prefix, 0)
        held = s.acc.read_kv(slot, 0, s.prefix)
        pk, pv = (f64(t) for t in held)
        for b, n in enumerate(s.lens[:-1]):
            if n:
                s.prompt(b, int(n), s.prefix)
        if goes_on:
            s.dlens[slot], s.dpos[slot] = s.prefix, s.prefix
        lens = s.dlens.cpu().numpy()
        for i in range(12):
            s.next_token()
            st = current()
            s.acc.qk_norm_rotary_step_device(s.x.data_ptr(), s.width, None, None, s.dpos.data_ptr(), s.q.data_ptr(), s.form,
                                             rows_ptr=s.dlens.data_ptr(), stream=st)
            stepping = (s.dpos >= 0).int()
            s.dlens += stepping
            s.dpos += stepping
            s.acc.decode_prefix_device(s.q.data_ptr(), slot, s.prefix, s.dlens.data_ptr(), s.o.data_ptr(), lse_ptr=s.lse.data_ptr(), stream=st)
            s.acc.attention_mass_step_device(s.q.data_ptr(), s.dlens.data_ptr(), s.lse.data_ptr(), s.mass.data_ptr(), stream=st)
            torch.cuda.synchronize()
            lens[:slot] += 1
            lens[slot] += goes_on
            assert np.array_equal(s.dlens.cpu().numpy(), lens)
            assert all(np.array_equal(a, b) for a, b in zip(held, s.acc.read_kv(slot, 0, s.prefix)))
            o, lse, qw = words(s.o), s.lse.cpu().numpy(), f64(words(s.q))
            for b in range(s.B):
                k, v = (f64(t) for t in s.acc.read_kv(b, 0, int(lens[b]))) if lens[b] else (np.zeros((s.HKV, 0, s.D)),) * 2
                if b != slot:
                    k, v = np.concatenate((pk, k), 1), np.concatenate((pv, v), 1)
                near(o[b], lse[b], qw[b], k, v, s.acc.scale)
            if i % 4 != 3:
                continue
            mass, rows = s.mass.cpu().numpy(), [s.acc.read_kv(b, 0, s.L) for b in range(s.B)]
            budget = s.dlens.clone()
            budget[slot] = 0
            s.acc.evict_device(s.mass.data_ptr(), budget.data_ptr(), s.KEEP, s.kept.data_ptr(), sinks=s.SINKS, recent=s.RECENT, stream=st)
            budget[slot] = s.dlens[slot]
            s.dlens.copy_(budget)
            torch.cuda.synchronize()
            for b in range(slot):
                now, n = s.acc.read_kv(b, 0, s.L), int(lens[b])
                for h in range(s.HKV):
                    at = lo.evict(mass[b, h, :n].tolist(), n, s.KEEP, s.SINKS, s.RECENT)
                    assert np.array_equal(s.kept[b, h, :len(at)].cpu().numpy(), at)
                    assert all(np.array_equal(y[h, :len(at)], x[h][at]) for x, y in zip(rows[b], now))
            assert all(np.array_equal(x, y) for x, y in zip(rows[slot], s.acc.read_kv(slot, 0, s.L)))
            assert s.kept[slot].eq(-1).all() and np.array_equal(s.mass[slot].cpu().numpy(), mass[slot])
            lens[:slot] = np.minimum(lens[:slot], s.KEEP)
            assert np.array_equal(s.dlens.cpu().numpy(), lens)
