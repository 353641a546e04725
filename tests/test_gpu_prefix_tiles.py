"""Decode over a shared prefix where two or four waves share a tile of its keys: values that are not finite, in every wave's
share, in several pieces and rounds; and what a sequence's words depend on.  Bounds as in test_gpu_prefix.py.
"""
import numpy as np
import pytest

from tests._serving import words
from tests.test_gpu_prefix import Batch, f64, near, stored

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

NAN, INF, LOW = 0x7FC0, 0x7F80, 0xFF80
BAD = {3: (NAN,), 17: (INF,), 40: (LOW,), 41: (INF, LOW)}  # words of a dim, in turn over the bad rows


@pytest.mark.parametrize("kv_format", ["bf16", "e4m3"])
@pytest.mark.parametrize("B,hq,hkv,d,prefix,page", [(7, 8, 2, 64, 700, None),      # a wave a tile, 28 query rows a kv head
                                                    (12, 8, 2, 64, 700, 64),       # two waves, 48
                                                    (16, 32, 8, 128, 4400, None),  # two waves, full: 64; pieces of two rounds
                                                    (18, 8, 2, 128, 700, None),    # four waves, the last with eight rows: 72
                                                    (40, 32, 8, 64, 4500, 64),     # four waves, two blocks: 160; pieces of three rounds
                                                    (33, 16, 1, 128, 900, 128)])   # five blocks
def test_values_that_are_not_finite(kv_format, B, hq, hkv, d, prefix, page):
    """Infinities and NaN in V stay in their dim and reach the sequences that see them, whose other dims and all others come out as
    without them; then a NaN in K, for those who see it, in all dims."""
    rng = np.random.default_rng(B * d + prefix)
    lens = rng.integers(0, 40, B)
    batch = Batch(rng, hq, hkv, d, prefix, list(lens), kv_format, page)
    rows = np.array([5, 37, 70, 127, 128 + 33, 256 + 64, 384 + 98, prefix - 2, prefix - 1])  # every wave's share of a round
    shared = np.append(rng.choice([0, 5, 6, 36, 38, 127, 128, 200, 321, 482, 483, prefix - 1, prefix, prefix + 7], B), 0)
    shared[:4] = 0, 5, 6, prefix
    clean = batch.v[-1].copy()
    clean[:, rows[:, None], list(BAD)] = 0
    for dim, turn in BAD.items():
        batch.v[-1][:, rows, dim] = [turn[i % len(turn)] for i in range(len(rows))]
    good = np.array([x for x in range(d) if x not in BAD])
    with batch.acc:
        batch.acc.load_kv(batch.k[-1], batch.v[-1], b=B)
        batch.v[-1] = clean

        def others(o, lse, b, dims):
            p, n = min(max(int(shared[b]), 0), prefix), int(batch.lens[b])
            k, v = batch.k[b][:, :n].copy(), batch.v[b][:, :n].copy()
            if n:
                k[:, -1], v[:, -1] = batch.k_new[b], batch.v_new[b]
            k, v = (np.concatenate((stored(x[:, :p], kv_format), stored(y, kv_format)), 1) for x, y in ((batch.k[-1], k), (batch.v[-1], v)))
            near(o[b][:, dims], lse[b], f64(batch.q[b]), k, v[..., dims], batch.acc.scale)

        for whole in (False, True):  # some of it each; all of it for everyone
            if whole:
                shared[:B] = prefix
            o, lse = batch.run(shared)
            torch.cuda.synchronize()
            o, lse = words(o), lse.cpu().numpy()
            got = f64(o)
            for b in range(B):
                seen = rows[rows < shared[b]]
                others(o, lse, b, good if len(seen) else slice(None))
                if not len(seen):
                    continue
                if kv_format == "e4m3":  # (rows of the 8-bit cache hold NaN for all)
                    assert np.isnan(got[b][:, list(BAD)]).all()
                    continue
                assert np.isnan(got[b, :, 3]).all() and np.all(got[b, :, 17] == np.inf) and np.all(got[b, :, 40] == -np.inf)
                assert np.all(got[b, :, 41] == np.inf) if len(seen) == 1 else np.isnan(got[b, :, 41]).all()
        # K: those who see row 161 are NaN, the others as they are
        batch.k[-1][:, 161, 9] = NAN
        batch.acc.load_kv(batch.k[-1], batch.v[-1], b=B)
        shared[:B] = rng.choice([0, 100, 161, 162, prefix], B)
        shared[:3] = 161, 162, prefix
        o, lse = batch.run(shared)
        torch.cuda.synchronize()
        o, lse = words(o), lse.cpu().numpy()
        for b in range(B):
            if shared[b] > 161:
                assert np.isnan(f64(o[b])).all() and np.isnan(lse[b]).all()
            else:
                others(o, lse, b, slice(None))


@pytest.mark.parametrize("kv_format", ["bf16", "e4m3"])
@pytest.mark.parametrize("B", [6, 14, 40])
def test_what_a_sequence_depends_on(kv_format, B):
    """The words of a sequence without own rows are the same whatever the others have; own rows are cut by the batch's steps, so
    that those of one with many are within the bounds whatever the others have."""
    rng = np.random.default_rng(B)
    lens = rng.integers(1, 80, B)
    lens[:3] = 0, 700, 65
    batch = Batch(rng, 8, 2, 64, 900, list(lens), kv_format)
    first = []
    with batch.acc:
        for load in range(3):
            now, shared = batch.lens.copy(), np.append(np.full(B, 900), 0)
            if load == 1:
                now[3:], shared[3:] = 0, 0
            if load == 2:
                now[2:B], shared[2:B] = batch.lens[2:B] // 2, rng.integers(0, 901, B - 2)
            o, lse = batch.run(shared, append=False, lens=now)
            torch.cuda.synchronize()
            batch.check(o, lse, shared, append=False, lens=now)
            first.append((o[0].clone(), lse[0].clone()))
        assert all(torch.equal(a, b) for other in first[1:] for a, b in zip(first[0], other))
