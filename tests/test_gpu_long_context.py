"""The long-context operators as a program uses them together: prompts through the rotary form into the cache, their attention
weight, decode steps over a shared prefix whose log-sum-exp feeds the accumulated weight, eviction, and decode on.

Each result is checked against float64 of what the step before left on the GPU, with the bounds of the operators' own tests.
Captured steps, other streams and two engines at once give the same words as the same steps one by one.
"""
import numpy as np
import pytest

from lara_amd import _lib, rope
from lara_amd.attn_driver import AttentionAccelerator
from oracle import gqa_oracle as orc
from oracle import long_context_oracle as lo
from tests._gen import bf16_normal
from tests._serving import dev, words
from tests.test_gpu_budget import bound
from tests.test_gpu_prefix import near
from tests.test_gpu_rotary import near_bf16

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

FORM = dict(rotary_dim=64, scaling="ramp", factor=4.0, original_len=256, low=1.0, high=32.0)


@pytest.fixture(autouse=True)
def a_stream():
    """What torch enqueues and what the engines are given: one stream that is not the default one."""
    with torch.cuda.stream(torch.cuda.Stream()):
        yield


def current():
    return torch.cuda.current_stream().cuda_stream


def f64(w):
    return orc.bf16_u16_to_fp32(w).astype(np.float64)


class Serving:
    """Sequences behind one system prompt, each with a budget of rows; every call on torch's current stream."""

    HQ, HKV, D, KEEP, SINKS, RECENT = 16, 4, 128, 40, 2, 8

    def __init__(self, seed, kv_format="bf16", page=None, prefix=150, prompts=(0, 1, 33, 100), L=256):
        rng = np.random.default_rng(seed)
        self.L = L
        self.rng, self.prefix, self.B = rng, prefix, len(prompts) + 1
        self.acc = AttentionAccelerator(batch=self.B, n_q_heads=self.HQ, n_kv_heads=self.HKV, head_dim=self.D, max_seq_len=self.L,
                                        max_q_len=256, kv_format=kv_format, page_size=page)
        for b in range(self.B if page else 0):
            self.acc.reserve(b, self.L)
        self.form = rope.form("halves", **FORM)
        self.width = (self.HQ + 2 * self.HKV) * self.D
        self.lens = np.array([*prompts, 0], np.int32)
        self.positions = (prefix + self.lens).astype(np.int32)
        self.positions[-1] = -1  # (the prefix's own sequence takes no steps)
        z = lambda *shape, dtype: torch.zeros(shape, dtype=dtype, device="cuda")  # noqa: E731
        self.x, self.q = z(self.B, self.width, dtype=torch.int16), z(self.B, self.HQ, self.D, dtype=torch.int16)
        self.o, self.lse = torch.zeros_like(self.q), z(self.B, self.HQ, dtype=torch.float32)
        self.mass = z(self.B, self.HKV, self.L, dtype=torch.float32)
        self.kept = z(self.B, self.HKV, self.KEEP, dtype=torch.int32)
        self.dlens, self.dpos = dev(self.lens), dev(self.positions)
        torch.cuda.synchronize()

    def prompt(self, b, n, first):
        """n prompt rows of sequence b at positions first..: (q [H_q, n, D] words, the tensors kept alive)."""
        x = dev(bf16_normal(self.rng, (n, self.width)))
        q = torch.zeros((self.HQ, n, self.D), dtype=torch.int16, device="cuda")
        self.acc.qk_norm_rotary_device(x.data_ptr(), self.width, n, None, None, q.data_ptr(), self.form, b=b, q_pos_base=first,
                                       kv_pos_base=first, stream=current())
        torch.cuda.synchronize()
        return q

    def next_token(self):
        self.x.copy_(dev(bf16_normal(self.rng, (self.B, self.width))))

    def step(self):
        """Enqueues a step: the token's heads into row `lens` of the cache, attention over it too, its weight."""
        s = current()
        self.acc.qk_norm_rotary_step_device(self.x.data_ptr(), self.width, None, None, self.dpos.data_ptr(), self.q.data_ptr(), self.form,
                                            rows_ptr=self.dlens.data_ptr(), stream=s)
        self.dlens[:-1] += 1
        self.dpos[:-1] += 1
        self.acc.decode_prefix_device(self.q.data_ptr(), self.B - 1, self.prefix, self.dlens.data_ptr(), self.o.data_ptr(),
                                      lse_ptr=self.lse.data_ptr(), stream=s)
        self.acc.attention_mass_step_device(self.q.data_ptr(), self.dlens.data_ptr(), self.lse.data_ptr(), self.mass.data_ptr(), decay=0.875,
                                            stream=s)

    def evict(self):
        self.acc.evict_device(self.mass.data_ptr(), self.dlens.data_ptr(), self.KEEP, self.kept.data_ptr(), sinks=self.SINKS,
                              recent=self.RECENT, stream=current())

    def results(self):
        torch.cuda.synchronize()
        rows = [self.acc.read_kv(b, 0, self.L) for b in range(self.B)]
        return [t.cpu().numpy().copy() for t in (self.q, self.o, self.lse, self.mass, self.kept, self.dlens)] + [t for r in rows for t in r]


def same(a, b):
    return len(a) == len(b) and all(np.array_equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("kv_format", ["bf16", "e4m3"])
@pytest.mark.parametrize("page,L", [(None, 256), (64, 256), (64, 2176)])
def test_steps_of_a_program(kv_format, page, L):
    s = Serving(1, kv_format, page, L=L)
    with s.acc:
        s.prompt(s.B - 1, s.prefix, 0)
        pk, pv = (f64(t) for t in s.acc.read_kv(s.B - 1, 0, s.prefix))
        for b, n in enumerate(s.lens[:-1]):
            if n == 0:
                continue
            q = s.prompt(b, int(n), s.prefix)
            _, lse = s.acc.prefill_chunk(words(q), b=b, q_pos_base=s.prefix, kv_len=int(n), kv_pos_base=s.prefix, return_lse=True)
            lsed = dev(np.asarray(lse, np.float32))
            s.acc.attention_mass_device(q.data_ptr(), int(n), int(n), lsed.data_ptr(), s.mass.data_ptr(), b=b, q_pos_base=s.prefix,
                                        kv_pos_base=s.prefix, stream=current())
            torch.cuda.synchronize()
            qq, k = f64(words(q)), f64(s.acc.read_kv(b, 0, int(n))[0])
            l64 = np.asarray(lse, np.float64).reshape(s.HQ, n)
            want = lo.mass(qq, k, l64, s.acc.scale, np.tril(np.ones((n, n), bool)))
            got = s.mass[b].cpu().numpy()
            assert np.all(np.abs(got[:, :n] - want) <= bound(want, qq, k, l64, s.acc.scale, 0.0, 1.0)) and not got[:, n:].any()
        lens = s.lens.copy()
        for i in range(30):
            before = s.mass.cpu().numpy().astype(np.float64)
            s.next_token()
            s.step()
            torch.cuda.synchronize()
            lens[:-1] += 1
            assert np.array_equal(s.dlens.cpu().numpy(), lens)
            o, lse, mass, qw = words(s.o), s.lse.cpu().numpy(), s.mass.cpu().numpy(), f64(words(s.q))
            for b in range(s.B - 1):
                n = int(lens[b])
                k, v = (f64(t) for t in s.acc.read_kv(b, 0, n))
                near(o[b], lse[b], qw[b], np.concatenate((pk, k), 1), np.concatenate((pv, v), 1), s.acc.scale)
                l64 = lse[b].astype(np.float64)[:, None]
                new = lo.mass(qw[b][:, None], k, l64, s.acc.scale)
                tol = bound(new, qw[b][:, None], k, l64, s.acc.scale, before[b, :, :n], 0.875)
                assert np.all(np.abs(mass[b, :, :n] - (0.875 * before[b, :, :n] + new)) <= tol)
            assert not o[-1].any() and np.all(lse[-1] == -np.inf)
            if i % 7 == 6:
                rows = [s.acc.read_kv(b, 0, s.L) for b in range(s.B)]
                s.evict()
                torch.cuda.synchronize()
                for b in range(s.B - 1):
                    now, n = s.acc.read_kv(b, 0, s.L), int(lens[b])
                    for h in range(s.HKV):
                        at = lo.evict(mass[b, h, :n].tolist(), n, s.KEEP, s.SINKS, s.RECENT)
                        assert np.array_equal(s.kept[b, h, :len(at)].cpu().numpy(), at)
                        for x, y in zip(rows[b], now):
                            assert np.array_equal(y[h, :len(at)], x[h][at]) and np.array_equal(y[h, n:], x[h, n:])
                for x, y in zip(rows[-1], s.acc.read_kv(s.B - 1, 0, s.L)):
                    assert np.array_equal(x, y)
                lens = np.minimum(lens, s.KEEP)


def fill(s):
    s.prompt(s.B - 1, s.prefix, 0)
    for b, n in enumerate(s.lens[:-1]):
        if n:
            s.prompt(b, int(n), s.prefix)


def twins(*args, **kw):
    a, b = Serving(*args, **kw), Serving(*args, **kw)
    for s in (a, b):
        fill(s)
    return a, b


@pytest.mark.parametrize("L", [256, 2176])
@pytest.mark.parametrize("kv_format", ["bf16", "e4m3"])
def test_captured_steps_replay(kv_format, L):
    """Two steps and an eviction in one graph, on a stream that is not the engine's; other work between the replays."""
    a, b = twins(2, kv_format, 64, L=L)
    with a.acc, b.acc:
        for s in (a, b):  # (the first call allocates)
            s.next_token()
            s.step()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
            b.step()
            b.step()
            b.evict()
        junk = torch.randn((512, 512), device="cuda")
        for _ in range(4):
            for s in (a, b):
                s.next_token()
            a.step()
            a.step()
            a.evict()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert same(a.results(), b.results())
            junk = (junk @ junk).clamp(-1, 1)  # (eager work between the replays)
            for s in (a, b):
                s.next_token()
                s.step()
            assert same(a.results(), b.results())


def test_the_first_step_over_a_prefix_is_not_captured():
    s = Serving(3, L=4096)  # (short contexts need nothing allocated)
    with s.acc:
        fill(s)
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
            with pytest.raises(_lib.GqaError) as e:
                s.acc.decode_prefix_device(s.q.data_ptr(), s.B - 1, s.prefix, s.dlens.data_ptr(), s.o.data_ptr(), stream=current())
            s.mass += 1.0
        assert e.value.code == _lib.GQA_ERR_UNSUPPORTED
        torch.cuda.synchronize()
        s.next_token()
        s.step()
        torch.cuda.synchronize()
        assert np.isfinite(s.lse.cpu().numpy()[:-1]).all()


def test_two_engines_at_once():
    """Steps of two engines on two streams, nothing waiting between them, and the same steps one engine after the other."""
    alone = []
    for seed in (4, 5):
        s = Serving(seed, L=2176)
        with s.acc:
            fill(s)
            for _ in range(12):
                s.next_token()
                s.step()
                torch.cuda.synchronize()
                s.evict()
                torch.cuda.synchronize()
            alone.append(s.results())
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    engines = [Serving(seed, L=2176) for seed in (4, 5)]
    with engines[0].acc, engines[1].acc:
        tokens = []
        for s in engines:
            fill(s)
            tokens.append([dev(bf16_normal(s.rng, (s.B, s.width))) for _ in range(12)])
        torch.cuda.synchronize()
        for i in range(12):
            for s, t, x in zip(engines, streams, tokens):
                with torch.cuda.stream(t):
                    s.x.copy_(x[i])
                    s.step()
                    s.evict()
        for s, want in zip(engines, alone):
            assert same(s.results(), want)


@pytest.mark.parametrize("page", [None, 64])
def test_offsets_past_32_bits(page):
    """A cache of 4.9 GB for K and as much for V: the last sequence's rows lie past 2^32 bytes and 2^31 elements."""
    rng = np.random.default_rng(6)
    hq, hkv, d, L, n = 16, 8, 128, 1_200_000, 90
    far = L - 200
    with AttentionAccelerator(batch=2, n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=L, max_q_len=64, page_size=page) as acc:
        for b in range(2 if page else 0):
            acc.reserve(b, L)
        k, v = (bf16_normal(rng, (2, hkv, n, d)) for _ in range(2))
        for b in range(2):
            acc.load_kv(k[b], v[b], b=b)
        q = bf16_normal(rng, (2, hq, d))
        qd, o, lse = dev(q), torch.zeros((2, hq, d), dtype=torch.int16, device="cuda"), torch.zeros((2, hq), device="cuda")
        torch.cuda.synchronize()
        for prefix_b in (0, 1):
            own = 1 - prefix_b
            lens = np.array([0, 0], np.int32)
            lens[own] = n
            ln = dev(lens)
            acc.decode_prefix_device(qd.data_ptr(), prefix_b, n, ln.data_ptr(), o.data_ptr(), lse_ptr=lse.data_ptr(),
                                     stream=current())
            torch.cuda.synchronize()
            both = [np.concatenate((f64(t[prefix_b]), f64(t[own])), 1) for t in (k, v)]
            near(words(o)[own], lse.cpu().numpy()[own], f64(q[own]), *both, acc.scale)
        # rows in the far end: the rotary step writes there, attention weight reaches there, eviction brings them back
        x = bf16_normal(rng, (2, (hq + 2 * hkv) * d))
        xd, pos, row = dev(x), dev(np.array([L - 1, far], np.int32)), dev(np.array([-1, far], np.int32))
        acc.qk_norm_rotary_step_device(xd.data_ptr(), x.shape[1], None, None, pos.data_ptr(), qd.data_ptr(), rope.form("halves"),
                                       rows_ptr=row.data_ptr(), stream=current())
        torch.cuda.synchronize()
        kr, vr = acc.read_kv(1, far, 1)
        freq, m = lo.frequencies(d, 10000.0)
        want, mag = lo.norm_rotary(f64(x[1, hq * d:(hq + hkv) * d]).reshape(hkv, 1, d), None, 0.0, [far], freq, m, True)
        near_bf16(kr, want, mag)
        assert np.array_equal(f64(vr[:, 0]), f64(x[1, (hq + hkv) * d:]).reshape(hkv, d))
        lens = dev(np.array([0, far + 1], np.int32))
        mass = torch.zeros((2, hkv, L), device="cuda")
        lse.fill_(0.0)
        acc.attention_mass_step_device(qd.data_ptr(), lens.data_ptr(), lse.data_ptr(), mass.data_ptr(), decay=0.0,
                                       stream=current())
        torch.cuda.synchronize()
        qq, l64 = f64(words(qd)[1])[:, None], np.zeros((hq, 1))
        for at, kk in ((slice(0, n), f64(k[1])), (slice(far, far + 1), f64(kr))):
            new = lo.mass(qq, kk, l64, acc.scale)
            assert np.all(np.abs(mass[1, :, at].cpu().numpy() - new) <= bound(new, qq, kk, l64, acc.scale, 0.0, 1.0))
        assert not mass[1, :, far + 1:].any()
        heavy = np.sort(rng.choice(far, 50, replace=False))
        heavy[-1] = far
        rows = np.concatenate([acc.read_kv(1, int(t), 1)[0] for t in heavy], 1)
        mass.zero_()
        mass[1, :, torch.from_numpy(heavy).cuda()] = 1.0
        kept = torch.zeros((2, hkv, 50), dtype=torch.int32, device="cuda")
        acc.evict_device(mass.data_ptr(), lens.data_ptr(), 50, kept.data_ptr(), stream=current())
        torch.cuda.synchronize()
        assert np.array_equal(kept[1].cpu().numpy(), np.broadcast_to(heavy, (hkv, 50)))
        assert np.array_equal(acc.read_kv(1, 0, 50)[0], rows)
        assert lens.cpu().tolist() == [0, 50] and mass[1, :, :50].eq(1).all() and not mass[1, :, 50:].any()
