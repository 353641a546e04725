"""A step over long contexts: positions turned the model's way, a prefix that the batch shares, a budget of cache rows.

Kinds of a case:

* ``rotary``: per-head RMSNorm of queries and keys with the position rotation (pairs side by side or in the two halves, part
  of a head, frequencies scaled for long contexts), into Q and the cache: a prompt's rows, or one row of each sequence.
* ``prefix``: one generated token per sequence -- its K/V row appended, attention over the rows of a prefix that the batch
  shares and over the sequence's own rows.
* ``mass``: the attention weight that every cache row gets, summed over the query heads of its kv head (and the query rows
  of a prompt), added to what it has.
* ``evict``: the cache cut down to a budget of rows per sequence: the first ones, the last ones and the heaviest between.

Sizes are those of this repository's workloads and tests and of the ranges between and around them.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

own = False

BF16, E4M3, E8M0 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu
TOP = 1.875 * 2.0**127  # the largest magnitude that an E4M3 cache row holds

LAYOUTS = {"pairs": 0, "halves": 1}
SCALINGS = {"plain": 0, "linear": 1, "bands": 2, "ramp": 3}


def listed():
    return [
        # The step of a busy server's layer between projection and attention, into the E4M3 cache; positions past the
        # length that the model was trained on.
        _rotary("rotary-step-b64-e4m3", True, 64, 32, 8, 128, 100000, kv8=True, scaling="bands", base=5e5),
        # A prompt's block far into a long context.
        _rotary("rotary-2048", False, 2048, 32, 8, 128, 60000, kv8=False, scaling="ramp", base=1e4),
        # A short prompt of a small model that turns half of every head.
        _rotary("rotary-200-part-d64", False, 200, 8, 2, 64, 0, kv8=False, layout="pairs", part=32, scaling="linear", base=1e4),
        # A few short conversations of a small model behind one system prompt; latency alone.
        _prefix("prefix-b4-d64-512", 4, 8, 2, 64, 512, 1, 40),
        # A busy server: answers of any length so far behind a system prompt of a few pages.
        _prefix("prefix-b64-4096", 64, 32, 8, 128, 4096, 1, 256),
        # Questions to one long document.
        _prefix("prefix-b24-g8-16384", 24, 64, 8, 128, 16384, 10, 300, page=64),
        # Long answers on a paged 8-bit cache, some slots idle, some sequences with a part of the prefix or none.
        _prefix("prefix-b64-8192-long-e4m3", 64, 32, 8, 128, 8192, 300, 2048, page=64, kv8=True, idle=3, mixed=True),
        # The weight of a step's attention, every step of a busy server.
        _mass("mass-step-b64-8192", 64, 32, 8, 128, 4000, 8192, decay=0.98),
        # What a prompt's last rows look at, before the prompt is cut down.
        _mass("mass-window-64", 1, 32, 8, 128, 8192, 8192, n=64, decay=0.0),
        # The same over a whole prompt.
        _mass("mass-prompt-2048", 1, 32, 8, 128, 2048, 2048, n=2048),
        # Prompts cut down to a quarter.
        _evict("evict-b8-8192-to-2048", 8, 8, 128, 8192, 8192, 2048, 4, 64),
        # A running batch back to its budget every 64 steps.
        _evict("evict-b64-2112-to-2048-e4m3", 64, 8, 128, 2000, 2112, 2048, 4, 256, page=64, kv8=True),
    ]


def draw(rng):
    """One more case of the ranges above; never dearer than the largest listed one of its kind."""
    kind = rng.choice(["rotary", "rotary", "prefix", "prefix", "prefix", "mass", "mass", "mass", "evict", "evict"])
    if kind == "rotary":
        hq, hkv, d = rng.choice([(32, 8, 128), (8, 2, 64), (64, 8, 128), (16, 8, 128), (32, 2, 64)])
        step = rng.random() < 0.5
        n = _log(rng, 1, 96) if step else _log(rng, 3, 2048 * 48 // (hq + 2 * hkv))
        return _rotary(None, step, n, hq, hkv, d, rng.choice([0, _log(rng, 100, 120000)]), kv8=rng.random() < 0.5,
                       layout=rng.choice(["pairs", "halves", "halves"]), part=rng.choice([0, 0, d // 2, d // 4]),
                       scaling=rng.choice(list(SCALINGS)), base=rng.choice([1e4, 5e5]))
    if kind == "prefix":
        hq, hkv, d = rng.choice([(8, 2, 64), (32, 8, 128), (64, 8, 128), (32, 2, 64), (16, 8, 128), (32, 8, 64)])
        batch, prefix = _log(rng, 1, 96), _log(rng, 5, 16384)
        prefix = min(prefix, 64 * 32 * 8192 * 128 // (batch * hq * d))
        hi = _log(rng, 1, min(2048, 64 * 8 * 2048 * 128 // (batch * hkv * d)))
        page = rng.choice([0, 64, 64, 256]) if (batch + 1) * hkv * d * max(prefix, hi) < 2**30 else 64
        return _prefix(None, batch, hq, hkv, d, prefix, max(1, hi // rng.choice([1, 4, 16])), hi, page=page,
                       kv8=rng.random() < 0.4, idle=rng.choice([0, batch // 8]), mixed=rng.random() < 0.4)
    if kind == "mass":
        hq, hkv, d = rng.choice([(8, 2, 64), (32, 8, 128), (64, 8, 128), (32, 2, 64), (16, 8, 128), (32, 8, 64)])
        kv8, page, decay = rng.random() < 0.4, rng.choice([0, 0, 64]), rng.choice([0.0, 0.9, 1.0])
        if rng.random() < 0.5:
            batch = _log(rng, 1, 96)
            hi = _log(rng, 20, min(20000, 64 * 8 * 8192 * 128 // (batch * hkv * d)))
            return _mass(None, batch, hq, hkv, d, max(1, hi // rng.choice([1, 2, 8])), hi, kv8=kv8, page=page, decay=decay)
        n = _log(rng, 2, 2048)
        rows = n + rng.choice([0, _log(rng, 10, 8000)])
        n = min(n, 32 * 2048 * 1024 // (hq * rows))
        return _mass(None, 1, hq, hkv, d, rows, rows, n=max(2, n), kv8=kv8, page=page, decay=decay, causal=rng.random() < 0.8)
    hkv, d = rng.choice([(8, 128), (2, 64), (4, 128), (8, 64)])
    batch = _log(rng, 1, 64)
    share = rng.choice([0.1, 0.25, 0.5, 0.97])
    hi = _log(rng, 30, min(16384, int(8 * 8 * 2048 * 128 / (batch * hkv * d * share))))
    keep = max(4, int(hi * share))
    return _evict(None, batch, hkv, d, max(1, hi // rng.choice([1, 1, 3])), hi, keep, rng.choice([0, min(4, keep // 4)]),
                  keep // rng.choice([2, 8, 30]), page=rng.choice([0, 64, 256]), kv8=rng.random() < 0.4)


def _log(rng, lo, hi):
    """A whole number of lo..hi, spread over its logarithm."""
    hi = max(lo, hi)
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _named(name, case):
    return case if name is None else {"name": name, **case}


def _rotary(name, step, n, hq, hkv, d, first, kv8, layout="halves", part=0, scaling="plain", base=1e4):
    return _named(name, {"kind": "rotary", "step": step, "n": n, "hq": hq, "hkv": hkv, "d": d, "first": first, "kv8": kv8,
                         "layout": layout, "part": part, "scaling": scaling, "base": base})


def _prefix(name, batch, hq, hkv, d, prefix, lo, hi, page=0, kv8=False, idle=0, mixed=False):
    return _named(name, {"kind": "prefix", "batch": batch, "hq": hq, "hkv": hkv, "d": d, "prefix": prefix, "lo": lo, "hi": hi,
                         "page": page, "kv8": kv8, "idle": idle, "mixed": mixed})


def _mass(name, batch, hq, hkv, d, lo, hi, n=0, page=0, kv8=False, decay=1.0, causal=True):
    """n: query rows of the one sequence (0: one row of every sequence)."""
    return _named(name, {"kind": "mass", "batch": batch, "hq": hq, "hkv": hkv, "d": d, "lo": lo, "hi": hi, "n": n, "page": page,
                         "kv8": kv8, "decay": decay, "causal": causal})


def _evict(name, batch, hkv, d, lo, hi, keep, sinks, recent, page=0, kv8=False):
    return _named(name, {"kind": "evict", "batch": batch, "hkv": hkv, "d": d, "lo": lo, "hi": hi, "keep": keep, "sinks": sinks,
                         "recent": recent, "page": page, "kv8": kv8})


# ---- inputs ---------------------------------------------------------------------------------------

def _generator(seed, stream=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000 * seed + stream)
    return g


def _normal(g, shape, amplitude=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * amplitude).to(BF16)


def _rows_of(case, seed, b, n):
    """K and V of n rows of sequence b, [H_kv, n, D]: some K rows larger than the others, which draw the weight."""
    g = _generator(seed, b + 1)
    shape = (case["hkv"], n, case["d"])
    k = torch.randn(shape, generator=g, device="cuda") * torch.exp(0.5 * torch.randn(shape[:2], generator=g, device="cuda"))[..., None]
    return k.to(BF16), _normal(g, shape)


def _spread(count, lo, hi, idle, seed):
    """Rows per sequence: the same numbers for every seed, in an order of its own; idle slots have none."""
    n = count - idle
    lens = np.round(np.linspace(lo, hi, n)) if n > 1 else np.array([hi] * n)
    return np.random.default_rng(seed).permutation(np.concatenate([np.zeros(idle), lens])).astype(np.int32)


def _prefix_plan(case, seed):
    """(own rows, rows of the prefix) of each sequence; the slot behind the batch holds the prefix and is idle."""
    own_lens = _spread(case["batch"], case["lo"], case["hi"], case["idle"], seed)
    shared = np.full(case["batch"], case["prefix"], np.int32)
    if case["mixed"]:
        kind = np.random.default_rng(seed + 1).permutation(np.arange(case["batch"]) % 5)
        shared[kind == 1] = 0
        shared[kind == 2] = (np.arange(case["batch"]) * case["prefix"] // case["batch"])[kind == 2]
    shared[own_lens == 0] = 0
    return np.append(own_lens, 0).astype(np.int32), np.append(shared, 0).astype(np.int32)


def _rotary_inputs(case, seed):
    """The projection's rows (heads of several magnitudes) and the two norms' weights, then each row's position and, of
    a step, its place in the cache."""
    g = _generator(seed)
    n, heads, d = case["n"], case["hq"] + 2 * case["hkv"], case["d"]
    x = torch.randn((n, heads, d), generator=g, device="cuda") * torch.exp(torch.randn((n, heads, 1), generator=g, device="cuda"))
    wq, wk = ((1 + 0.1 * torch.randn((d,), generator=g, device="cuda")).to(BF16) for _ in range(2))
    if case["step"]:
        pos = torch.randint(0, case["first"] + 64, (n,), generator=g, device="cuda", dtype=torch.int32)
        rows = torch.randint(0, 64, (n,), generator=g, device="cuda", dtype=torch.int32)
    else:
        pos = torch.arange(case["first"], case["first"] + n, device="cuda", dtype=torch.int32)
        rows = torch.arange(n, device="cuda", dtype=torch.int32)
    return x.reshape(n, heads * d).to(BF16), wq, wk, pos, rows


def _rope_of(case):
    """The rotation's numbers: (dims that turn, length trained on, factor, low, high)."""
    r = case["part"] or case["d"]
    return {"plain": (r, 0, 0.0, 0.0, 0.0), "linear": (r, 0, 4.0, 0.0, 0.0), "bands": (r, 8192, 8.0, 1.0, 4.0),
            "ramp": (r, 4096, 16.0, 1.0, 32.0)}[case["scaling"]]


def _step_inputs(case, seed, batch):
    g = _generator(seed)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    return _normal(g, (batch, hq, d)), _normal(g, (batch, hkv, d)), _normal(g, (batch, hkv, d))


def _mass_inputs(case, seed):
    """Rows per sequence, q ([B, H_q, D], or [H_q, n, D] of the one sequence) and the mass that the rows have."""
    g = _generator(seed)
    lens = _spread(case["batch"], case["lo"], case["hi"], 0, seed)
    shape = (case["hq"], case["n"], case["d"]) if case["n"] else (case["batch"], case["hq"], case["d"])
    q = _normal(g, shape)
    return lens, q, torch.rand((case["batch"], case["hkv"], case["hi"]), generator=g, device="cuda")


def _weight_sums(case, seed, lens, q, kv8):
    """log-sum-exp of the scaled scores of every query row, as attention gives it."""
    out, group = [], case["hq"] // case["hkv"]
    for b, rows in enumerate(lens.tolist()):
        k, _ = _rows_of(case, seed, b, rows)
        k = _decoded(*_encode(k.float())) if kv8 else k.float()
        rows_q = (q if case["n"] else q[b][:, None]).float().reshape(case["hkv"], -1, case["d"])
        s = rows_q @ k.transpose(1, 2).contiguous() / math.sqrt(case["d"])
        if case["n"]:
            at = torch.arange(case["n"], device="cuda") + rows - case["n"]
            seen = torch.arange(rows, device="cuda") <= at[:, None]
            s = s.reshape(case["hkv"], group, case["n"], rows).masked_fill(~seen, -math.inf) if case["causal"] else s
        out.append(torch.logsumexp(s, -1).reshape(case["hq"], -1))
    return out[0] if case["n"] else torch.cat(out, 1).t().contiguous()


def _evict_inputs(case, seed):
    """Rows per sequence and their mass: most rows little, a few much, some none at all."""
    g = _generator(seed)
    lens = _spread(case["batch"], case["lo"], case["hi"], 0, seed)
    shape = (case["batch"], case["hkv"], case["hi"])
    mass = torch.exp(2 * torch.randn(shape, generator=g, device="cuda"))
    return lens, torch.where(torch.rand(shape, generator=g, device="cuda") < 0.05, 0.0, mass)


# ---- caches in plain form ---------------------------------------------------------------------------

def _encode(x):
    """fp32 [..., D] as codes and one scale byte per row: the least 2^(byte - 127) whose 448-fold holds the row."""
    c = x.clamp(-TOP, TOP)
    bits = c.abs().amax(-1).view(torch.int32)
    byte = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(min=1)
    inverse = ((254 - byte) << 23).view(torch.float32)
    return (c * inverse[..., None]).to(E4M3).view(torch.uint8), byte.to(torch.uint8)


def _decoded(codes, byte):
    return codes.view(E4M3).float() * byte.view(E8M0).float()[..., None]


def _stored(case, k, v):
    """Rows as the pools take them."""
    if not case["kv8"]:
        return k.to(BF16), v.to(BF16)
    (kc, kb), (vc, vb) = _encode(k.float()), _encode(v.float())
    return kc, vc, kb, vb


def _pool_outputs(case, pools):
    """A cache's pools as the numbers that their bytes are (8-bit rows: codes, and the scales that multiply them)."""
    if not case["kv8"]:
        return dict(zip("kv", pools))
    return {"k": pools[0].view(E4M3), "v": pools[1].view(E4M3), "k_scale": pools[2].view(E8M0), "v_scale": pools[3].view(E8M0)}


def _page_order(lens, page):
    """Reservations that hand out the pages in turn, so that every sequence's rows are scattered over the pool."""
    if page:
        for p in range(1, -(-max(lens) // page) + 1):
            for b, n in enumerate(lens):
                if n > (p - 1) * page:
                    yield b, min(n, p * page)


def _plain_cache(case, lens):
    """Pools of an empty cache and, for a paged one, the page of each sequence's run of rows."""
    page, hkv, d, table = case.get("page", 0), case["hkv"], case["d"], None
    if page:
        table = -torch.ones((len(lens), -(-max(lens) // page)), dtype=torch.int64)
        for at, (b, n) in enumerate(_page_order(lens, page)):
            table[b, (n - 1) // page] = at
        shape, table = (int(table.max()) + 1, hkv, page), table.cuda()
    else:
        shape = (len(lens), hkv, -(-max(1, max(lens)) // 64) * 64)
    if case["kv8"]:
        return [torch.zeros(s, dtype=torch.uint8, device="cuda") for s in ((*shape, d), (*shape, d), shape, shape)], table
    return [torch.zeros((*shape, d), dtype=BF16, device="cuda") for _ in range(2)], table


def _places(pools, table, b, t):
    """Where rows t of sequences b lie in a pool: indices of its first dimension and of its rows."""
    page = pools[0].shape[2]
    return (table[b, t // page], t % page) if table is not None else (b, t)


def _plain_load(pools, table, b, rows):
    """Writes [H_kv, n, ...] rows of sequence b into each pool, from its first row on."""
    t = torch.arange(rows[0].shape[1], device="cuda")
    lead, at = _places(pools, table, torch.full_like(t, b), t)
    for pool, new in zip(pools, rows):
        pool[lead, :, at] = new.transpose(0, 1)


def _sequences(pools, table, rows, which=slice(None)):
    """The first rows of sequences, [B, H_kv, rows, D] fp32 (K, V)."""
    if table is not None:
        pages = table[which, :-(-rows // pools[0].shape[2])].clamp(min=0)
        pools = [p[pages].transpose(1, 2).flatten(2, 3)[:, :, :rows] for p in pools]
    else:
        pools = [p[which, :, :rows] for p in pools]
    if len(pools) == 2:
        return pools[0].float(), pools[1].float()
    return _decoded(pools[0], pools[2]), _decoded(pools[1], pools[3])


# ---- the engine -----------------------------------------------------------------------------------

class _Memory:
    """An engine's pool as a tensor's memory (keeps the engine alive)."""

    def __init__(self, engine, ptr, shape, typestr):
        self.engine = engine
        self.__cuda_array_interface__ = {"shape": shape, "typestr": typestr, "data": (ptr, False), "version": 2}


class _Engine:
    """A context of the C ABI: its library and its caches as tensors."""

    def __init__(self, case, lens, q_rows=1):
        from lara_amd import _lib

        self._lib, self.lib, self.ctx = _lib, _lib.lib(), ctypes.c_void_p()
        page, hkv, d, kv8 = case.get("page", 0), case["hkv"], case["d"], case["kv8"]
        pages = sum(-(-n // page) for n in lens) if page else 0
        cfg = _lib.GqaConfig(len(lens), case.get("hq", 4 * hkv), hkv, d, max(1, max(lens)), q_rows, 0.0, torch.cuda.current_device())
        if kv8:
            self.check(self.lib.gqa_create_kv8(ctypes.byref(cfg), page, pages, 1, ctypes.byref(self.ctx)))
        elif page:
            self.check(self.lib.gqa_create_paged(ctypes.byref(cfg), page, pages, ctypes.byref(self.ctx)))
        else:
            self.check(self.lib.gqa_create(ctypes.byref(cfg), ctypes.byref(self.ctx)))
        for b, n in _page_order(lens, page):
            self.check(self.lib.gqa_paged_reserve(self.ctx, b, n))
        k, v, ks, vs, cap = *(ctypes.c_void_p() for _ in range(4)), ctypes.c_int32()
        self.check(self.lib.gqa_cache_pointers(self.ctx, ctypes.byref(k), ctypes.byref(v), ctypes.byref(cap)))
        shape = (pages if page else len(lens), hkv, cap.value)
        if kv8:
            self.check(self.lib.gqa_kv8_scales(self.ctx, ctypes.byref(ks), ctypes.byref(vs)))
            self.pools = [self.tensor(p, s, "|u1") for p, s in ((k, (*shape, d)), (v, (*shape, d)), (ks, shape), (vs, shape))]
        else:
            self.pools = [self.tensor(p, (*shape, d), "<i2").view(BF16) for p in (k, v)]

    def tensor(self, p, shape, typestr):
        return torch.as_tensor(_Memory(self, p.value, shape, typestr), device="cuda")

    def check(self, rc):
        self._lib.check(rc, "libgqa")

    def load(self, b, k, v):
        if k.shape[1]:
            self.check(self.lib.gqa_load_kv_device(self.ctx, b, 0, k.shape[1], _ptr(k), _ptr(v), None))

    def __del__(self):
        if self.ctx:
            self.lib.gqa_destroy(self.ctx)


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


class _State:
    """What a program keeps between calls: buffers and, where the framework runs them, the calls of one pass."""

    def __init__(self, case, **kept):
        self.case, self.engine, self.call, self.outputs = case, None, None, None
        self.__dict__.update(kept)

    def bind(self, engine, name, args, outputs):
        self.engine, self.call, self.outputs = engine, (getattr(engine.lib, name), args), outputs


def prepare(case, seed):
    return {"rotary": _prepare_rotary, "prefix": _prepare_prefix, "mass": _prepare_mass, "evict": _prepare_evict}[case["kind"]](case, seed)


def _filled(s, case, seed, lens, q_rows=1):
    """A cache that holds the sequences' rows: the framework's, or plain pools."""
    if own:
        engine = _Engine(case, lens, q_rows)
        for b, n in enumerate(lens):
            engine.load(b, *_rows_of(case, seed, b, n))
        return engine
    s.pools, s.table = _plain_cache(case, lens)
    for b, n in enumerate(lens):
        if n:
            _plain_load(s.pools, s.table, b, _stored(case, *_rows_of(case, seed, b, n)))
    return None


def _prepare_rotary(case, seed):
    n, hq, hkv, d, step = case["n"], case["hq"], case["hkv"], case["d"], case["step"]
    x, wq, wk, pos, rows = _rotary_inputs(case, seed)
    s = _State(case, x=x, wq=wq, wk=wk, pos=pos, rows=rows)
    lens = [64] * n if step else [n]
    if own:
        engine = _Engine(case, lens, 1 if step else n)
        r, trained, factor, low, high = _rope_of(case)
        s.rope = engine._lib.GqaRope(LAYOUTS[case["layout"]], r, SCALINGS[case["scaling"]], trained, case["base"], factor, low, high, 0.0)
        s.q = torch.zeros((n, hq, d) if step else (hq, n, d), dtype=BF16, device="cuda")
        out = {"q": s.q, **_pool_outputs(case, engine.pools)}
        if step:
            s.bind(engine, "gqa_qk_norm_rotary_step_device",
                   (engine.ctx, _ptr(x), x.shape[1], _ptr(wq), _ptr(wk), 1e-6, _ptr(pos), _ptr(rows), ctypes.byref(s.rope), _ptr(s.q), None), out)
        else:
            s.bind(engine, "gqa_qk_norm_rotary_device",
                   (engine.ctx, 0, _ptr(x), x.shape[1], n, _ptr(wq), _ptr(wk), 1e-6, case["first"], case["first"], 0,
                    ctypes.byref(s.rope), _ptr(s.q), None), out)
        return s
    s.pools, _ = _plain_cache(case, lens)
    return s


def _prepare_prefix(case, seed):
    own_lens, shared = _prefix_plan(case, seed)
    batch = case["batch"]
    q, k_new, v_new = _step_inputs(case, seed, batch + 1)
    lens = torch.from_numpy(own_lens).cuda()
    s = _State(case, q=q, k=k_new, v=v_new, lens=lens, positions=lens - 1, shared=torch.from_numpy(shared).cuda())
    engine = _filled(s, case, seed, [*own_lens[:batch].tolist(), case["prefix"]])
    if own:
        s.o, s.lse = torch.empty_like(q), torch.empty((batch + 1, case["hq"]), device="cuda")
        s.bind(engine, "gqa_decode_append_prefix_device",
               (engine.ctx, _ptr(q), _ptr(k_new), _ptr(v_new), _ptr(s.positions), batch, case["prefix"], _ptr(s.shared), _ptr(lens),
                _ptr(s.o), _ptr(s.lse), None), {"o": s.o, "lse": s.lse, **_pool_outputs(case, engine.pools)})
    return s


def _prepare_mass(case, seed):
    lens, q, mass = _mass_inputs(case, seed)
    lse = _weight_sums(case, seed, lens, q, case["kv8"])
    s = _State(case, q=q, lse=lse, mass=mass, lens=torch.from_numpy(lens).cuda())
    engine = _filled(s, case, seed, lens.tolist(), max(1, case["n"]))
    if own and case["n"]:
        rows = int(lens[0])
        s.bind(engine, "gqa_attention_mass_device",
               (engine.ctx, 0, _ptr(q), case["n"], rows - case["n"], rows, 0, int(case["causal"]), _ptr(lse), case["decay"], _ptr(mass), None),
               {"mass": mass})
    elif own:
        s.bind(engine, "gqa_attention_mass_step_device",
               (engine.ctx, _ptr(q), _ptr(s.lens), _ptr(lse), case["decay"], _ptr(mass), None), {"mass": mass})
    return s


def _prepare_evict(case, seed):
    lens, mass = _evict_inputs(case, seed)
    s = _State(case, mass=mass, lens=torch.from_numpy(lens).cuda(), new_mass=torch.zeros_like(mass))
    engine = _filled(s, case, seed, lens.tolist())
    if own:
        s.new_lens = torch.zeros_like(s.lens)
        s.kept = torch.zeros((case["batch"], case["hkv"], case["keep"]), dtype=torch.int32, device="cuda")
        s.bind(engine, "gqa_evict_device",
               (engine.ctx, _ptr(mass), _ptr(s.lens), case["keep"], case["sinks"], case["recent"], _ptr(s.new_mass), _ptr(s.new_lens),
                _ptr(s.kept), None), {"kept": s.kept, "lens": s.new_lens, "mass": s.new_mass, **_pool_outputs(case, engine.pools)})
    return s


# ---- one pass ----------------------------------------------------------------------------------------

def run(state):
    if own:
        fn, args = state.call
        rc = fn(*args)
        if rc:
            state.engine.check(rc)
        return state.outputs
    return {"rotary": _plain_rotary, "prefix": _plain_prefix, "mass": _plain_mass, "evict": _plain_evict}[state.case["kind"]](state)


def _frequencies(case):
    """Angle per position of each pair that turns (64 bits), and what multiplies cosine and sine."""
    r, trained, factor, low, high = _rope_of(case)
    p = torch.arange(r // 2, device="cuda", dtype=torch.float64)
    f = case["base"] ** (-2.0 * p / r)
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] == "bands":  # by turns over the length trained on: many kept, few divided, blended between
        turns = trained * f / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        return f * keep + f / factor * (1 - keep), 1.0
    if case["scaling"] == "ramp":  # the same two ends, joined along the pair's index
        first, last = (r * math.log(trained / (t * 2 * math.pi)) / (2 * math.log(case["base"])) for t in (high, low))
        first, last = max(math.floor(first), 0), min(math.ceil(last), r - 1)
        part = ((p - first) / max(last - first, 0.001)).clamp(0, 1)
        return f / factor * part + f * (1 - part), 0.1 * math.log(factor) + 1
    return f, 1.0


def _plain_rotary(s):
    case = s.case
    n, hq, hkv, d = case["n"], case["hq"], case["hkv"], case["d"]
    h = s.x.float().reshape(n, hq + 2 * hkv, d)
    qk = h[:, :hq + hkv]
    weight = torch.cat((s.wq.float().expand(hq, d), s.wk.float().expand(hkv, d)))
    qk = qk / torch.sqrt((qk * qk).mean(-1, keepdim=True) + 1e-6) * weight
    f, magnitude = _frequencies(case)
    angle = s.pos.double()[:, None] * f
    cos, sin = (magnitude * torch.cos(angle)).float()[:, None], (magnitude * torch.sin(angle)).float()[:, None]
    r = 2 * f.numel()
    turned, rest = qk[..., :r], qk[..., r:]
    a, b = (turned[..., :r // 2], turned[..., r // 2:]) if case["layout"] == "halves" else (turned[..., 0::2], turned[..., 1::2])
    ab = (a * cos - b * sin, a * sin + b * cos)
    qk = torch.cat((torch.cat(ab, -1) if case["layout"] == "halves" else torch.stack(ab, -1).flatten(-2), rest), -1)
    lead = torch.arange(n, device="cuda") if case["step"] else torch.zeros_like(s.rows)
    for pool, rows in zip(s.pools, _stored(case, qk[:, hq:], h[:, hq + hkv:])):
        pool[lead, :, s.rows] = rows
    q = qk[:, :hq].to(BF16)
    return {"q": q if case["step"] else q.transpose(0, 1).contiguous(), **_pool_outputs(case, s.pools)}


def _plain_prefix(s):
    case, pos = s.case, s.positions
    batch, hkv, d, prefix = case["batch"], case["hkv"], case["d"], case["prefix"]
    b = torch.arange(batch + 1, device="cuda")
    # idle slots write nothing: they repeat the last writing slot's row
    src = torch.where(pos >= 0, b, torch.where(pos >= 0, b, -1).amax().clamp(min=0))
    lead, at = _places(s.pools, s.table, src, pos[src].long().clamp(min=0))
    for pool, new in zip(s.pools, _stored(case, s.k, s.v)):
        pool[lead, :, at] = new[src]
    kp, vp = _sequences(s.pools, s.table, prefix, slice(batch, batch + 1))
    ko, vo = _sequences(s.pools, s.table, case["hi"])
    q = s.q.float().reshape(batch + 1, hkv, -1, d)
    every = q.transpose(0, 1).reshape(hkv, -1, d)  # the queries of all sequences, by kv head
    sp = (every @ kp[0].transpose(1, 2).contiguous()).reshape(hkv, batch + 1, -1, prefix).transpose(0, 1) / math.sqrt(d)
    so = q @ ko.transpose(2, 3).contiguous() / math.sqrt(d)
    sp = torch.where(torch.arange(prefix, device="cuda") < s.shared[:, None, None, None], sp, -math.inf)
    so = torch.where(torch.arange(case["hi"], device="cuda") < s.lens[:, None, None, None], so, -math.inf)
    m = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
    base = torch.where(torch.isinf(m), 0.0, m)
    ep, eo = torch.exp(sp - base), torch.exp(so - base)
    total = ep.sum(-1, keepdim=True) + eo.sum(-1, keepdim=True)
    o = (ep.transpose(0, 1).reshape(hkv, -1, prefix) @ vp[0]).reshape(hkv, batch + 1, -1, d).transpose(0, 1) + eo @ vo
    o = o / torch.where(total > 0, total, 1.0)
    return {"o": o.reshape(s.q.shape).to(BF16), "lse": (m + torch.log(total)).reshape(batch + 1, -1), **_pool_outputs(case, s.pools)}


def _plain_mass(s):
    case = s.case
    n, hkv, d, rows = case["n"], case["hkv"], case["d"], case["hi"]
    k, _ = _sequences(s.pools, s.table, rows)
    q = (s.q.reshape(1, hkv, -1, d) if n else s.q.reshape(case["batch"], hkv, -1, d)).float()
    lse = s.lse.reshape(q.shape[0], hkv, -1, 1)
    p = torch.exp(q @ k.transpose(2, 3).contiguous() / math.sqrt(d) - lse)
    at = torch.arange(rows, device="cuda")
    if n and case["causal"]:
        p = torch.where(at <= (torch.arange(p.shape[2], device="cuda") % n + rows - n)[:, None], p, 0.0)
    new = p.sum(2)
    there = at < s.lens[:, None, None]
    s.mass.copy_(torch.where(there, case["decay"] * s.mass + new, s.mass))
    return {"mass": s.mass}


def _plain_evict(s):
    case = s.case
    batch, hkv, keep, sinks, recent, rows = case["batch"], case["hkv"], case["keep"], case["sinks"], case["recent"], case["hi"]
    t = torch.arange(rows, device="cuda")
    lens = s.lens.long()[:, None, None]
    new_lens = lens.clamp(max=keep)
    # the first and last rows come before every other, rows that are not there behind all; equal ones by their index
    order = torch.where((t < sinks) | (t >= lens - recent) & (t < lens), math.inf, s.mass)
    order = torch.where(t < lens, order, -math.inf)
    ranked = torch.sort(order, dim=-1, descending=True, stable=True).indices
    chosen = torch.zeros((batch, hkv, rows), dtype=torch.bool, device="cuda").scatter_(-1, ranked, (t < new_lens).expand(batch, hkv, rows))
    kept = torch.sort(torch.where(chosen, t, rows), dim=-1).values[..., :keep]
    if kept.shape[-1] < keep:
        kept = torch.cat((kept, torch.full((batch, hkv, keep - kept.shape[-1]), rows, device="cuda")), -1)
    there = kept < rows
    b, h, j = (x[there] for x in torch.broadcast_tensors(torch.arange(batch, device="cuda")[:, None, None], torch.arange(hkv, device="cuda")[:, None],
                                                         torch.arange(keep, device="cuda")))
    lead, at = _places(s.pools, s.table, b, kept[there])
    to_lead, to = _places(s.pools, s.table, b, j)
    for pool in s.pools:
        pool[to_lead, h, to] = pool[lead, h, at]
    s.new_mass.copy_(torch.where(t < lens, 0.0, s.new_mass))
    s.new_mass[b, h, j] = s.mass[b, h, kept[there]]
    return {"kept": torch.where(there, kept, -1).to(torch.int32), "lens": new_lens[:, 0, 0].to(torch.int32), "mass": s.new_mass,
            **_pool_outputs(case, s.pools)}


# ---- what a pass has to do, and its results in 64 bits --------------------------------------------------

def _row_bytes(case):
    return case["d"] + 1 if case["kv8"] else 2 * case["d"]


def work(case):
    d, hkv = case["d"], case["hkv"]
    if case["kind"] == "rotary":
        n, hq = case["n"], case["hq"]
        return {"bytes": n * ((hq + 2 * hkv) * 2 * d + hq * 2 * d + 2 * hkv * _row_bytes(case)) + 4 * d, "flops": 7 * n * (hq + hkv) * d}
    if case["kind"] == "prefix":
        own_lens, shared = _prefix_plan(case, 0)
        keys, new = int(own_lens.sum()), int((own_lens > 0).sum())
        moved = 2 * hkv * ((keys + int(shared.max())) * _row_bytes(case) + new * 2 * d) + (case["batch"] + 1) * case["hq"] * (4 * d + 4)
        return {"bytes": moved, "flops": 4 * case["hq"] * d * (keys + int(shared.sum()))}
    if case["kind"] == "mass":
        rows = int(_spread(case["batch"], case["lo"], case["hi"], 0, 0).sum())
        n = case["n"]
        pairs = rows if not n else n * (rows - n) + n * (n + 1) // 2 if case["causal"] else n * rows
        moved = hkv * rows * (_row_bytes(case) + (8 if case["decay"] else 4)) + case["hq"] * max(n, case["batch"]) * (2 * d + 4)
        return {"bytes": moved, "flops": 2 * case["hq"] * d * pairs}
    lens = _spread(case["batch"], case["lo"], case["hi"], 0, 0)
    kept = int(np.minimum(lens, case["keep"])[lens > case["keep"]].sum())
    return {"bytes": hkv * (int(lens.sum()) * 8 + kept * (4 * _row_bytes(case) + 4)), "flops": hkv * int(lens.sum())}


def _exact_row(x):
    """A row as the 8-bit cache holds it, in 64 bits: the rounding to four significant bits written out."""
    x = x.double().clamp(-TOP, TOP)
    top = x.abs().amax(-1, keepdim=True)
    _, e = torch.frexp(top)  # top = f * 2^e, 1/2 <= f < 1
    e = torch.where(top == 0, -126, e)
    scale = torch.exp2((torch.where(top > 448.0 * torch.exp2((e - 9).double()), e - 8, e - 9)).clamp(min=-126).double())
    _, ce = torch.frexp(x / scale)
    step = torch.exp2((ce - 1).clamp(min=-6).double() - 3) * scale
    return torch.round(x / step) * step


def _rows64(case, k, v):
    return [_exact_row(t) if case["kv8"] else t.double() for t in (k, v)]


def _no_pools(case):
    return dict.fromkeys(("k", "v", "k_scale", "v_scale") if case["kv8"] else ("k", "v"))


def _exact_rotary(case, seed):
    x, wq, _, pos, _ = _rotary_inputs(case, seed)
    n, hq, d = case["n"], case["hq"], case["d"]
    r, trained, factor, low, high = _rope_of(case)
    q = x.double().reshape(n, -1, d)[:, :hq]
    q = q * (q.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * wq.double()
    rates, length = [], 1.0
    for pair in range(r // 2):
        rate = math.exp(-2 * pair / r * math.log(case["base"]))
        wave = 2 * math.pi / rate
        if case["scaling"] == "linear":
            rate /= factor
        elif case["scaling"] == "bands" and wave > trained / low:
            rate /= factor
        elif case["scaling"] == "bands" and wave > trained / high:
            blend = (trained / wave - low) / (high - low)
            rate *= (1 - blend) / factor + blend
        elif case["scaling"] == "ramp":
            ends = [r * math.log(trained / (2 * math.pi * turns)) / (2 * math.log(case["base"])) for turns in (high, low)]
            a, b = max(math.floor(ends[0]), 0), min(math.ceil(ends[1]), r - 1)
            part = min(max((pair - a) / (b - a if b > a else 0.001), 0.0), 1.0)
            rate *= part / factor + 1 - part
            length = 1 + 0.1 * math.log(factor)
        rates.append(rate)
    angle = pos.double()[:, None, None] * torch.tensor(rates, dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.full_like(angle, length), angle)
    if case["layout"] == "halves":
        z = torch.complex(q[..., :r // 2].contiguous(), q[..., r // 2:r].contiguous()) * turn
        turned = torch.cat((z.real, z.imag), -1)
    else:
        turned = torch.view_as_real(torch.view_as_complex(q[..., :r].reshape(n, hq, r // 2, 2).contiguous()) * turn).flatten(-2)
    q = torch.cat((turned, q[..., r:]), -1)
    return {"q": q if case["step"] else q.transpose(0, 1).contiguous(), **_no_pools(case)}


def _exact_prefix(case, seed):
    own_lens, shared = _prefix_plan(case, seed)
    batch, hq, d = case["batch"], case["hq"], case["d"]
    q, k_new, v_new = _step_inputs(case, seed, batch + 1)
    o = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    kp, vp = _rows64(case, *_rows_of(case, seed, batch, case["prefix"]))
    for b in range(batch):
        n, p = int(own_lens[b]), int(shared[b])
        if not n + p:
            continue
        k, v = _rows_of(case, seed, b, n)
        if n:
            k[:, -1], v[:, -1] = k_new[b], v_new[b]
        k, v = (torch.cat((x[:, :p], y), 1) for x, y in zip((kp, vp), _rows64(case, k, v)))
        s = q[b].double().reshape(case["hkv"], -1, d) @ k.transpose(1, 2).contiguous() / math.sqrt(d)
        o[b] = (torch.softmax(s, -1) @ v).reshape(hq, d)
        lse[b] = torch.logsumexp(s, -1).reshape(hq)
    return {"o": o, "lse": lse, **_no_pools(case)}


def _exact_mass(case, seed):
    lens, q, mass = _mass_inputs(case, seed)
    lse = _weight_sums(case, seed, lens, q, case["kv8"]).double()
    out, n, group = mass.double(), case["n"], case["hq"] // case["hkv"]
    for b, rows in enumerate(lens.tolist()):
        k, _ = _rows64(case, *_rows_of(case, seed, b, rows))
        for h in range(case["hkv"]):
            heads = slice(h * group, (h + 1) * group)
            qs, ls = (q[heads], lse[heads]) if n else (q[b, heads, None], lse[b, heads, None])
            p = torch.exp(qs.double().reshape(-1, case["d"]) @ k[h].t().contiguous() / math.sqrt(case["d"]) - ls.reshape(-1, 1)).reshape(group, -1, rows)
            if n and case["causal"]:
                p = p.tril(rows - n)
            out[b, h, :rows] = case["decay"] * out[b, h, :rows] + p.sum((0, 1))
    return {"mass": out}


def _exact_evict(case, seed):
    lens, mass = _evict_inputs(case, seed)
    new_mass = torch.zeros_like(mass, dtype=torch.float64)
    rows_of = []
    host = mass.cpu().numpy()
    for b, n in enumerate(lens.tolist()):
        kept = []
        for h in range(case["hkv"]):
            at = np.arange(n)
            if n > case["keep"]:
                last = n - case["recent"]
                middle = at[case["sinks"]:last]
                best = middle[np.argsort(-host[b, h, middle], kind="stable")[:case["keep"] - case["sinks"] - case["recent"]]]
                at = np.concatenate((at[:case["sinks"]], np.sort(best), at[last:]))
            kept.append(torch.from_numpy(at).cuda())
            new_mass[b, h, :at.size] = mass[b, h][kept[-1]].double()
        rows_of.append(torch.stack(kept))
    out = {"kept": None, "lens": None, "mass": new_mass, **_no_pools(case)}
    if not case["kv8"] and not case["page"]:
        for name, side in (("k", 0), ("v", 1)):
            pool = torch.zeros((len(lens), case["hkv"], -(-int(lens.max()) // 64) * 64, case["d"]), dtype=torch.float64, device="cuda")
            for b, n in enumerate(lens.tolist()):
                x = _rows_of(case, seed, b, n)[side].double()
                pool[b, :, :n] = x
                pool[b, :, :rows_of[b].shape[1]] = torch.take_along_dim(x, rows_of[b][..., None], 1)
            out[name] = pool
    return out


def exact(case, seed):
    return {"rotary": _exact_rotary, "prefix": _exact_prefix, "mass": _exact_mass, "evict": _exact_evict}[case["kind"]](case, seed)
