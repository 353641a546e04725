"""Products with 4-bit weights against float64, and a decode step of all the serving operators together.

Bound of y: its rounding to bf16 (2^-8 of it); with a norm weight that is no power of two the rounding of x * gamma (2^-8
of each term, so of S = sum |w x gamma| / rms); and fp32.  The codes enter as 128 + c and leave through -136 x, so the sums
are over terms of up to 264 |x| per group, scaled by s: with at most 40 additions per group of 128 (each MFMA's 32 terms
may be added in sequence), hidden / 128 groups and the waves' parts, each off by 2^-24 of sums of at most
T = 264 sum s |x gamma| / rms: 2^-18 of T.
"""
import ctypes

import numpy as np
import pytest

from lara_amd import _lib, w4
from lara_amd.attn_driver import AttentionAccelerator
from oracle import gqa_oracle as orc
from oracle import serving_oracle as so
from tests._gen import bf16_normal
from tests._serving import call, dev, ptr, scatter_reserve, words

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def f64(w):
    return orc.bf16_u16_to_fp32(w).astype(np.float64)


@pytest.fixture(scope="module")
def acc():
    with AttentionAccelerator(n_q_heads=8, n_kv_heads=2, head_dim=64, max_seq_len=64) as a:
        yield a


def matrix(rng, rows, hidden, group):
    codes = rng.integers(0, 256, (rows, hidden // 2)).astype(np.uint8)
    scales = orc.bf16_rne((0.3 * hidden**-0.5 * np.exp(rng.standard_normal((rows, hidden // group))) *
                           rng.choice([-1, 1], (rows, hidden // group))).astype(np.float32))
    return codes, scales


def packed(acc, codes, scales, group):
    rows, hidden = codes.shape[0], 2 * codes.shape[1]
    wb, sb = w4.packed_bytes(rows, hidden, group)
    w, s = torch.empty(wb, dtype=torch.uint8, device="cuda"), torch.empty(sb, dtype=torch.uint8, device="cuda")
    c, g = dev(codes), dev(scales)
    acc.w4_pack_device(c.data_ptr(), g.data_ptr(), rows, hidden, group, w.data_ptr(), s.data_ptr())
    torch.cuda.synchronize()
    return w, s


def check(y, x, gamma, eps, codes, scales, exact_gamma=False):
    m = so.w4_matrix(codes, f64(scales))
    s = np.repeat(np.abs(f64(scales)), m.shape[1] // scales.shape[1], 1)
    xn = f64(x)
    if gamma is not None:
        xn = xn / np.sqrt((xn * xn).mean(-1, keepdims=True) + eps) * f64(gamma)
    ref = xn @ m.T
    bound = 2.0**-8 * np.abs(ref) + 2.0**-18 * 264 * (np.abs(xn) @ s.T)
    if gamma is not None and not exact_gamma:
        bound += 2.0**-8 * (np.abs(xn) @ np.abs(m).T)
    err = np.abs(f64(y) - ref)
    assert np.all(err <= bound), float((err / bound).max())
    # (the roundings of many terms do not add up: a wrong term shows here)
    assert np.linalg.norm(f64(y) - ref) <= 2.0**-7 * np.linalg.norm(ref)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,rows,hidden", [(1, 16, 128), (1, 768, 1024), (3, 17, 256), (16, 100, 1152), (17, 256, 384), (64, 48, 2048),
                                           (130, 33, 128)])
def test_project_against_float64(acc, group, n, rows, hidden):
    rng = np.random.default_rng(n * rows + group)
    codes, scales = matrix(rng, rows, hidden, group)
    w, s = packed(acc, codes, scales, group)
    x = bf16_normal(rng, (n, hidden))
    gamma = orc.bf16_rne((1 + 0.2 * rng.standard_normal(hidden)).astype(np.float32))
    two = orc.bf16_rne(2.0 ** rng.integers(-3, 4, hidden).astype(np.float32))
    ldy = rows + 3
    for g, kind in ((None, "plain"), (two, "powers"), (gamma, "any")):
        y = torch.full((n + 1, ldy), 7, dtype=torch.int16, device="cuda")
        xd, gd = dev(x), dev(g) if g is not None else None
        acc.w4_project_device(xd.data_ptr(), n, hidden, w.data_ptr(), s.data_ptr(), group, rows, y.data_ptr(),
                              rms_weight_ptr=gd.data_ptr() if g is not None else None, rms_eps=1e-5, ldy=ldy)
        torch.cuda.synchronize()
        got = words(y)
        check(got[:n, :rows], x, g, 1e-5, codes, scales, kind == "powers")
        assert np.all(got[n:] == 7) and np.all(got[:, rows:] == 7)  # what is not y is as it was


@pytest.mark.parametrize("n,rows,hidden,group", [(1, 5200, 256, 32), (16, 5187, 160, 32), (5, 5200, 384, 128), (3, 10250, 128, 64),
                                                 (16, 10250, 288, 32), (33, 5203, 288, 32), (64, 5200, 192, 64),
                                                 (47, 5200, 1152, 128), (40, 10241, 96, 32)])
def test_many_rows_take_several_tiles_a_work_group(acc, n, rows, hidden, group):
    """Against float64, and a token alone and among others gives the same words."""
    rng = np.random.default_rng(n + rows + hidden)
    codes, scales = matrix(rng, rows, hidden, group)
    w, s = packed(acc, codes, scales, group)
    x = bf16_normal(rng, (n, hidden))
    gamma = orc.bf16_rne((1 + 0.2 * rng.standard_normal(hidden)).astype(np.float32))
    xd, gd = dev(x), dev(gamma)
    for g in (None, gamma):
        y = torch.full((n + 1, rows + 1), 7, dtype=torch.int16, device="cuda")
        gp = gd.data_ptr() if g is not None else None
        acc.w4_project_device(xd.data_ptr(), n, hidden, w.data_ptr(), s.data_ptr(), group, rows, y.data_ptr(), rms_weight_ptr=gp,
                              rms_eps=1e-5, ldy=rows + 1)
        last = torch.zeros(96, dtype=torch.int16, device="cuda")  # (the first 96 rows alone: another form of the kernel)
        acc.w4_project_device(xd[n - 1 :].data_ptr(), 1, hidden, w.data_ptr(), s.data_ptr(), group, 96, last.data_ptr(),
                              rms_weight_ptr=gp, rms_eps=1e-5)
        torch.cuda.synchronize()
        got = words(y)
        check(got[:n, :rows], x, g, 1e-5, codes, scales)
        assert np.all(got[n:] == 7) and np.all(got[:, rows:] == 7)
        assert torch.equal(last, y[n - 1, :96])


@pytest.mark.parametrize("hidden,group", [(160, 32), (96, 32), (192, 64), (2080, 32)])
def test_hidden_that_ends_inside_a_block(acc, hidden, group):
    rng = np.random.default_rng(hidden)
    codes, scales = matrix(rng, 40, hidden, group)
    w, s = packed(acc, codes, scales, group)
    x = bf16_normal(rng, (5, hidden))
    y = torch.zeros((5, 40), dtype=torch.int16, device="cuda")
    xd = dev(x)
    acc.w4_project_device(xd.data_ptr(), 5, hidden, w.data_ptr(), s.data_ptr(), group, 40, y.data_ptr())
    torch.cuda.synchronize()
    check(words(y), x, None, 0.0, codes, scales)


def test_norm_of_small_and_large_tokens(acc):
    """Tokens whose squares leave the normal range of fp32: their mean is subnormal (2^-21 of it at 2^-128), or near the top.
    x * gamma is 2^-64 and 2^60 here, so the products and their sums stay normal."""
    rng = np.random.default_rng(7)
    codes, scales = matrix(rng, 48, 256, 64)
    w, s = packed(acc, codes, scales, 64)
    x = orc.bf16_rne((f64(bf16_normal(rng, (6, 256))) * np.array([2.0**-64, 2.0**60, 1, 2.0**-40, 2.0**-64, 2.0**-63])[:, None]).astype(np.float32))
    gamma = orc.bf16_rne(2.0 ** rng.integers(-3, 4, 256).astype(np.float32))
    xd, gd = dev(x), dev(gamma)
    for n in (6, 1):
        y = torch.zeros((n, 48), dtype=torch.int16, device="cuda")
        acc.w4_project_device(xd.data_ptr(), n, 256, w.data_ptr(), s.data_ptr(), 64, 48, y.data_ptr(), rms_weight_ptr=gd.data_ptr(), rms_eps=0.0)
        torch.cuda.synchronize()
        check(words(y), x[:n], gamma, 0.0, codes, scales, exact_gamma=True)


def test_unpacked_matrix_is_exactly_rounded(acc):
    rng = np.random.default_rng(5)
    for rows, hidden, group in ((33, 288, 32), (64, 256, 128), (7, 64, 64)):
        codes, scales = matrix(rng, rows, hidden, group)
        w, s = packed(acc, codes, scales, group)
        out = torch.full((rows + 1, hidden), 7, dtype=torch.int16, device="cuda")
        acc.w4_unpack_device(w.data_ptr(), s.data_ptr(), rows, hidden, group, out.data_ptr())
        torch.cuda.synchronize()
        want = orc.bf16_rne(so.w4_matrix(codes, f64(scales)).astype(np.float32))  # (12 significant bits: exact in fp32)
        assert np.array_equal(f64(words(out)[:rows]), f64(want)) and np.all(words(out)[rows] == 7)


def test_a_token_does_not_depend_on_the_others(acc):
    rng = np.random.default_rng(6)
    codes, scales = matrix(rng, 96, 512, 64)
    w, s = packed(acc, codes, scales, 64)
    x, gamma = dev(bf16_normal(rng, (70, 512))), dev(bf16_normal(rng, (512,)))

    def run(x):
        y = torch.zeros((x.shape[0], 96), dtype=torch.int16, device="cuda")
        acc.w4_project_device(x.data_ptr(), x.shape[0], 512, w.data_ptr(), s.data_ptr(), 64, 96, y.data_ptr(),
                              rms_weight_ptr=gamma.data_ptr())
        torch.cuda.synchronize()
        return y

    whole = run(x)
    for a, b in ((0, 1), (5, 17), (16, 64), (69, 70)):
        assert torch.equal(run(x[a:b].clone()), whole[a:b])
    x[3] = 0x7FC0  # one token of NaN
    again = run(x)
    keep = [t for t in range(70) if t != 3]
    assert torch.equal(again[keep], whole[keep])


def test_refusals(acc):
    lib, R, U, N = _lib.lib(), _lib.GQA_ERR_RANGE, _lib.GQA_ERR_UNSUPPORTED, _lib.GQA_ERR_NULL
    t = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    p = [ctypes.c_void_p(t.data_ptr() + 8192 * i) for i in range(6)]
    odd = ctypes.c_void_p(t.data_ptr() + 1)
    c = acc._ctx

    def project(x=p[0], n=2, hidden=128, w=p[1], s=p[2], group=32, rows=16, g=None, eps=0.0, y=p[3], ldy=16):
        return lib.gqa_w4_project_device(c, x, n, hidden, w, s, group, rows, g, eps, y, ldy, None)

    assert project(group=16) == U
    assert project(x=None) == project(y=None) == project(w=None) == project(s=None) == N
    for bad in (dict(n=0), dict(n=_lib.GQA_W4_MAX_TOKENS + 1), dict(hidden=144), dict(hidden=0), dict(rows=0), dict(ldy=15),
                dict(eps=-1.0), dict(eps=float("nan")), dict(x=odd), dict(g=odd), dict(w=odd), dict(s=odd), dict(y=odd),
                dict(y=p[0]), dict(y=p[1]), dict(y=p[2]), dict(y=p[4], g=p[4])):
        assert project(**bad) == R, bad
    assert lib.gqa_w4_pack_device(c, p[0], p[1], 16, 128, 48, p[2], p[3], None) == U
    assert lib.gqa_w4_pack_device(c, p[0], odd, 16, 128, 32, p[2], p[3], None) == R
    assert lib.gqa_w4_pack_device(c, p[0], p[1], 16, 128, 32, odd, p[3], None) == R
    assert lib.gqa_w4_pack_device(c, p[0], p[1], 16, 128, 32, p[0], p[3], None) == R
    assert lib.gqa_w4_pack_device(c, p[0], p[1], 16, 128, 32, p[2], p[2], None) == R
    assert lib.gqa_w4_unpack_device(c, p[0], p[1], 16, 128, 32, p[0], None) == R
    assert lib.gqa_w4_unpack_device(c, p[0], p[1], 16, 100, 32, p[2], None) == R
    assert lib.gqa_w4_unpack_device(c, p[0], p[1], 16, 128, 32, None, None) == N
    assert project() == _lib.GQA_OK
    torch.cuda.synchronize()


def test_refuses_a_stride_past_31_bits(acc):
    t = torch.zeros(1 << 14, dtype=torch.int16, device="cuda")
    at = [ptr(t[1024 * i :]) for i in range(4)]
    assert _lib.lib().gqa_w4_project_device(acc._ctx, at[0], 1, 64, at[1], at[2], 64, 16, None, 0.0, at[3], 1 << 31, None) == _lib.GQA_ERR_RANGE


def test_a_decode_step_of_all_operators():
    """Projection with 4-bit weights, norms with RoPE into a paged E4M3 cache, attention: two layers' caches, four steps,
    each operator checked on what the one before it gave; then the same steps from a captured graph, word for word."""
    rng = np.random.default_rng(7)
    B, hq, hkv, d, hidden, group, L, steps = 3, 8, 2, 64, 256, 64, 140, 4
    width = (hq + 2 * hkv) * d
    start = np.array([61, 0, 127], np.int32)
    kw = dict(batch=B, n_q_heads=hq, n_kv_heads=hkv, head_dim=d, max_seq_len=L, page_size=64, n_layers=2, kv_format="e4m3")
    hist = orc.bf16_rne(rng.standard_normal((2, 2, hkv, B, 127, d)).astype(np.float32))
    w_layers = []
    for _ in range(2):
        codes, scales = w4.quantize((rng.standard_normal((width, hidden)) * hidden**-0.5).astype(np.float32), group)
        w_layers.append((codes, scales, orc.bf16_rne((1 + 0.1 * rng.standard_normal(hidden)).astype(np.float32)),
                         *(orc.bf16_rne((1 + 0.1 * rng.standard_normal(d)).astype(np.float32)) for _ in range(2))))
    tokens = bf16_normal(rng, (steps, B, hidden))
    with AttentionAccelerator(**kw) as eager, AttentionAccelerator(**kw) as captured:
        engines = []
        for eng in (eager, captured):
            scatter_reserve(eng, [L] * B, 64)
            for layer in range(2):
                eng.select_layer(layer)
                for b in range(B):
                    if start[b]:
                        eng.load_kv(hist[layer, 0, :, b, :start[b]], hist[layer, 1, :, b, :start[b]], b=b)
            weights = [(*packed(eng, codes, scales, group), dev(g), dev(a), dev(k)) for codes, scales, g, a, k in w_layers]
            buf = dict(x=torch.zeros((B, hidden), dtype=torch.int16, device="cuda"), pos=dev(start),
                       lens=dev(start + 1),
                       **{f"{name}{layer}": torch.zeros((B, n), dtype=torch.int16, device="cuda")
                          for layer in range(2) for name, n in (("qkv", width), ("q", hq * d), ("o", hq * d))})
            engines.append((eng, weights, buf))

        def step(eng, weights, buf, stream):
            s = ctypes.c_void_p(stream) if stream else None
            for layer in range(2):
                eng.select_layer(layer)
                w, ws, g, a, k = weights[layer]
                qkv, q, o = (buf[f"{n}{layer}"] for n in ("qkv", "q", "o"))
                call("gqa_w4_project_device", eng._ctx, ptr(buf["x"]), B, hidden, ptr(w), ptr(ws), group, width, ptr(g), 1e-5,
                     ptr(qkv), width, s)
                call("gqa_qk_norm_rope_step_device", eng._ctx, ptr(qkv), width, ptr(a), ptr(k), 1e-6, ptr(buf["pos"]), None, 1e4,
                     ptr(q), s)
                call("gqa_decode_device", eng._ctx, ptr(q), ptr(buf["lens"]), ptr(o), None, s)

        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            step(*engines[1], torch.cuda.current_stream().cuda_stream)
        caches = [[[so.stored(f64(hist[layer, i, :, b, :start[b]])) for b in range(B)] for i in range(2)] for layer in range(2)]
        for t in range(steps):
            for _, _, buf in engines:
                buf["x"].copy_(dev(tokens[t]))
                buf["pos"].copy_(dev(start + t))
                buf["lens"].copy_(dev(start + t + 1))
            torch.cuda.synchronize()
            step(*engines[0], None)
            graph.replay()
            torch.cuda.synchronize()
            buf = engines[0][2]
            for name in buf:
                assert torch.equal(buf[name], engines[1][2][name]), (t, name)
            for layer in range(2):
                codes, scales, g, a, k = w_layers[layer]
                qkv, q, o = (words(buf[f"{n}{layer}"]) for n in ("qkv", "q", "o"))
                check(qkv, tokens[t], g, 1e-5, codes, scales)
                h = f64(qkv).reshape(B, -1, d)
                want, mag = so.norm_rope(h[:, :hq].transpose(1, 0, 2), f64(a), 1e-6, start + t, 1e4)
                got = f64(q).reshape(B, hq, d).transpose(1, 0, 2)
                assert np.all(np.abs(got - want) <= 2.0**-8 * np.abs(want) + 2.0**-19 * mag)
                eager.select_layer(layer)
                want_k, mag = so.norm_rope(h[:, hq:hq + hkv].transpose(1, 0, 2), f64(k), 1e-6, start + t, 1e4)
                for b in range(B):
                    kr, vr = (f64(r) for r in eager.read_kv(b, start[b] + t, 1))
                    _, scale = so.e4m3_row(want_k[:, b])
                    near = np.maximum(2.0**-4 * np.abs(want_k[:, b]), 2.0**-10 * scale[:, None]) + 2.0**-19 * mag[:, b]
                    assert np.all(np.abs(kr[:, 0] - want_k[:, b]) <= near)
                    assert np.array_equal(vr[:, 0], so.stored(h[b, hq + hkv:]))
                    for i, r in enumerate((kr, vr)):
                        caches[layer][i][b] = np.concatenate([caches[layer][i][b], r], 1)
                    ref, _, avg = so.decode(f64(q[b]).reshape(hq, d), caches[layer][0][b], caches[layer][1][b], eager.scale)
                    got_o = f64(o[b]).reshape(hq, d)
                    assert np.all(np.abs(got_o - ref) <= 2.0**-8 * np.abs(ref) + (2.0**-8 + 2.0**-13) * avg)


@pytest.mark.parametrize("rows,hidden,group", [((1 << 15) + 7, 1 << 16, 32), (1 << 19, 1 << 12, 128)])
def test_matrices_of_about_2_20_work_groups(acc, rows, hidden, group):
    """Packed and unpacked again: every value of the matrix, rounded once."""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    codes = torch.randint(0, 256, (rows, hidden // 2), dtype=torch.uint8, device="cuda", generator=gen)
    scales = (0.01 * torch.randn((rows, hidden // group), device="cuda", generator=gen)).bfloat16()
    wb, sb = w4.packed_bytes(rows, hidden, group)
    w, s = torch.empty(wb, dtype=torch.uint8, device="cuda"), torch.empty(sb, dtype=torch.uint8, device="cuda")
    out = torch.full((rows, hidden), float("nan"), dtype=torch.bfloat16, device="cuda")
    acc.w4_pack_device(codes.data_ptr(), scales.data_ptr(), rows, hidden, group, w.data_ptr(), s.data_ptr())
    acc.w4_unpack_device(w.data_ptr(), s.data_ptr(), rows, hidden, group, out.data_ptr())
    torch.cuda.synchronize()
    for at in range(0, rows, 4096):
        two = codes[at:at + 4096]
        c = torch.stack((two & 15, two >> 4), -1).view(two.shape[0], -1).float() - 8  # (8 codes times a bf16: exact in fp32)
        want = (c.view(two.shape[0], -1, group) * scales[at:at + 4096].float()[..., None]).view(two.shape[0], -1).bfloat16()
        assert torch.equal(out[at:at + 4096], want), at
