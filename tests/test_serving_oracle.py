"""The serving oracle against hand-derived values, torch's E4M3 type and brute force; the host quantiser of 4-bit weights;
refusals that need no device."""
import ctypes

import numpy as np
import pytest

from lara_amd import _lib, w4
from lara_amd.attn_driver import AttentionAccelerator
from oracle import gqa_oracle as orc
from oracle import serving_oracle as so


def test_e4m3_codes_are_torchs():
    torch = pytest.importorskip("torch")
    ref = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(so.e4m3_values(), ref, equal_nan=True)


def test_e4m3_row_known_answers():
    # 448 is held at scale 1, anything above takes the next power of two
    assert so.e4m3_row(np.array([448.0, 1.0]))[1] == 1.0
    assert so.e4m3_row(np.array([448.5, 1.0]))[1] == 2.0
    assert so.e4m3_row(np.array([224.0, 1.0]))[1] == 0.5
    # ties to even, subnormals of the type, NaN and infinities, zeros, the top
    v, s = so.e4m3_row(np.array([256.0 + 16, 256.0 + 48, 2.0**-10, 3 * 2.0**-10, np.nan, -np.inf, 448.0]))
    assert s == 1.0 and np.array_equal(v, [256.0, 320.0, 0.0, 2 * 2.0**-9, np.nan, np.nan, 448.0], equal_nan=True)
    v, s = so.e4m3_row(np.zeros(4))
    assert s == 2.0**-126 and not v.any()
    big = float(orc.bf16_u16_to_fp32(np.uint16(0x7F7F)))
    assert so.stored(np.array([big, -big]))[0] == so.TOP


def test_e4m3_row_is_the_nearest_code():
    rng = np.random.default_rng(3)
    table = so.e4m3_values()
    table = np.sort(table[np.isfinite(table)])
    x = rng.standard_normal((200, 16)) * np.exp(4 * rng.standard_normal((200, 1)))
    v, s = so.e4m3_row(x)
    for row, got, scale in zip(x, v, s):
        assert 448 * scale >= np.abs(row).max() > 224 * scale
        want = np.abs(row[:, None] / scale - table).min(-1)
        assert np.array_equal(np.abs(got - row / scale), want)


def test_decode_against_loops():
    rng = np.random.default_rng(4)
    q, k, v = rng.standard_normal((6, 8)), rng.standard_normal((2, 5, 8)), rng.standard_normal((2, 5, 8))
    o, lse, a = so.decode(q, k, v, 0.3)
    for h in range(6):
        w = [np.exp(0.3 * sum(q[h, d] * k[h // 3, t, d] for d in range(8))) for t in range(5)]
        for d in range(8):
            assert o[h, d] == pytest.approx(sum(w[t] * v[h // 3, t, d] for t in range(5)) / sum(w), rel=1e-12)
            assert a[h, d] == pytest.approx(sum(w[t] * abs(v[h // 3, t, d]) for t in range(5)) / sum(w), rel=1e-12)
        assert lse[h] == pytest.approx(np.log(sum(w)), rel=1e-12)
    o, lse, _ = so.decode(q, k[:, :0], v[:, :0], 0.3)
    assert not o.any() and np.all(lse == -np.inf)


def test_norm_rope_against_loops():
    rng = np.random.default_rng(5)
    h, w = rng.standard_normal((3, 8)), rng.standard_normal(8)
    y, mag = so.norm_rope(h, w, 1e-3, [0, 7, 1000], 10000.0)
    for t, pos in enumerate((0, 7, 1000)):
        n = [h[t, d] / (sum(h[t] ** 2) / 8 + 1e-3) ** 0.5 * w[d] for d in range(8)]
        for p in range(4):
            angle = pos * 10000.0 ** (-2 * p / 8)
            assert y[t, 2 * p] == pytest.approx(n[2 * p] * np.cos(angle) - n[2 * p + 1] * np.sin(angle), abs=1e-12)
            assert y[t, 2 * p + 1] == pytest.approx(n[2 * p] * np.sin(angle) + n[2 * p + 1] * np.cos(angle), abs=1e-12)
    assert np.all(mag >= np.abs(y) - 1e-12)
    assert np.array_equal(so.norm_rope(h, None, 0.0, [1, 2, 3], 0)[0], h)


@pytest.mark.parametrize("group", w4.GROUPS)
def test_w4_quantiser(group):
    rng = np.random.default_rng(group)
    w = rng.standard_normal((5, 256)).astype(np.float32)
    w[1, :group] = 0
    codes, scales = w4.quantize(w, group)
    assert codes.shape == (5, 128) and scales.shape == (5, 256 // group)
    s = orc.bf16_u16_to_fp32(scales).astype(np.float64)
    back = so.w4_matrix(codes, s)
    # the nearest code; the value of the group's largest magnitude takes -8, values of the other sign reach 7 at most
    err = np.abs(back - w).reshape(5, -1, group)
    assert np.all(err <= np.abs(s)[..., None] * 1.07)
    inside = np.abs(w.reshape(5, -1, group)) <= 7 * np.abs(s)[..., None]
    assert np.all(err[inside] <= (np.broadcast_to(np.abs(s)[..., None], err.shape) * 0.5 * (1 + 1e-12))[inside])
    assert not back[1, :group].any()
    with pytest.raises(ValueError):
        w4.quantize(w[:, :200], 128)
    with pytest.raises(ValueError):
        w4.quantize(np.full((1, 128), np.nan), 128)


def test_w4_sizes_and_refusals():
    assert w4.packed_bytes(16, 128, 128) == (1024, 32)
    assert w4.packed_bytes(17, 160, 32) == (2 * 2 * 1024, 2 * 8 * 32)  # padded to whole tiles
    lib, a, b = _lib.lib(), ctypes.c_int64(), ctypes.c_int64()
    for rows, hidden, group, code in ((16, 128, 48, _lib.GQA_ERR_UNSUPPORTED), (0, 128, 32, _lib.GQA_ERR_RANGE),
                                      (16, 144, 32, _lib.GQA_ERR_RANGE), (16, 0, 32, _lib.GQA_ERR_RANGE),
                                      ((1 << 20) + 1, 128, 32, _lib.GQA_ERR_RANGE), (16, (1 << 16) + 128, 32, _lib.GQA_ERR_RANGE)):
        assert lib.gqa_w4_bytes(rows, hidden, group, ctypes.byref(a), ctypes.byref(b)) == code
    assert lib.gqa_w4_bytes(16, 128, 32, None, ctypes.byref(b)) == _lib.GQA_ERR_NULL


def _cfg(**kw):
    base = dict(batch=1, n_q_heads=32, n_kv_heads=8, head_dim=128, max_seq_len=512, max_q_len=512, scale=0.0, device=0)
    base.update(kw)
    return _lib.GqaConfig(**base)


def test_create_kv8_refusals_before_a_device():
    lib, ctx = _lib.lib(), ctypes.c_void_p()

    def create(page, pages, layers, **kw):
        return lib.gqa_create_kv8(ctypes.byref(_cfg(**kw)), page, pages, layers, ctypes.byref(ctx))

    assert lib.gqa_create_kv8(None, 0, 0, 1, ctypes.byref(ctx)) == _lib.GQA_ERR_NULL
    for page, pages, layers in ((0, 8, 1), (0, 0, 2), (0, 0, 0), (48, 8, 1), (32, 8, 1), (64, 0, 1), (64, 8, 0),
                                (64, 8, _lib.GQA_MAX_LAYERS + 1), (-64, 8, 1), (1 << 17, 8, 1)):
        assert create(page, pages, layers) == _lib.GQA_ERR_BAD_CFG
    assert create(0, 0, 1, head_dim=96) == _lib.GQA_ERR_UNSUPPORTED
    assert create(0, 0, 1, n_q_heads=34, n_kv_heads=2) == _lib.GQA_ERR_UNSUPPORTED  # 17 heads a group
    assert create(0, 0, 1, n_q_heads=30) == _lib.GQA_ERR_BAD_CFG
    assert not ctx.value
    with pytest.raises(ValueError):
        AttentionAccelerator(kv_format="int8")


def test_null_arguments_are_refused():
    lib, n = _lib.lib(), _lib.GQA_ERR_NULL
    assert lib.gqa_kv8_scales(None, None, None) == n
    assert lib.gqa_read_kv_device(None, 0, 0, 1, None, None, None) == n
    assert lib.gqa_qk_norm_rope_device(None, 0, None, 0, 1, None, None, 0.0, 0, 0, 0, 0.0, None, None) == n
    assert lib.gqa_qk_norm_rope_step_device(None, None, 0, None, None, 0.0, None, None, 0.0, None, None) == n
    assert lib.gqa_w4_pack_device(None, None, None, 16, 128, 32, None, None, None) == n
    assert lib.gqa_w4_unpack_device(None, None, None, 16, 128, 32, None, None) == n
    assert lib.gqa_w4_project_device(None, None, 1, 128, None, None, 32, 16, None, 0.0, None, 16, None) == n
