"""CPU tests of the microscaled 4-bit operators: the oracle against brute force
and the format's definition, and every refusal of the C-ABI and of its Python
binding, none of which needs a device."""
import ctypes as C

import numpy as np
import pytest

from oracle import mxfp4_oracle as mx


@pytest.fixture(scope="module")
def capi():
    import tt_capi

    return tt_capi


# ------------------------------------------------------------------ the oracle

def test_quantize_by_brute_force():
    """Each element against all sixteen codes; ties to the even code."""
    rng = np.random.default_rng(1)
    x = np.ldexp(rng.standard_normal((40, 64)), rng.integers(-20, 20, (40, 1)))
    x[0] = np.arange(64) * 0.125  # every tie of a block whose scale is one half or one
    codes, scales = mx.quantize(x)
    c = np.stack((codes & 15, codes >> 4), -1).reshape(40, 64)
    for r in range(40):
        for b in range(2):
            blk = x[r, 32 * b:32 * b + 32]
            s = 2.0 ** (np.floor(np.log2(np.abs(blk).max())) - 2)
            assert scales[r, b] == int(np.log2(s)) + 127
            for e, v in enumerate(blk):
                d = np.abs(mx.GRID - min(abs(v) / s, 6.0))
                near = np.flatnonzero(d == d.min())
                want = near[0] if len(near) == 1 else near[near % 2 == 0][0]
                assert c[r, 32 * b + e] == want + 8 * (v < 0)


def test_values_of_every_code_and_scale():
    codes = np.tile(np.arange(256, dtype=np.uint8).reshape(16, 16), (256, 1))
    scales = np.repeat(np.arange(256, dtype=np.uint8), 16)[:, None]
    v = mx.dequantize(codes, scales, 32)
    mag = [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    for i in (0, 17, 128 * 16 + 5, 254 * 16 + 15):
        for j in range(16):
            for h, c in enumerate((int(codes[i, j]) & 15, int(codes[i, j]) >> 4)):
                assert v[i, 2 * j + h] == (-1) ** (c >> 3) * mag[c & 7] * 2.0 ** (int(scales[i, 0]) - 127)
    assert np.isnan(v[255 * 16:]).all()


def test_quantize_edges():
    x = np.zeros((7, 33), np.float32)
    x[1, 3] = np.inf
    x[2, 32] = np.nan
    x[3] = -0.0
    x[4, 0] = 1e-45  # the smallest fp32: scale clamped at 2^-127
    x[5] = np.finfo(np.float32).max
    x[6, :32] = 7.9  # saturates: 7.9 / 1 is beyond 6
    codes, scales = mx.quantize(x)
    assert codes.shape == (7, 32) and scales.shape == (7, 2)
    assert list(scales[:, 0]) == [0, 255, 0, 0, 0, 252, 127] and list(scales[:, 1]) == [0, 0, 255, 0, 0, 252, 0]
    v = mx.dequantize(codes, scales, 33)
    assert np.isnan(v[1, :32]).all() and v[1, 32] == 0 and np.isnan(v[2, 32]) and np.signbit(v[3]).all()
    assert (v[6, :32] == 6).all() and v[4, 0] == 0 and np.allclose(v[5], 6 * 2.0 ** 125)
    # a block whose largest element is a code of at least 4 stays as it is
    y = mx.GRID[np.arange(32) % 8] * 2.0 ** -9
    assert np.array_equal(mx.dequantize(*mx.quantize(y), 32), y)


def test_append_and_decode_by_definition():
    rng = np.random.default_rng(3)
    kc, ks = mx.quantize(rng.standard_normal((3, 2, 9, 32)))
    new = rng.standard_normal((3, 2, 4, 32))
    codes, scales = mx.append(kc, ks, new, [9, 2, 0])
    assert np.array_equal(codes[0, :, :5], kc[0, :, :5]) and np.array_equal(codes[0, :, 5:], mx.quantize(new)[0][0])
    assert np.array_equal(codes[1, :, :2], mx.quantize(new)[0][1, :, 2:]) and np.array_equal(codes[1, :, 2:], kc[1, :, 2:])
    assert np.array_equal(codes[2], kc[2]) and np.array_equal(scales[2], ks[2])
    # one key: its value whatever the score; none: zeros and -inf
    v = rng.standard_normal((3, 2, 9, 32))
    o, lse, _, _ = mx.decode(rng.standard_normal((3, 4, 2, 32)), v, v, [2, 1, 0], 0.5)
    assert np.allclose(o[0, 3, 0], v[0, 1, 0]) and np.allclose(o[1, 1, 1], v[1, 0, 0])
    assert not o[1, :, 0].any() and np.isneginf(lse[1, :, 0]).all() and not o[2].any() and np.isneginf(lse[2]).all()


# ------------------------------------------------------------------ refusals

P = [C.c_void_p(0x1000 * (i + 1) * 4096) for i in range(10)]  # distinct addresses, never read


def test_quantize_refusals(capi):
    L = capi.lib()
    q, dq = L.lib.tt_mxfp4_quantize, L.lib.tt_mxfp4_dequantize
    F, H = capi.TT_F32, capi.TT_BF16
    assert q(capi.TT_F64, 0, P[0], P[1], P[2], 4, 32, None) == capi.TT_ERR_ARG and "dtype" in L.last_error()
    assert q(F, 2, P[0], P[1], P[2], 4, 32, None) == capi.TT_ERR_ARG and "trans" in L.last_error()
    assert q(F, 0, P[0], P[1], P[2], -1, 32, None) == capi.TT_ERR_ARG and "negative" in L.last_error()
    assert q(F, 0, P[0], P[1], P[2], 1, 1 << 31, None) == capi.TT_ERR_ARG and "2^31" in L.last_error()
    for i in range(3):
        a = [None if i == j else P[j] for j in range(3)]
        assert q(F, 0, *a, 4, 32, None) == capi.TT_ERR_ARG and "null pointer" in L.last_error()
        assert dq(F, *a, 4, 32, None) == capi.TT_ERR_ARG and "null pointer" in L.last_error()
    assert q(H, 0, P[0], C.c_void_p(P[1].value + 8), P[2], 4, 32, None) == capi.TT_ERR_ARG and "aligned" in L.last_error()
    assert q(H, 0, P[0], P[0], P[2], 4, 32, None) == capi.TT_ERR_ARG and "overlaps input x" in L.last_error()
    assert q(H, 1, P[0], P[1], C.c_void_p(P[1].value + 63), 4, 32, None) == capi.TT_ERR_ARG and "overlap" in L.last_error()
    assert dq(H, P[0], P[1], P[1], 4, 32, None) == capi.TT_ERR_ARG and "overlaps input scales" in L.last_error()
    for rows, cols in ((0, 32), (4, 0)):
        assert q(H, 0, None, None, None, rows, cols, None) == capi.TT_OK
        assert dq(H, None, None, None, rows, cols, None) == capi.TT_OK


def test_product_refusals(capi):
    L = capi.lib()
    g, fc = L.lib.tt_gemm_mxfp4, L.lib.tt_fc_forward_mxfp4
    F = capi.TT_F32
    assert g(capi.TT_I32, 4, 4, 32, 1.0, *P[:4], 0.0, P[4], None) == capi.TT_ERR_ARG and "dtype" in L.last_error()
    assert g(F, 4, -4, 32, 1.0, *P[:4], 0.0, P[4], None) == capi.TT_ERR_ARG
    assert g(F, 1 << 31, 4, 32, 1.0, *P[:4], 0.0, P[4], None) == capi.TT_ERR_ARG
    for i in range(5):
        a = [None if i == j else P[j] for j in range(5)]
        assert g(F, 4, 4, 32, 1.0, *a[:4], 0.0, a[4], None) == capi.TT_ERR_ARG and "null pointer" in L.last_error()
        assert fc(F, 4, 32, 4, *a[:4], 0, a[4], None) == capi.TT_ERR_ARG and "null pointer" in L.last_error()
    odd = C.c_void_p(P[2].value + 4)
    assert g(F, 4, 4, 32, 1.0, P[0], P[1], odd, P[3], 0.0, P[4], None) == capi.TT_ERR_ARG and "aligned" in L.last_error()
    assert fc(F, 4, 32, 4, P[0], odd, P[1], P[3], 0, P[4], None) == capi.TT_ERR_ARG and "aligned" in L.last_error()
    assert g(F, 4, 4, 32, 1.0, *P[:4], 0.0, P[1], None) == capi.TT_ERR_ARG and "overlaps input a_scales" in L.last_error()
    assert fc(F, 4, 32, 4, *P[:4], 0, P[0], None) == capi.TT_ERR_ARG and "overlaps input in" in L.last_error()
    assert g(F, 0, 4, 32, 1.0, None, None, None, None, 0.0, None, None) == capi.TT_OK
    assert fc(F, 4, 32, 0, None, None, None, None, 0, None, None) == capi.TT_OK


def test_cache_refusals(capi):
    L = capi.lib()
    ap, at = L.lib.tt_kv_append_mxfp4, L.lib.tt_attn_decode_mxfp4
    H = capi.TT_BF16

    def append(B=2, Hkv=2, T=1, cap=8, d=64, a=P[:7], dt=H):
        return ap(dt, *a, B, Hkv, T, cap, d, None)

    def attend(B=2, Hq=4, Hkv=2, T=1, cap=8, d=64, a=P[:8], dt=H):
        return at(dt, *a, B, Hq, Hkv, T, cap, d, 0.1, None)

    for f in (append, attend):
        assert f(dt=capi.TT_I32) == capi.TT_ERR_ARG and "dtype" in L.last_error()
        assert f(d=96) == capi.TT_ERR_UNSUPPORTED and "head dim" in L.last_error()
        assert f(B=-1) == capi.TT_ERR_ARG and f(T=-1) == capi.TT_ERR_ARG and f(cap=-1) == capi.TT_ERR_ARG
        assert f(cap=(1 << 30) + 1) == capi.TT_ERR_ARG and "too long" in L.last_error()
        assert f(B=1 << 25) == capi.TT_ERR_ARG and "too many" in L.last_error()
    for i in range(7):
        assert append(a=[None if i == j else P[j] for j in range(7)]) == capi.TT_ERR_ARG
        assert "null pointer" in L.last_error()
        assert attend(a=[None if i == j else P[j] for j in range(8)]) == capi.TT_ERR_ARG
        assert "null pointer" in L.last_error()
    for i in (2, 4):
        a = list(P[:7])
        a[i] = C.c_void_p(P[i].value + 2)
        assert append(a=a) == capi.TT_ERR_ARG and "aligned" in L.last_error()
        a = list(P[:8])
        a[i - 1] = C.c_void_p(P[i].value + 2)
        assert attend(a=a) == capi.TT_ERR_ARG and "aligned" in L.last_error()
    a = list(P[:7])
    a[4] = a[2]
    assert append(a=a) == capi.TT_ERR_ARG and "overlap" in L.last_error()
    a = list(P[:8])
    a[6] = a[0]
    assert attend(a=a) == capi.TT_ERR_ARG and "overlaps input q" in L.last_error()
    assert attend(Hq=3) == capi.TT_ERR_ARG and "multiple" in L.last_error()
    assert attend(Hkv=0) == capi.TT_ERR_ARG and "multiple" in L.last_error()
    assert append(B=0, a=[None] * 7) == capi.TT_OK and append(cap=0, a=[None] * 7) == capi.TT_OK
    assert attend(B=0, a=[None] * 8) == capi.TT_OK and attend(T=0, a=[None] * 8) == capi.TT_OK
    assert attend(Hq=0, Hkv=0, a=[None] * 8) == capi.TT_OK


class Fake:
    """What the binding reads of a buffer, without a device."""

    def __init__(self, shape, dtype):
        self.shape, self.dtype, self.ptr = tuple(shape), dtype, None
        self.nbytes = int(np.prod(shape)) * {"f32": 4, "bf16": 2, "i32": 4, "u8": 1}[dtype]


def test_binding_refusals(capi):
    x, c, s = Fake((4, 33), "f32"), Fake((4, 32), "u8"), Fake((4, 2), "u8")
    for bad in ((Fake((4, 33), "i32"), c, s), (x, Fake((4, 17), "u8"), s), (x, c, Fake((4, 1), "u8")),
                (x, Fake((4, 8), "f32"), s)):
        with pytest.raises(ValueError):
            capi.mxfp4_quantize(*bad)
        with pytest.raises(ValueError):
            capi.mxfp4_dequantize(bad[1], bad[2], bad[0])
    with pytest.raises(ValueError):
        capi.mxfp4_quantize(x, c, s, trans=True)
    with pytest.raises(ValueError):
        capi.gemm_mxfp4(33, 1.0, c, s, c, s, 0.0, Fake((4, 5), "f32"))
    with pytest.raises(ValueError):
        capi.fc_forward_mxfp4(x, c, s, Fake((4,), "bf16"), Fake((4, 4), "f32"))
    with pytest.raises(ValueError):
        capi.fc_forward_mxfp4(x, c, s, Fake((3,), "f32"), Fake((4, 4), "f32"))
    kc, ks = Fake((2, 2, 8, 32), "u8"), Fake((2, 2, 8, 2), "u8")
    k, n = Fake((2, 2, 3, 64), "bf16"), Fake((2,), "i32")
    for bad in ((k, k, kc, ks, kc, ks, Fake((3,), "i32")), (k, k, kc, ks, kc, ks, Fake((2,), "f32")),
                (k, Fake((2, 2, 2, 64), "bf16"), kc, ks, kc, ks, n), (k, Fake((2, 2, 3, 64), "f32"), kc, ks, kc, ks, n),
                (k, k, kc, ks, kc, kc, n)):
        with pytest.raises(ValueError):
            capi.kv_append_mxfp4(*bad)
    q = Fake((2, 4, 3, 64), "bf16")
    for bad in ((q, kc, ks, kc, ks, n, k, None), (q, kc, ks, kc, ks, n, q, Fake((2, 4), "f32")),
                (q, kc, ks, kc, ks, n, Fake(q.shape, "f32"), None)):
        with pytest.raises(ValueError):
            capi.attn_decode_mxfp4(*bad, 0.1)


def test_attention_size_refusals(capi):
    """B H T below 2^31, and below 2^24 tiles of 16 rows that share a K / V head."""
    L = capi.lib()

    def attend(B, H, Hkv, T):
        return L.lib.tt_attn_decode_mxfp4(capi.TT_BF16, *P[:8], B, H, Hkv, T, 8, 32, 0.1, None)

    assert attend(1, 2, 1, 1 << 30) == capi.TT_ERR_ARG and "too many rows" in L.last_error()
    assert attend(1 << 24, 1, 1, 1) == capi.TT_ERR_ARG and "grid too large" in L.last_error()
    assert attend(1 << 22, 4, 4, 1) == capi.TT_ERR_ARG and "grid too large" in L.last_error()
    assert attend(1 << 23, 1, 1, 17) == capi.TT_ERR_ARG and "grid too large" in L.last_error()
    a = [None] + P[1:8]
    for B, H, Hkv, T in (((1 << 24) - 1, 1, 1, 1), (1 << 22, 4, 1, 4), (1, 1, 1, (1 << 28) - 16), (1 << 9, 1 << 9, 1, 1023)):
        assert L.lib.tt_attn_decode_mxfp4(capi.TT_BF16, *a, B, H, Hkv, T, 8, 32, 0.1, None) == capi.TT_ERR_ARG
        assert "null pointer" in L.last_error()  # the sizes are taken


def test_transposed_size_refusals(capi):
    """Fewer than 2^24 pieces of 64 rows by 128 columns; no such limit for rows as they are stored."""
    L, F = capi.lib(), capi.TT_F32
    q = L.lib.tt_mxfp4_quantize
    overlap = (P[0], P[0], P[1])  # refused once the sizes are taken
    for rows, cols in ((1, (1 << 31) - 1), (1 << 20, 1 << 17)):
        assert q(F, 1, *overlap, rows, cols, None) == capi.TT_ERR_ARG and "too large" in L.last_error()
        assert q(F, 0, *overlap, rows, cols, None) == capi.TT_ERR_ARG and "overlap" in L.last_error()
    for rows, cols in ((1, (1 << 31) - 128), ((1 << 20) - 64, 1 << 17)):
        assert q(F, 1, *overlap, rows, cols, None) == capi.TT_ERR_ARG and "overlap" in L.last_error()
