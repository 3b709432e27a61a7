"""GPU tests of the microscaled 4-bit operators against the oracle.

Tolerances.  Quantising is exact but for the rounding that defines it, so codes
and scales are compared bit for bit, also those of a cache after an append.
Products: the product of two elements is exact in fp32, so a sum of k of them is
off by at most k 2^-24 of the sum of magnitudes, and a bf16 store by 2^-8 of the
value.  Attention: with e the error of a score (below) the weights are off by
a factor e^(+-2 e); the weights' bf16 terms cost 2^-16 (two) or 2^-24 (three),
exp2 and the sums over n keys (n + 4) 2^-24 each, so o is off by at most
(2 e + t + 2 (n + 4) 2^-24) sum p |v| and the store's rounding, and lse by
e + (n + 4) 2^-24 + 2^-22 |lse|.  A score, a sum of d exact products times a
scale that was rounded twice, is off by e = (d + 4) 2^-24 sum |q| |k| scale."""
import numpy as np
import pytest

from oracle import attn_oracle as orc
from oracle import mxfp4_oracle as mx

pytestmark = pytest.mark.gpu
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}
U = 2.0 ** -24


@pytest.fixture(scope="module")
def capi():
    import tt_capi

    assert tt_capi.lib().device_count() >= 1, "no HIP device visible"
    tt_capi.lib().call("tt_init", 0)
    return tt_capi


def normal(rng, shape, dtype, std=1.0):
    x = (rng.standard_normal(shape) * std).astype(np.float32)
    return orc.bf16_round(x) if dtype == "bf16" else x


def quantized(capi, x, dtype, trans=False):
    rows = x.shape if not trans else x.shape[::-1]
    codes, scales = capi.mxfp4_buffers(rows)
    capi.mxfp4_quantize(capi.DeviceBuffer.from_numpy(x, dtype), codes, scales, trans)
    capi.lib().sync()
    return codes, scales


def held(capi, x):
    """x in 4 bits on the device, quantised by the oracle."""
    c, s = mx.quantize(x)
    return capi.DeviceBuffer.from_numpy(c, "u8"), capi.DeviceBuffer.from_numpy(s, "u8")


# ------------------------------------------------------------------ quantise, read back

SHAPES = [(1, 1), (1, 31), (1, 32), (3, 33), (5, 64), (7, 100), (64, 96), (65, 129), (130, 4096), (1000, 40), (2, 70000)]


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize_and_read_back(capi, rows, cols, dtype, trans):
    rng = np.random.default_rng(rows * 131 + cols)
    x = normal(rng, (rows, cols), dtype) * np.ldexp(1.0, rng.integers(-30, 30, (rows, 1))).astype(np.float32)
    x[rng.random(x.shape) < 0.05] = 0.0
    codes, scales = quantized(capi, np.ascontiguousarray(x.T) if trans else x, dtype, trans)
    rc, rs = mx.quantize(x)
    assert np.array_equal(scales.download(), rs)
    assert np.array_equal(codes.download(), rc)
    for out in ("f32", "bf16"):
        y = capi.DeviceBuffer((rows, cols), out)
        capi.mxfp4_dequantize(codes, scales, y)
        capi.lib().sync()
        assert np.array_equal(y.download().astype(np.float64), mx.dequantize(rc, rs, cols)), out


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quantize_ties_and_extremes(capi, dtype, trans):
    """Every tie, both signs, zeros, subnormals, the largest values, infinities and NaN."""
    ties = np.array([0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 4, 6, 7, 7.75], np.float32)
    near = np.concatenate((ties * (1 + 2.0 ** -7), ties * (1 - 2.0 ** -7))) if dtype == "bf16" else \
        np.concatenate((np.nextafter(ties, 9), np.nextafter(ties, -9)))
    blk = np.concatenate((ties, -ties, near))[:36]
    x = np.zeros((24, 64), np.float32)
    for i in range(12):
        x[i, :36] = orc.bf16_round(np.ldexp(blk, 10 * i - 60).astype(np.float32)) if dtype == "bf16" else np.ldexp(blk, 10 * i - 60)
        x[i, 31] = np.ldexp(4.0, 10 * i - 60)  # the scale's element
        x[i, 63] = -np.ldexp(7.0, 10 * i - 60)
    top = np.float32(3.3895314e38) if dtype == "bf16" else np.finfo(np.float32).max
    x[12, 5], x[13, 40], x[14, 0], x[15, 63], x[16, 7] = np.inf, -np.inf, np.nan, np.nan, top
    x[17] = -0.0
    x[18, 3], x[18, 34] = 2.0 ** -126, -(2.0 ** -127)
    x[19] = 2.0 ** -128 * np.arange(64)
    x[20, 0], x[20, 33] = 2.0 ** -133, -(2.0 ** -133)
    x[21] = top
    x[22] = -(2.0 ** -125) * (np.arange(64) % 8)
    x[23, :32] = 1.0
    assert dtype == "f32" or np.array_equal(orc.bf16_round(x), x, equal_nan=True)
    codes, scales = quantized(capi, np.ascontiguousarray(x.T) if trans else x, dtype, trans)
    rc, rs = mx.quantize(x)
    assert np.array_equal(scales.download(), rs)
    assert np.array_equal(codes.download(), rc)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_every_code_and_scale_reads_back(capi, dtype):
    codes = np.tile(np.arange(256, dtype=np.uint8).reshape(16, 16), (256, 1))
    scales = np.repeat(np.arange(256, dtype=np.uint8), 16)[:, None].copy()
    y = capi.DeviceBuffer((4096, 32), dtype)
    capi.mxfp4_dequantize(capi.DeviceBuffer.from_numpy(codes, "u8"), capi.DeviceBuffer.from_numpy(scales, "u8"), y)
    capi.lib().sync()
    with np.errstate(over="ignore"):
        want = mx.dequantize(codes, scales, 32).astype(np.float32)
    assert np.array_equal(y.download(), want, equal_nan=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(9, 64), (9, 61)])
def test_rows_at_any_element_alignment(capi, dtype, rows, cols):
    """x and y one element into a buffer; what lies around y stays."""
    x = normal(np.random.default_rng(4), (rows * cols + 2,), dtype)
    buf, e = capi.DeviceBuffer.from_numpy(x, dtype), capi.DeviceBuffer.ITEM[dtype]
    codes, scales = capi.mxfp4_buffers((rows, cols))
    code = capi.TT_BF16 if dtype == "bf16" else capi.TT_F32
    L = capi.lib()
    L.call("tt_mxfp4_quantize", code, 0, buf.ptr + e, codes.ptr, scales.ptr, rows, cols, None)
    rc, rs = mx.quantize(x[1:-1].reshape(rows, cols))
    L.sync()
    assert np.array_equal(codes.download(), rc) and np.array_equal(scales.download(), rs)
    y = capi.DeviceBuffer.from_numpy(np.full(rows * cols + 2, 77.0, np.float32), dtype)
    L.call("tt_mxfp4_dequantize", code, codes.ptr, scales.ptr, y.ptr + e, rows, cols, None)
    L.sync()
    got = y.download()
    assert got[0] == got[-1] == 77.0
    assert np.array_equal(got[1:-1].astype(np.float64), mx.dequantize(rc, rs, cols).ravel())


# ------------------------------------------------------------------ product

GEMM_SHAPES = [(1, 16, 32), (1, 4096, 4096), (3, 17, 33), (16, 100, 784), (17, 64, 96), (64, 64, 128), (65, 63, 160),
               (128, 128, 256), (129, 130, 288), (200, 513, 1000), (256, 256, 512), (300, 300, 1056), (512, 384, 4128),
               (700, 1025, 2049), (2049, 260, 544), (31, 5000, 31), (1024, 1024, 31), (257, 2000, 8224)]


def product_bound(av, bv, k, dtype, ref, alpha=1.0, extra=0.0):
    with np.errstate(invalid="ignore"):
        mag = np.abs(alpha) * (np.abs(av) @ np.abs(bv).T) + extra
    return (k + 4) * U * mag + HALF[dtype] * np.abs(ref) + 1e-37


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", GEMM_SHAPES)
def test_gemm(capi, m, n, k, dtype):
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    a, b = rng.standard_normal((m, k)), rng.standard_normal((n, k)) * np.ldexp(1.0, rng.integers(-6, 6, (n, 1)))
    (ac, as_), (bc, bs) = held(capi, a), held(capi, b)
    av, bv = mx.dequantize(*mx.quantize(a), k), mx.dequantize(*mx.quantize(b), k)
    c = capi.DeviceBuffer.from_numpy(np.full((m, n), np.nan, np.float32), dtype)  # beta = 0 does not read it
    capi.gemm_mxfp4(k, 1.0, ac, as_, bc, bs, 0.0, c)
    capi.lib().sync()
    ref = av @ bv.T
    assert (np.abs(c.download() - ref) <= product_bound(av, bv, k, dtype, ref)).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(5, 40, 70), (300, 270, 600)])
def test_gemm_alpha_beta(capi, m, n, k, dtype):
    rng = np.random.default_rng(9)
    a, b, c0 = rng.standard_normal((m, k)), rng.standard_normal((n, k)), normal(rng, (m, n), dtype)
    (ac, as_), (bc, bs) = held(capi, a), held(capi, b)
    av, bv = mx.dequantize(*mx.quantize(a), k), mx.dequantize(*mx.quantize(b), k)
    c = capi.DeviceBuffer.from_numpy(c0, dtype)
    capi.gemm_mxfp4(k, -0.75, ac, as_, bc, bs, 0.5, c)
    capi.lib().sync()
    ref = -0.75 * (av @ bv.T) + 0.5 * c0
    assert (np.abs(c.download() - ref) <= product_bound(av, bv, k, dtype, ref, 0.75, np.abs(c0))).all()


def test_gemm_of_no_k_is_beta_c(capi):
    c = capi.DeviceBuffer.from_numpy(np.arange(12, dtype=np.float32).reshape(3, 4))
    capi.lib().call("tt_gemm_mxfp4", capi.TT_F32, 3, 4, 0, 1.0, None, None, None, None, 0.5, c.ptr, None)
    capi.lib().sync()
    assert np.array_equal(c.download(), np.arange(12).reshape(3, 4) * 0.5)


@pytest.mark.parametrize("m,n,k", [(4, 20, 200), (300, 270, 1100)])
def test_gemm_nan_blocks_reach_their_rows_alone(capi, m, n, k):
    """Also where the last block is padded, and beside rows past the end of a tile."""
    rng = np.random.default_rng(10)
    a, b = rng.standard_normal((m, k)), rng.standard_normal((n, k))
    a[m - 1, k - 1], b[2, 5] = np.nan, np.inf
    (ac, as_), (bc, bs) = held(capi, a), held(capi, b)
    c = capi.DeviceBuffer((m, n), "f32")
    capi.gemm_mxfp4(k, 1.0, ac, as_, bc, bs, 0.0, c)
    capi.lib().sync()
    got = np.isnan(c.download())
    want = np.zeros((m, n), bool)
    want[m - 1], want[:, 2] = True, True
    assert np.array_equal(got, want)


def test_gemm_extreme_scales(capi):
    """Scale bytes from 0 to 254 that cancel, and codes of zero under any scale."""
    k, m, n = 96, 20, 40
    rng = np.random.default_rng(11)
    ac, bc = (rng.integers(0, 256, (r, 48)).astype(np.uint8) for r in (m, n))
    as_, bs = rng.integers(0, 30, (m, 3)).astype(np.uint8), rng.integers(225, 255, (n, 3)).astype(np.uint8)
    ac[3], as_[3] = 0, 254
    c = capi.DeviceBuffer((m, n), "f32")
    dev = [capi.DeviceBuffer.from_numpy(x, "u8") for x in (ac, as_, bc, bs)]
    capi.gemm_mxfp4(k, 1.0, *dev, 0.0, c)
    capi.lib().sync()
    av, bv = mx.dequantize(ac, as_, k), mx.dequantize(bc, bs, k)
    ref = av @ bv.T
    assert (np.abs(c.download() - ref) <= product_bound(av, bv, k, "f32", ref)).all()


# ------------------------------------------------------------------ fully connected layer

@pytest.mark.parametrize("scalar_bias", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(1, 100, 784), (1, 4096, 4096), (7, 33, 65), (16, 40, 31), (17, 40, 31), (100, 1000, 96),
                                   (256, 100, 784), (300, 520, 1000)])
def test_fc(capi, m, n, k, dtype, scalar_bias):
    rng = np.random.default_rng(m + n + k)
    x, w, bias = normal(rng, (m, k), dtype), rng.standard_normal((n, k)), normal(rng, (1 if scalar_bias else n,), dtype)
    wc, ws = held(capi, w)
    out = capi.DeviceBuffer((m, n), dtype)
    capi.fc_forward_mxfp4(capi.DeviceBuffer.from_numpy(x, dtype), wc, ws, capi.DeviceBuffer.from_numpy(bias, dtype), out)
    capi.lib().sync()
    xv, wv = mx.dequantize(*mx.quantize(x), k), mx.dequantize(*mx.quantize(w), k)
    ref = xv @ wv.T + bias
    assert (np.abs(out.download() - ref) <= product_bound(xv, wv, k, dtype, ref, 1.0, np.abs(bias))).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(1, 50, 4096), (1, 50, 8200), (4, 50, 4100), (5, 50, 4100), (16, 50, 2048), (16, 50, 2049),
                                   (17, 8200, 40), (530, 240, 100), (600, 240, 100)])
def test_fc_on_both_sides_of_its_rule(capi, m, n, k, dtype):
    """Rows of 4, 8 and 16 KiB, 32 KiB of them, and 512 blocks of 16 x 16, from both sides."""
    rng = np.random.default_rng(m + n + k)
    x, w, b = normal(rng, (m, k), dtype), normal(rng, (n, k), "f32"), normal(rng, (n,), dtype)
    wc, ws = held(capi, w)
    out = capi.DeviceBuffer((m, n), dtype)
    capi.fc_forward_mxfp4(capi.DeviceBuffer.from_numpy(x, dtype), wc, ws, capi.DeviceBuffer.from_numpy(b, dtype), out)
    capi.lib().sync()
    xv, wv = mx.dequantize(*mx.quantize(x), k), mx.dequantize(*mx.quantize(w), k)
    ref = xv @ wv.T + b
    tol = (k + 1) * U * (np.abs(xv) @ np.abs(wv.T) + np.abs(b))
    assert (np.abs(out.download() - ref) <= tol * (1 + HALF[dtype]) + HALF[dtype] * np.abs(ref)).all()


def test_fc_of_no_input_is_the_bias(capi):
    bias = capi.DeviceBuffer.from_numpy(np.arange(5, dtype=np.float32))
    out = capi.DeviceBuffer((40, 5), "f32")
    capi.lib().call("tt_fc_forward_mxfp4", capi.TT_F32, 40, 0, 5, None, None, None, bias.ptr, 0, out.ptr, None)
    capi.lib().sync()
    assert np.array_equal(out.download(), np.tile(np.arange(5), (40, 1)))


def test_fc_in_several_pieces_of_rows(capi):
    """More rows than the workspace holds quantised: 32 MiB / (17 * 2048 bytes) = 963."""
    m, n, k = 2000, 48, 65536
    rng = np.random.default_rng(12)
    x, w = normal(rng, (m, 64), "bf16"), rng.standard_normal((n, k))
    x = np.tile(x, (1, k // 64))
    wc, ws = held(capi, w)
    out, bias = capi.DeviceBuffer((m, n), "f32"), capi.DeviceBuffer.from_numpy(np.zeros(n, np.float32))
    capi.fc_forward_mxfp4(capi.DeviceBuffer.from_numpy(x), wc, ws, bias, out)
    capi.lib().sync()
    xv, wv = mx.dequantize(*mx.quantize(x[:, :64]), 64), mx.dequantize(*mx.quantize(w), k)
    ref = xv @ wv.reshape(n, -1, 64).sum(1).T
    mag = np.abs(xv) @ np.abs(wv).reshape(n, -1, 64).sum(1).T
    assert (np.abs(out.download() - ref) <= (k + 4) * U * mag).all()


# ------------------------------------------------------------------ cache

class Cache:
    """A quantised cache on the device with random rows, and its values."""

    def __init__(self, capi, rng, B, Hkv, cap, d, lengths, std=1.0):
        self.capi, self.shape = capi, (B, Hkv, cap, d)
        self.kc, self.ks = mx.quantize(rng.standard_normal(self.shape) * std)
        self.vc, self.vs = mx.quantize(rng.standard_normal(self.shape) * np.ldexp(1.0, rng.integers(-3, 3, (B, Hkv, cap, 1))))
        self.lengths = np.array(lengths, np.int32)

    def upload(self):
        f = self.capi.DeviceBuffer.from_numpy
        self.dev = [f(x, "u8") for x in (self.kc, self.ks, self.vc, self.vs)]
        self.len = f(self.lengths, "i32")
        return self

    def values(self):
        d = self.shape[3]
        return mx.dequantize(self.kc, self.ks, d), mx.dequantize(self.vc, self.vs, d)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("B,Hkv,T,cap,lengths", [
    (1, 1, 1, 1, [1]), (3, 2, 1, 40, [40, 0, 17]), (4, 3, 5, 33, [33, 5, 3, 0]), (2, 1, 7, 4, [9, 2]),
    (3, 2, 4, 20, [23, -1, 30]), (2, 4, 100, 128, [128, 61]), (1, 2, 3, 1 << 12, [4096])])
def test_append(capi, B, Hkv, T, cap, lengths, d, dtype):
    """Padded prompts, idle slots, tokens that do not fit: every other row as it was."""
    rng = np.random.default_rng(B * T + cap + d)
    c = Cache(capi, rng, B, Hkv, cap, d, lengths).upload()
    k, v = (normal(rng, (B, Hkv, T, d), dtype) for _ in range(2))
    k[0, 0, 0, 3] = np.nan
    f = capi.DeviceBuffer.from_numpy
    capi.kv_append_mxfp4(f(k, dtype), f(v, dtype), *c.dev, c.len)
    capi.lib().sync()
    for got, (codes, scales), new in ((c.dev[:2], (c.kc, c.ks), k), (c.dev[2:], (c.vc, c.vs), v)):
        rc, rs = mx.append(codes, scales, new, lengths)
        assert np.array_equal(got[0].download(), rc) and np.array_equal(got[1].download(), rs)


def attend(capi, c, q, dtype, scale, lse=True, stream=None):
    o = capi.DeviceBuffer.from_numpy(np.full(q.shape, 77.0, np.float32), dtype)
    l = capi.DeviceBuffer.from_numpy(np.full(q.shape[:3], 77.0, np.float32)) if lse else None
    capi.attn_decode_mxfp4(capi.DeviceBuffer.from_numpy(q, dtype), *c.dev, c.len, o, l, scale, stream)
    capi.lib().call("tt_stream_sync", stream)
    return o.download(), l.download() if lse else None


def check_attention(c, q, dtype, scale, o, lse):
    k, v = c.values()
    d = q.shape[3]
    ro, rl, mag, smax = mx.decode(q, k, v, c.lengths, scale)
    n = c.shape[2]
    e = (d + 4) * U * smax
    terms = U if dtype == "f32" else 2.0 ** -16
    assert (np.abs(o - ro) <= (2 * e + terms + 2 * (n + 4) * U)[..., None] * mag + HALF[dtype] * np.abs(ro)).all()
    if lse is not None:
        empty = np.isneginf(rl)
        assert np.array_equal(np.isneginf(lse), empty)
        f = ~empty
        assert (np.abs(lse[f] - rl[f]) <= e[f] + (n + 4) * U + 4 * U * np.abs(rl[f])).all()


SHAPES_ATT = [  # B, H, Hkv, T, cap, lengths
    (1, 1, 1, 1, 1, [1]),
    (2, 4, 4, 1, 31, [31, 1]),
    (3, 4, 2, 1, 300, [300, 0, 129]),
    (4, 8, 2, 3, 257, [257, 2, 0, 100]),
    (2, 5, 1, 7, 70, [70, 3]),  # 35 rows: three tiles, rows without a key
    (1, 17, 1, 1, 500, [499]),
    (2, 2, 2, 40, 64, [64, 20]),  # a prompt's tokens
    (1, 2, 1, 33, 33, [33]),
    (2, 2, 1, 2, 50, [60, -3]),  # longer than the cache; a negative length
    (1, 4, 4, 1, 5000, [4999]),  # several splits
    (64, 16, 16, 1, 40, [(7 * b) % 41 for b in range(64)]),  # no splits
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("B,H,Hkv,T,cap,lengths", SHAPES_ATT)
def test_attention(capi, B, H, Hkv, T, cap, lengths, d, dtype):
    rng = np.random.default_rng(B + H + T + cap + d)
    c = Cache(capi, rng, B, Hkv, cap, d, lengths).upload()
    q = normal(rng, (B, H, T, d), dtype)
    o, lse = attend(capi, c, q, dtype, 1.0 / np.sqrt(d))
    check_attention(c, q, dtype, float(np.float32(1.0 / np.sqrt(d))), o, lse)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
def test_attention_scales(capi, dtype, scale):
    """No scale, a negative one, and one that makes the softmax a maximum; no lse."""
    rng = np.random.default_rng(20)
    c = Cache(capi, rng, 2, 2, 90, 64, [90, 33]).upload()
    q = normal(rng, (2, 4, 3, 64), dtype)
    o, _ = attend(capi, c, q, dtype, scale, lse=False)
    check_attention(c, q, dtype, float(np.float32(scale)), o, None)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_attention_ignores_what_no_token_sees(capi, d, dtype):
    """Rows behind each length, all of them NaN blocks, and a NaN that only the newest token sees."""
    rng = np.random.default_rng(21)
    lengths = [37, 0, 64, 700]
    c = Cache(capi, rng, 4, 2, 700, d, lengths)
    q = normal(rng, (4, 4, 5, d), dtype)
    clean = Cache(capi, np.random.default_rng(21), 4, 2, 700, d, lengths)
    for b, n in enumerate(lengths):
        for x in (c.ks, c.vs):
            x[b, :, n:] = 255
    c.upload()
    o, lse = attend(capi, c, q, dtype, 0.2)
    check_attention(clean, q, dtype, float(np.float32(0.2)), o, lse)
    # key len - 3 is seen by tokens 2, 3, 4 of 5
    for b, n in ((0, 37), (2, 64), (3, 700)):
        c.vs[b, 1, n - 3, 0] = 255
        clean.vs[b, 1, n - 3, 0] = 255
    c.upload()
    o, lse = attend(capi, c, q, dtype, 0.2)
    k, v = clean.values()
    ro, rl, _, _ = mx.decode(q, k, np.nan_to_num(v), lengths, 0.2)
    want = np.zeros(o.shape, bool)
    for b in (0, 2, 3):
        want[b, 2:, 2:, :32] = True
    assert np.array_equal(np.isnan(o), want)
    assert np.allclose(o[~want], ro[~want], rtol=0.02, atol=0.02) and np.allclose(lse[np.isfinite(rl)], rl[np.isfinite(rl)], atol=1e-3)
    # a NaN key among them: the same tokens' whole rows
    c.vs[c.vs == 255] = 127
    for b, n in ((0, 37), (2, 64), (3, 700)):
        c.ks[b, 0, n - 3, 0] = 255
    c.upload()
    o, lse = attend(capi, c, q, dtype, 0.2)
    want = np.zeros(lse.shape, bool)
    for b in (0, 2, 3):
        want[b, :2, 2:] = True
    assert np.array_equal(np.isnan(lse), want) and np.array_equal(np.isnan(o).all(-1), want)
    assert np.array_equal(np.isnan(o).any(-1), want)


def test_attention_of_large_scores(capi):
    """Scores of some thousands: weights of one and zero, and none of the sums overflows."""
    rng = np.random.default_rng(22)
    c = Cache(capi, rng, 1, 1, 400, 128, [400], std=20.0).upload()
    q = normal(rng, (1, 2, 2, 128), "f32", 50.0)
    o, lse = attend(capi, c, q, "f32", 1.0)
    check_attention(c, q, "f32", 1.0, o, lse)


def test_cache_past_32_bit_offsets(capi):
    """The third sequence's rows begin 4 GiB into the codes."""
    B, cap, d = 3, (1 << 25) + 40, 128
    L = capi.lib()
    codes = [capi.DeviceBuffer((B, 1, cap, d // 2), "u8") for _ in range(2)]
    scales = [capi.DeviceBuffer((B, 1, cap, d // 32), "u8") for _ in range(2)]
    lengths = np.array([3, 0, cap - 1], np.int32)
    rng = np.random.default_rng(23)
    k, v = (normal(rng, (B, 1, 3, d), "bf16") for _ in range(2))
    f = capi.DeviceBuffer.from_numpy
    dev = (codes[0], scales[0], codes[1], scales[1], f(lengths, "i32"))
    capi.kv_append_mxfp4(f(k, "bf16"), f(v, "bf16"), *dev)
    # the last sequence's new rows, by an address formed here
    row = 2 * cap + cap - 4
    y = capi.DeviceBuffer((3, d), "bf16")
    L.call("tt_mxfp4_dequantize", capi.TT_BF16, codes[1].ptr + row * 64, scales[1].ptr + row * 4, y.ptr, 3, d, None)
    L.sync()
    assert np.array_equal(y.download(), mx.dequantize(*mx.quantize(v[2, 0]), d).astype(np.float32))
    # attention over the first rows of each: of the third as a cache of its own place
    for b, at in ((0, 0), (2, row)):
        q = normal(rng, (1, 2, 3, d), "bf16")
        o, qb, n = capi.DeviceBuffer((1, 2, 3, d), "bf16"), f(q, "bf16"), f(np.array([3], np.int32), "i32")
        L.call("tt_attn_decode_mxfp4", capi.TT_BF16, qb.ptr, codes[0].ptr + at * 64, scales[0].ptr + at * 4,
               codes[1].ptr + at * 64, scales[1].ptr + at * 4, n.ptr, o.ptr, None, 1, 2, 1, 3, 3, d, 0.1, None)
        L.sync()
        kv, vv = (mx.dequantize(*mx.quantize(x[b:b + 1]), d) for x in (k, v))
        ro, _, mag, smax = mx.decode(q, kv, vv, [3], float(np.float32(0.1)))
        assert (np.abs(o.download() - ro) <= (2 * (d + 4) * U * smax + 2.0 ** -16 + 14 * U)[..., None] * mag + 2.0 ** -8 * np.abs(ro)).all()
    # the third's own length, on the whole cache: 2^25 keys of one value and three others
    for x in codes + scales:
        L.call("tt_memset", x.ptr, 0x22 if x in codes else 127, x.nbytes)  # 1.0 everywhere
    o, lse = capi.DeviceBuffer((B, 1, 1, d), "f32"), capi.DeviceBuffer((B, 1, 1), "f32")
    qf = f(np.zeros((B, 1, 1, d), np.float32))
    capi.attn_decode_mxfp4(qf, *dev, o, lse, 0.1)
    L.sync()
    assert np.array_equal(o.download()[1], np.zeros((1, 1, d))) and np.abs(o.download()[[0, 2]] - 1).max() <= 1e-3
    assert np.abs(lse.download()[2, 0, 0] - np.log(cap - 1)) <= 1e-3


# ------------------------------------------------------------------ as they are used

def test_tokens_one_after_another(capi):
    """Prompts padded on the left, then tokens: append, attend and a layer with
    quantised weights, on a caller stream, the lengths advanced on the device."""
    B, H, Hkv, d, cap, E = 3, 4, 2, 64, 40, 48
    rng = np.random.default_rng(30)
    st = capi.Stream()
    f = capi.DeviceBuffer.from_numpy
    zero = np.zeros((B, Hkv, cap, d))
    (kc, ks), (vc, vs) = mx.quantize(zero), mx.quantize(zero)
    dev = [f(x, "u8") for x in (kc, ks, vc, vs)]
    w = rng.standard_normal((E, H * d)).astype(np.float32)
    wc, ws = quantized(capi, np.ascontiguousarray(w.T), "f32", trans=True)
    bias = normal(rng, (E,), "bf16")
    lengths = np.array([9, 4, 0], np.int32)
    for T in (9, 1, 1, 2):
        if T != 9:
            lengths = np.where(lengths > 0, lengths + T, 0).astype(np.int32)
        n = f(lengths, "i32")
        k, v, q = normal(rng, (B, Hkv, T, d), "bf16"), normal(rng, (B, Hkv, T, d), "bf16"), normal(rng, (B, H, T, d), "bf16")
        o, y = capi.DeviceBuffer((B, H, T, d), "bf16"), capi.DeviceBuffer((B * T, E), "bf16")
        bufs = [f(x, "bf16") for x in (k, v, q, bias)]
        capi.kv_append_mxfp4(bufs[0], bufs[1], *dev, n, stream=st.handle)
        capi.attn_decode_mxfp4(bufs[2], *dev, n, o, None, 0.125, stream=st.handle)
        st.sync()
        (kc, ks), (vc, vs) = mx.append(kc, ks, k, lengths), mx.append(vc, vs, v, lengths)
        for got, want in zip(dev, (kc, ks, vc, vs)):
            assert np.array_equal(got.download(), want)
        ro, _, mag, smax = mx.decode(q, mx.dequantize(kc, ks, d), mx.dequantize(vc, vs, d), lengths, 0.125)
        got = o.download()
        assert (np.abs(got - ro) <= (2 * (d + 4) * U * smax + 2.0 ** -16 + 2 * (cap + 4) * U)[..., None] * mag + 2.0 ** -8 * np.abs(ro)).all()
        x = np.ascontiguousarray(got.transpose(0, 2, 1, 3).reshape(B * T, H * d))
        capi.fc_forward_mxfp4(f(x, "bf16"), wc, ws, bufs[3], y, stream=st.handle)
        st.sync()
        xv, wv = mx.dequantize(*mx.quantize(x), H * d), mx.dequantize(*mx.quantize(w), H * d)
        ref = xv @ wv.T + bias
        assert (np.abs(y.download() - ref) <= product_bound(xv, wv, H * d, "bf16", ref, 1.0, np.abs(bias))).all()
    st.destroy()


@pytest.mark.parametrize("warm", [False, True])
def test_captured_step_replays(capi, warm):
    """Quantise, layer, append and attention in one graph, its scratch there
    (warm) or not; new inputs and lengths each replay, eager work between."""
    from test_capture_gpu import Capture

    B, H, Hkv, T, d, cap = 2, 4, 2, 2, 64, 3000
    m, n, k = 40, 100, 200
    st, f = capi.Stream(), capi.DeviceBuffer.from_numpy
    rng = np.random.default_rng(31)
    c = Cache(capi, rng, B, Hkv, cap, d, [cap, 5]).upload()
    w = rng.standard_normal((n, k))
    wc, ws = held(capi, w)
    wv = mx.dequantize(*mx.quantize(w), k)
    b = {"k": capi.DeviceBuffer((B, Hkv, T, d), "bf16"), "v": capi.DeviceBuffer((B, Hkv, T, d), "bf16"),
         "q": capi.DeviceBuffer((B, H, T, d), "bf16"), "x": capi.DeviceBuffer((m, k), "bf16"),
         "bias": f(np.zeros(n, np.float32), "bf16")}
    out = {"o": capi.DeviceBuffer((B, H, T, d), "bf16"), "y": capi.DeviceBuffer((m, n), "bf16")}
    xc, xs = capi.mxfp4_buffers((m, k))
    z = capi.DeviceBuffer((m, n), "f32")

    def call(o, y, z):
        capi.kv_append_mxfp4(b["k"], b["v"], *c.dev, c.len, stream=st.handle)
        capi.attn_decode_mxfp4(b["q"], *c.dev, c.len, o, None, 0.125, stream=st.handle)
        capi.fc_forward_mxfp4(b["x"], wc, ws, b["bias"], y, stream=st.handle)
        capi.mxfp4_quantize(b["x"], xc, xs, stream=st.handle)
        capi.gemm_mxfp4(k, 1.0, xc, xs, wc, ws, 0.0, z, stream=st.handle)

    def fill(seed):
        r = np.random.default_rng(seed)
        x = {a: normal(r, b[a].shape, "bf16") for a in ("k", "v", "q", "x")}
        for a in x:
            b[a].upload(x[a])
        c.lengths = np.array([cap - 10 * seed, 5 + seed], np.int32)
        c.len.upload(c.lengths)
        (c.kc, c.ks), (c.vc, c.vs) = mx.append(c.kc, c.ks, x["k"], c.lengths), mx.append(c.vc, c.vs, x["v"], c.lengths)
        return x

    def check(x, o, y, z):
        check_attention(c, x["q"], "bf16", 0.125, o.download(), None)
        xv = mx.dequantize(*mx.quantize(x["x"]), k)
        ref = xv @ wv.T
        assert (np.abs(y.download() - ref) <= product_bound(xv, wv, k, "bf16", ref)).all()
        assert (np.abs(z.download() - ref) <= product_bound(xv, wv, k, "f32", ref)).all()

    eager = (capi.DeviceBuffer((B, H, T, d), "bf16"), capi.DeviceBuffer((m, n), "bf16"), capi.DeviceBuffer((m, n), "f32"))
    capi.lib().call("tt_empty_cache")
    if warm:
        x = fill(0)
        call(*eager)
        st.sync()
        check(x, *eager)
    with Capture(capi, st.handle) as g:
        call(out["o"], out["y"], z)
    for seed in (1, 2, 3):
        x = fill(seed)
        for buf in (out["o"], out["y"], z):
            buf.upload(np.full(buf.shape, 77.0, np.float32))
        g.launch()
        check(x, out["o"], out["y"], z)
        call(*eager)  # eager work on the same stream between replays
        st.sync()
        check(x, *eager)
    g.destroy()
    st.destroy()


def test_two_streams_at_once(capi):
    """Split attention and layers queued on two streams: each has scratch of its own."""
    rng = np.random.default_rng(32)
    f = capi.DeviceBuffer.from_numpy
    runs = []
    for i in range(2):
        c = Cache(capi, rng, 1, 2, 2500, 64, [2500 - i]).upload()
        q, x, w = normal(rng, (1, 4, 1, 64), "bf16"), normal(rng, (50, 96), "bf16"), rng.standard_normal((33, 96))
        wc, ws = held(capi, w)
        runs.append(dict(c=c, q=q, x=x, w=w, st=capi.Stream(), wc=wc, ws=ws, qb=f(q, "bf16"), xb=f(x, "bf16"),
                         bias=f(np.zeros(33, np.float32), "bf16"), o=capi.DeviceBuffer(q.shape, "bf16"),
                         y=capi.DeviceBuffer((50, 33), "bf16")))
    for _ in range(20):
        for r in runs:
            capi.attn_decode_mxfp4(r["qb"], *r["c"].dev, r["c"].len, r["o"], None, 0.125, stream=r["st"].handle)
            capi.fc_forward_mxfp4(r["xb"], r["wc"], r["ws"], r["bias"], r["y"], stream=r["st"].handle)
    for r in runs:
        r["st"].sync()
        check_attention(r["c"], r["q"], "bf16", 0.125, r["o"].download(), None)
        xv, wv = mx.dequantize(*mx.quantize(r["x"]), 96), mx.dequantize(*mx.quantize(r["w"]), 96)
        ref = xv @ wv.T
        assert (np.abs(r["y"].download() - ref) <= product_bound(xv, wv, 96, "bf16", ref)).all()
        r["st"].destroy()


@pytest.mark.parametrize("warm", [False, True])
def test_two_graphs_and_two_streams_of_long_rows(capi, warm):
    """Layers of rows that are quantised into the workspace, beside split
    attention: two graphs captured on one stream and replayed in turn, with eager
    calls between and on a second stream at the same time."""
    from test_capture_gpu import Capture

    m, n, k = 20, 33, 3000  # 6000 bytes a row, 120000 together
    rng = np.random.default_rng(33)
    f = capi.DeviceBuffer.from_numpy
    st, other = capi.Stream(), capi.Stream()
    jobs = []
    for i in range(3):
        c = Cache(capi, rng, 1, 2, 2500, 64, [2400 - i]).upload()
        q, x, w = normal(rng, (1, 4, 1, 64), "bf16"), normal(rng, (m, k), "bf16"), rng.standard_normal((n, k))
        wc, ws = held(capi, w)
        xv, wv = mx.dequantize(*mx.quantize(x), k), mx.dequantize(*mx.quantize(w), k)
        jobs.append(dict(c=c, q=q, qb=f(q, "bf16"), xb=f(x, "bf16"), wc=wc, ws=ws, bias=f(np.zeros(n, np.float32), "bf16"),
                         o=capi.DeviceBuffer(q.shape, "bf16"), y=capi.DeviceBuffer((m, n), "bf16"), xv=xv, wv=wv))

    def call(j, s):
        capi.attn_decode_mxfp4(j["qb"], *j["c"].dev, j["c"].len, j["o"], None, 0.125, stream=s.handle)
        capi.fc_forward_mxfp4(j["xb"], j["wc"], j["ws"], j["bias"], j["y"], stream=s.handle)

    def check(j):
        check_attention(j["c"], j["q"], "bf16", 0.125, j["o"].download(), None)
        ref = j["xv"] @ j["wv"].T
        assert (np.abs(j["y"].download() - ref) <= product_bound(j["xv"], j["wv"], k, "bf16", ref)).all()

    capi.lib().call("tt_empty_cache")
    if warm:
        call(jobs[0], st)
        st.sync()
    graphs = []
    for j in jobs[:2]:
        with Capture(capi, st.handle) as g:
            call(j, st)
        graphs.append(g)
    for _ in range(3):
        for j in jobs:
            for buf in (j["o"], j["y"]):
                buf.upload(np.full(buf.shape, 77.0, np.float32))
        call(jobs[2], other)
        for g in graphs:
            g.launch()
        st.sync()
        other.sync()
        for j in jobs:
            check(j)
        call(jobs[2], st)  # eager, on the graphs' stream
        st.sync()
        check(jobs[2])
    for g in graphs:
        g.destroy()
    st.destroy()
    other.destroy()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T", [1, 3])
def test_a_row_is_the_same_whatever_is_beside_it(capi, T, dtype):
    """The query rows that share a K / V head are one tile: what the others hold,
    NaN and rows whose maximum rises with every key included, changes no bit."""
    from test_capture_gpu import Capture

    H, d, cap = 4, 64, 5000
    rng = np.random.default_rng(34 + T)
    c = Cache(capi, rng, 1, 1, cap, d, [cap])
    rising = np.linspace(0.0, 20.0, cap)[:, None] * np.eye(1, d, 1)  # along one axis, which only some queries have
    c.kc, c.ks = mx.quantize((mx.dequantize(c.kc, c.ks, d)[0, 0] + rising)[None, None])
    c.upload()
    q = normal(rng, (1, H, T, d), dtype)
    q[:, 0, :, 1] = 0.0
    q[:, 0, :, 0] = 40.0  # scores far from zero
    beside = [q.copy() for _ in range(3)]
    beside[0][:, 1:] = 0.0
    beside[1][:, 1:] = np.nan
    beside[2][:, 1:, :, 1] = 8.0
    for warm in (True, False):  # split over workgroups, and not
        outs = []
        for x in beside:
            b, st = capi.DeviceBuffer.from_numpy(x, dtype), capi.Stream()
            o, lse = capi.DeviceBuffer(x.shape, dtype), capi.DeviceBuffer(x.shape[:3])
            if warm:
                capi.attn_decode_mxfp4(b, *c.dev, c.len, o, lse, 0.125, stream=st.handle)
            else:
                with Capture(capi, st.handle) as g:
                    capi.attn_decode_mxfp4(b, *c.dev, c.len, o, lse, 0.125, stream=st.handle)
                g.launch()
                g.destroy()
            st.sync()
            outs.append((o.download()[:, 0], lse.download()[:, 0]))
            if x is beside[1]:
                assert np.isnan(o.download()[:, 1:]).all()
            st.destroy()
        for o, lse in outs[1:]:
            assert np.array_equal(o, outs[0][0]) and np.array_equal(lse, outs[0][1])


# ------------------------------------------------------------------ products of many tiles

MANY = [(2900, 3001, 31), (2900, 3001, 96), (2816, 3328, 160), (3001, 2900, 544), (2561, 3500, 1100), (2820, 3329, 4128)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", MANY)
def test_gemm_of_many_tiles(capi, m, n, k, dtype):
    """More than 512 tiles of 128 x 128: whole and partly filled larger ones, odd
    numbers of blocks, C at every alignment of its rows, and nothing beside it."""
    rng = np.random.default_rng(m + n + k)
    a, b = rng.standard_normal((m, k)), rng.standard_normal((n, k)) * np.ldexp(1.0, rng.integers(-6, 6, (n, 1)))
    (ac, as_), (bc, bs) = held(capi, a), held(capi, b)
    av, bv = mx.dequantize(*mx.quantize(a), k), mx.dequantize(*mx.quantize(b), k)
    ref = av @ bv.T
    for off in (0, 1):
        buf = capi.DeviceBuffer.from_numpy(np.full(m * n + 64, 77.0, np.float32), dtype)
        capi.lib().call("tt_gemm_mxfp4", capi.TT_BF16 if dtype == "bf16" else capi.TT_F32, m, n, k, 1.0, ac.ptr, as_.ptr,
                        bc.ptr, bs.ptr, 0.0, buf.ptr + (8 + off) * capi.DeviceBuffer.ITEM[dtype], None)
        capi.lib().sync()
        got = buf.download()
        assert (got[:8 + off] == 77.0).all() and (got[8 + off + m * n:] == 77.0).all()
        got = got[8 + off:8 + off + m * n].reshape(m, n)
        assert (np.abs(got - ref) <= product_bound(av, bv, k, dtype, ref)).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(600, 1101, 200), (2900, 3001, 200), (2816, 3328, 96)])
def test_tiles_with_old_c_and_with_a_bias(capi, m, n, k, dtype):
    """128 x 128 and 256 x 256 tiles: alpha and beta; the layer with a bias of each output and of all."""
    rng = np.random.default_rng(m + n)
    x, b, c0 = normal(rng, (m, k), dtype), rng.standard_normal((n, k)), normal(rng, (m, n), dtype)
    (ac, as_), (bc, bs) = held(capi, x), held(capi, b)
    av, bv = mx.dequantize(*mx.quantize(x), k), mx.dequantize(*mx.quantize(b), k)
    ref = av @ bv.T
    f = capi.DeviceBuffer.from_numpy
    c = f(c0, dtype)
    capi.gemm_mxfp4(k, -0.75, ac, as_, bc, bs, 0.5, c)
    capi.lib().sync()
    want = -0.75 * ref + 0.5 * c0
    assert (np.abs(c.download() - want) <= product_bound(av, bv, k, dtype, want, 0.75, np.abs(c0))).all()
    for size in (n, 1):
        bias = normal(rng, (size,), dtype)
        capi.fc_forward_mxfp4(f(x, dtype), bc, bs, f(bias, dtype), c)
        capi.lib().sync()
        want = ref + bias
        assert (np.abs(c.download() - want) <= product_bound(av, bv, k, dtype, want, 1.0, np.abs(bias))).all()


def test_nan_blocks_of_many_tiles_reach_their_rows_alone(capi):
    m, n, k = 2900, 3001, 200
    rng = np.random.default_rng(35)
    a, b = rng.standard_normal((m, k)), rng.standard_normal((n, k))
    a[[0, 300, 2899], [5, 199, 64]] = np.nan
    b[[1, 1500, 3000], [0, 100, 199]] = np.inf
    (ac, as_), (bc, bs) = held(capi, a), held(capi, b)
    c = capi.DeviceBuffer((m, n), "f32")
    capi.gemm_mxfp4(k, 1.0, ac, as_, bc, bs, 0.0, c)
    capi.lib().sync()
    want = np.zeros((m, n), bool)
    want[[0, 300, 2899]] = True
    want[:, [1, 1500, 3000]] = True
    assert np.array_equal(np.isnan(c.download()), want)


@pytest.mark.parametrize("off", [1, 6, 15])
@pytest.mark.parametrize("m,n,k", [(5, 40, 1000), (300, 520, 1000), (600, 1101, 1000), (2900, 3001, 544)])
def test_scales_at_any_address_among_others(capi, m, n, k, off):
    """Scales in the middle of a buffer whose other bytes read as NaN."""
    rng = np.random.default_rng(m + off)
    a, b = rng.standard_normal((m, k)), rng.standard_normal((n, k))
    (qa, sa), (qb, sb) = mx.quantize(a), mx.quantize(b)

    def among(s):
        buf = np.full(s.size + 64, 255, np.uint8)
        buf[off:off + s.size] = s.reshape(-1)
        return capi.DeviceBuffer.from_numpy(buf, "u8")

    f = capi.DeviceBuffer.from_numpy
    ac, bc, as_, bs = f(qa, "u8"), f(qb, "u8"), among(sa), among(sb)
    c = capi.DeviceBuffer((m, n), "f32")
    capi.lib().call("tt_gemm_mxfp4", capi.TT_F32, m, n, k, 1.0, ac.ptr, as_.ptr + off, bc.ptr, bs.ptr + off, 0.0, c.ptr, None)
    capi.lib().sync()
    av, bv = mx.dequantize(qa, sa, k), mx.dequantize(qb, sb, k)
    ref = av @ bv.T
    assert (np.abs(c.download() - ref) <= product_bound(av, bv, k, "f32", ref)).all()
    x, bias = f(a.astype(np.float32)), f(np.zeros(n, np.float32))
    capi.lib().call("tt_fc_forward_mxfp4", capi.TT_F32, m, k, n, x.ptr, bc.ptr, bs.ptr + off, bias.ptr, 0, c.ptr, None)
    capi.lib().sync()
    av = mx.dequantize(*mx.quantize(a.astype(np.float32)), k)
    ref = av @ bv.T
    assert (np.abs(c.download() - ref) <= product_bound(av, bv, k, "f32", ref)).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [1, 7, 33, 39, 61, 95, 1023])
def test_a_rows_end_does_not_take_in_the_next_row(capi, cols, dtype):
    """Rows behind a row that is NaN, infinite or large from its first value on."""
    rng = np.random.default_rng(cols)
    x = normal(rng, (41, cols), dtype)
    x[1::8] = np.nan
    x[3::8] = np.inf
    x[5::8] *= 2.0 ** 60
    codes, scales = quantized(capi, x, dtype)
    rc, rs = mx.quantize(x)
    assert np.array_equal(scales.download(), rs) and np.array_equal(codes.download(), rc)


def test_two_host_threads_on_one_stream(capi):
    """Calls of two threads share the stream's scratch: each call's kernels are queued together."""
    import threading

    m, n, k = 24, 40, 3000
    rng = np.random.default_rng(36)
    f = capi.DeviceBuffer.from_numpy
    jobs, st = [], capi.Stream()
    for i in range(2):
        c = Cache(capi, rng, 1, 2, 2500, 64, [2300 - i]).upload()
        q, x, w = normal(rng, (1, 4, 1, 64), "bf16"), normal(rng, (m, k), "bf16"), rng.standard_normal((n, k))
        wc, ws = held(capi, w)
        xv, wv = mx.dequantize(*mx.quantize(x), k), mx.dequantize(*mx.quantize(w), k)
        jobs.append(dict(c=c, q=q, qb=f(q, "bf16"), xb=f(x, "bf16"), wc=wc, ws=ws, bias=f(np.zeros(n, np.float32), "bf16"),
                         o=[capi.DeviceBuffer(q.shape, "bf16") for _ in range(30)],
                         y=[capi.DeviceBuffer((m, n), "bf16") for _ in range(30)], xv=xv, wv=wv, error=None))

    def work(j):
        try:
            for o, y in zip(j["o"], j["y"]):
                capi.attn_decode_mxfp4(j["qb"], *j["c"].dev, j["c"].len, o, None, 0.125, stream=st.handle)
                capi.fc_forward_mxfp4(j["xb"], j["wc"], j["ws"], j["bias"], y, stream=st.handle)
        except Exception as e:  # reported by the test's own thread
            j["error"] = e

    threads = [threading.Thread(target=work, args=(j,)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    st.sync()
    for j in jobs:
        assert j["error"] is None
        ref = j["xv"] @ j["wv"].T
        for o, y in zip(j["o"], j["y"]):
            check_attention(j["c"], j["q"], "bf16", 0.125, o.download(), None)
            assert (np.abs(y.download() - ref) <= product_bound(j["xv"], j["wv"], k, "bf16", ref)).all()
    st.destroy()
