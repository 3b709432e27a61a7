"""GPU tests of the 4-bit operators where values, sizes or addresses are at
their limits.  Bounds as in test_mxfp4_gpu, whose helpers they use; where an
infinity or a NaN is expected, it is expected exactly there."""
import numpy as np
import pytest

from oracle import attn_oracle as orc
from oracle import mxfp4_oracle as mx
from test_mxfp4_gpu import HALF, U, Cache, attend, capi, check_attention, held, normal, product_bound  # noqa: F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ attention: infinite values

def attention_with_infinities(c, q, dtype, scale, o, lse):
    """As check_attention, values from 2^128 on being infinite: a row that sees one is infinite in its column."""
    k, v = c.values()
    d, n = q.shape[3], c.shape[2]
    with np.errstate(over="ignore"):
        k, v = k.astype(np.float32).astype(np.float64), v.astype(np.float32).astype(np.float64)
    with np.errstate(invalid="ignore"):
        ro, rl, mag, _ = mx.decode(q, k, v, c.lengths, scale)
        smax = mx.decode(q, np.where(np.isinf(k), 0.0, k), v, c.lengths, scale)[3]  # infinite keys have no error
        e = (d + 4) * U * smax
        tol = (2 * e + (U if dtype == "f32" else 2.0 ** -16) + 2 * (n + 4) * U)[..., None] * mag + HALF[dtype] * np.abs(ro)
        off = np.abs(o - ro)
    f = np.isfinite(ro)
    assert np.array_equal(np.isnan(o), np.isnan(ro))
    assert np.array_equal(np.isposinf(o), np.isposinf(ro)) and np.array_equal(np.isneginf(o), np.isneginf(ro))
    assert (off[f] <= tol[f]).all()
    f = np.isfinite(rl)
    assert np.array_equal(np.isneginf(lse), np.isneginf(rl))
    assert (np.abs(lse[f] - rl[f]) <= e[f] + (n + 4) * U + 4 * U * np.abs(rl[f])).all()
    return ro


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("byte", [253, 254])
def test_infinite_values_reach_only_the_tokens_that_see_them(capi, byte, d, dtype):
    """The newest token's V block infinite in some columns and large in others, behind the older tokens' mask."""
    rng = np.random.default_rng(byte + d)
    lengths = [37, 3, 64, 700]
    c = Cache(capi, rng, 4, 2, 700, d, lengths)
    for b, n in enumerate(lengths):
        c.vs[b, 0, n - 1, d // 32 - 1] = byte
        c.vc[b, 0, n - 1, -16:] = rng.permutation(16).astype(np.uint8) * 17  # every code twice
    q = normal(rng, (4, 4, 3, d), dtype)
    o, lse = attend(capi, c.upload(), q, dtype, 0.2)
    ro = attention_with_infinities(c, q, dtype, float(np.float32(0.2)), o, lse)
    assert np.isfinite(ro[:, :, :2]).all() and np.isinf(ro[:, :2, 2]).any() and (np.abs(ro[:, :2, 2]) > 1e36).any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("at", [0, 10, 31, 70, 299])
def test_an_infinite_value_that_every_token_sees(capi, at, d, dtype):
    """Weights of exactly one and of any other value; a column is infinite, not NaN, and the others are as before."""
    rng = np.random.default_rng(at + d)
    c = Cache(capi, rng, 1, 1, 300, d, [300])
    c.vs[0, 0, at, 0] = 254
    c.vc[0, 0, at, :16] = rng.integers(0, 256, 16)
    c.upload()
    for q in (np.zeros((1, 3, 1, d), np.float32), normal(rng, (1, 3, 1, d), dtype)):
        o, lse = attend(capi, c, q, dtype, 0.2)
        ro = attention_with_infinities(c, q, dtype, float(np.float32(0.2)), o, lse)
        assert np.isinf(ro).any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_infinite_and_nan_values_in_one_cache(capi, d, dtype):
    """Blocks of bytes 253 to 255 anywhere, several in a step, some rows' border among them."""
    rng = np.random.default_rng(d)
    lengths = [300, 65, 1000]
    c = Cache(capi, rng, 3, 2, 1000, d, lengths)
    at = rng.random((3, 2, 1000, d // 32)) < 0.01
    c.vs[at] = rng.integers(253, 256, int(at.sum()))
    c.vs[:, :, :30] = 127
    c.vs[2, :, :, 0] = 127  # columns with none
    q = normal(rng, (3, 4, 3, d), dtype) * np.float32(0.25)
    q = orc.bf16_round(q)
    o, lse = attend(capi, c.upload(), q, dtype, 0.2)
    ro = attention_with_infinities(c, q, dtype, float(np.float32(0.2)), o, lse)
    assert np.isnan(ro).any() and np.isfinite(ro).any() and (d == 32 or np.isinf(ro).any())


# ------------------------------------------------------------------ attention: infinite scores

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_infinite_queries(capi, d, dtype):
    """A query value of -inf: scores of -inf over positive keys leave nothing (o = 0, lse = -inf), and hide positive
    keys beside others; over a key of zero, or with a score of +inf, the row is NaN.  A NaN query is NaN."""
    rng = np.random.default_rng(d)
    c = Cache(capi, rng, 1, 5, 70, d, [70])
    k = mx.dequantize(c.kc, c.ks, d)
    k[0, :, :, 0] = 1.5
    k[0, 1, 20:30, 0] = -1.5
    k[0, 2, 40, 0] = 0.0
    c.kc, c.ks = mx.quantize(k)
    q = normal(rng, (1, 5, 2, d), dtype)
    q[0, :, 0, 0] = -np.inf
    q[0, 1, 0, 0] = np.inf
    q[0, 3, 1, 5] = np.nan
    q[0, 4, 0, 0] = np.inf
    if dtype == "f32":  # a NaN of which the upper half alone would be infinite
        q[0, 3, 1, 5] = np.array(0x7F800001, np.uint32).view(np.float32)
    o, lse = attend(capi, c.upload(), q, dtype, 0.2)
    assert (o[0, 0, 0] == 0).all() and np.isneginf(lse[0, 0, 0])
    for h, t in ((1, 0), (2, 0), (3, 1), (4, 0)):
        assert np.isnan(o[0, h, t]).all() and np.isnan(lse[0, h, t])
    keep = np.zeros((1, 5, 2), bool)
    keep[0, [0, 1, 2, 4], 1] = True
    q[~keep] = 0.0
    k, v = c.values()
    ro, rl, mag, smax = mx.decode(q, k, v, c.lengths, float(np.float32(0.2)))
    e = (d + 4) * U * smax
    tol = (2 * e + (U if dtype == "f32" else 2.0 ** -16) + 2 * 74 * U)[..., None] * mag + HALF[dtype] * np.abs(ro)
    assert (np.abs(o - ro)[keep] <= tol[keep]).all()
    assert (o[0, 3, 0] == 0).all() and np.isneginf(lse[0, 3, 0])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("byte", [253, 254])
def test_infinite_keys(capi, byte, d, dtype):
    """Keys of infinite elements under queries of one bf16 term: a score of -inf takes its key out, and no more."""
    rng = np.random.default_rng(byte + d)
    c = Cache(capi, rng, 2, 1, 500, d, [500, 90])
    for b, j in ((0, 3), (0, 450), (1, 88), (1, 89)):
        c.ks[b, 0, j] = byte
        c.kc[b, 0, j] = 0x77  # 6 everywhere: infinite
    q = -np.abs(normal(rng, (2, 3, 2, d), "bf16")) - np.float32(2.0 ** -10)
    q = orc.bf16_round(q)
    o, lse = attend(capi, c.upload(), q, dtype, 0.2)
    attention_with_infinities(c, q, dtype, float(np.float32(0.2)), o, lse)


def test_weights_of_two_terms(capi):
    """The weights of a bf16 call are off by 2^-17.  Two keys of weight one and values 6 and 6 2^-7 against twelve
    of weight p = (1 + 2^-7 - x) / 2 and value -1: o = 6 x / 8 and a little, so its store rounds nearly nothing.

    Bound: 2^-17 of 12 p; the store's 2^-8 |o|; of p itself and of the sums, none of which passes 6.1, the score's three
    exact products and its scale (4 2^-24 0.7), exp2 (2^-23) and 16 additions (2^-24 each): 30 2^-24 6.1, over 2 + 12 p."""
    H, d = 64, 32
    k, v = np.zeros((1, 1, 14, d)), np.full((1, 1, 14, d), -1.0)
    k[:, :, 2:] = 1.0
    v[:, :, 0], v[:, :, 1] = 6.0, 6.0 * 2.0 ** -7
    c = Cache(capi, np.random.default_rng(0), 1, 1, 14, d, [14])
    (c.kc, c.ks), (c.vc, c.vs) = mx.quantize(k), mx.quantize(v)
    p = 0.5 * (1 + 2.0 ** -7 - 2.0 ** -11 * (np.arange(H) + 0.5) / H)
    q = np.zeros((1, H, 1, d), np.float32)
    left = np.log(p)
    for e in range(3):
        q[0, :, 0, e] = orc.bf16_round(left.astype(np.float32))
        left = left - q[0, :, 0, e]
    o, _ = attend(capi, c.upload(), q, "bf16", 1.0)
    ro = mx.decode(q, k, v, [14], 1.0)[0]
    tol = (2.0 ** -17 * 12 * p + 30 * U * 6.1) / (2 + 12 * p)
    assert (np.abs(o - ro)[0, :, 0] <= tol[:, None] + 2.0 ** -8 * np.abs(ro[0, :, 0])).all()


# ------------------------------------------------------------------ attention: sizes, scales, offsets

def test_attention_of_more_rows_than_the_merge_could_launch(capi):
    """2^24 + 40 tokens of one head: the keys are not split, so nothing merges them."""
    T, d, cap = (1 << 24) + 40, 32, 48
    rng = np.random.default_rng(41)
    c = Cache(capi, rng, 1, 1, cap, d, [T]).upload()
    q, o, lse = capi.DeviceBuffer((1, 1, T, d), "bf16"), capi.DeviceBuffer((1, 1, T, d), "bf16"), capi.DeviceBuffer((1, 1, T))
    L, some = capi.lib(), normal(rng, (2, 1, 1, 200, d), "bf16")
    L.call("tt_memset", q.ptr, 0, q.nbytes)
    head = capi.DeviceBuffer.from_numpy(some, "bf16")
    places = (0, T - 200)  # the first tokens, which see few keys, and the last
    for i, t in enumerate(places):
        L.call("tt_memcpy_d2d", q.ptr + t * 2 * d, head.ptr + i * 400 * d, 400 * d)
    capi.attn_decode_mxfp4(q, *c.dev, c.len, o, lse, 0.2)
    L.sync()
    k, v = c.values()
    got, gl = capi.DeviceBuffer((2, 1, 1, 200, d), "bf16"), capi.DeviceBuffer((2, 1, 1, 200))
    for i, t in enumerate(places):
        L.call("tt_memcpy_d2d", got.ptr + i * 400 * d, o.ptr + t * 2 * d, 400 * d)
        L.call("tt_memcpy_d2d", gl.ptr + i * 800, lse.ptr + t * 4, 800)
    L.sync()
    for i, n in enumerate((200, cap + 200)):  # as the last 200 tokens of so many keys
        ro, rl, mag, smax = mx.decode(some[i], k, v, [n], float(np.float32(0.2)))
        e = (d + 4) * U * smax
        assert (np.abs(got.download()[i] - ro) <= (2 * e + 2.0 ** -16 + 104 * U)[..., None] * mag + HALF["bf16"] * np.abs(ro)).all()
        assert (np.abs(gl.download()[i] - rl) <= e + 52 * U + 4 * U * np.abs(rl)).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [0.0, 1e-38, -1e-38, 1e-41])
def test_attention_of_no_scale_over_large_scores(capi, scale, dtype):
    """Products up to 10^38 under a scale of zero, or one that makes them small."""
    rng = np.random.default_rng(40)
    c = Cache(capi, rng, 2, 2, 90, 64, [90, 33], std=2.0 ** 122).upload()
    q = np.zeros((2, 4, 3, 64), np.float32)
    q[..., 0] = orc.bf16_round(rng.uniform(-1, 1, (2, 4, 3)).astype(np.float32))
    o, lse = attend(capi, c, q, dtype, scale)
    check_attention(c, q, dtype, float(np.float32(scale)), o, lse)


@pytest.mark.parametrize("scale", [0.0, 1e-41])
def test_attention_of_no_scale_where_the_host_flushes_small_values(capi, scale):
    import torch

    rng = np.random.default_rng(43)
    c = Cache(capi, rng, 2, 2, 90, 64, [90, 33]).upload()
    q = normal(rng, (2, 4, 3, 64), "bf16")
    assert torch.set_flush_denormal(True)
    try:
        o, lse = attend(capi, c, q, "bf16", scale)
    finally:
        torch.set_flush_denormal(False)
    check_attention(c, q, "bf16", 0.0, o, lse)  # 10^-41 of scores below 10^3 is nothing


def test_attention_past_32_bit_offsets(capi):
    """The third sequence's keys begin 4 GiB into the codes and end in three that hold nearly all of the weight: by an
    offset cut to 32 bits they would be rows of other sequences, which are 1 throughout."""
    B, cap, d = 3, (1 << 25) + 40, 128
    L, f = capi.lib(), capi.DeviceBuffer.from_numpy
    codes = [capi.DeviceBuffer((B, 1, cap, d // 2), "u8") for _ in range(2)]
    scales = [capi.DeviceBuffer((B, 1, cap, d // 32), "u8") for _ in range(2)]
    for x in codes + scales:
        L.call("tt_memset", x.ptr, 0x22 if x in codes else 127, x.nbytes)  # 1.0 everywhere
    lengths = np.array([cap, 0, cap - 1], np.int32)
    rng = np.random.default_rng(42)
    k, v = (normal(rng, (B, 1, 3, d), "bf16") for _ in range(2))
    dev = (codes[0], scales[0], codes[1], scales[1], f(lengths, "i32"))
    capi.kv_append_mxfp4(f(k, "bf16"), f(v, "bf16"), *dev)
    kv, vv = (mx.dequantize(*mx.quantize(x), d) for x in (k, v))
    # a query that the last sequence's own newest keys answer with scores far above those of the others
    q = np.zeros((B, 1, 1, d), np.float32)
    q[0, 0, 0] = orc.bf16_round((kv[0, 0, 1] - 1.0).astype(np.float32))
    q[2, 0, 0] = orc.bf16_round((kv[2, 0, 0] - 1.0).astype(np.float32))
    o, lse = capi.DeviceBuffer((B, 1, 1, d), "f32"), capi.DeviceBuffer((B, 1, 1), "f32")
    capi.attn_decode_mxfp4(f(q), *dev, o, lse, 1.0)
    L.sync()
    o, lse = o.download(), lse.download()
    assert np.array_equal(o[1], np.zeros((1, 1, d))) and np.isneginf(lse[1]).all()
    for b in (0, 2):
        n = int(lengths[b]) - 3
        s = np.append(kv[b, 0] @ q[b, 0, 0].astype(np.float64), q[b, 0, 0].astype(np.float64).sum())
        w = np.exp(s - s.max()) * np.array([1, 1, 1, n])
        want = (w[:3] @ vv[b, 0] + w[3]) / w.sum()
        # More than 0.999 of the weight on the appended keys, so the roundings of a sum of 2^25 weights (2^-24 each of
        # what they add up to) stay below 2^25 2^-24 0.001; weights below the smallest fp32, 2^-149, may be lost, at
        # most 2^25 of them.
        assert w[:3].sum() > 0.999 * w.sum()
        lost = 2.0 ** (25 - 149) * max(1.0, np.abs(vv[b, 0]).max())
        assert np.abs(want - 1.0).max() > 0.5  # what keys of other rows would give
        e = (d + 4) * U * (np.abs(kv[b, 0]) @ np.abs(q[b, 0, 0])).max()
        assert (np.abs(o[b, 0, 0] - want) <= (2 * e + 2e-3) * (w[:3] @ np.abs(vv[b, 0]) + w[3]) / w.sum() + lost).all()
        assert abs(lse[b, 0, 0] - s.max() - np.log(w.sum())) <= e + 2e-3


# ------------------------------------------------------------------ products of extreme and narrow shapes

def test_layer_of_many_blocks_without_its_workspace(capi):
    """65552 x 32768 outputs are more blocks of 16 x 16 than one launch takes: captured before a call has left the
    workspace on the stream, the layer quantises its rows as it reads them, in several launches."""
    from test_capture_gpu import Capture

    m, n, k = 65552, 32768, 32
    rng = np.random.default_rng(50)
    f, L = capi.DeviceBuffer.from_numpy, capi.lib()
    x, w, bias = normal(rng, (m, k), "bf16"), rng.standard_normal((n, k)), normal(rng, (n,), "bf16")
    wc, ws = held(capi, w)
    xb, bb, out = f(x, "bf16"), f(bias, "bf16"), capi.DeviceBuffer((m, n), "bf16")
    L.call("tt_memset", out.ptr, 0, out.nbytes)
    L.call("tt_empty_cache")
    st = capi.Stream()
    with Capture(capi, st.handle) as g:
        capi.fc_forward_mxfp4(xb, wc, ws, bb, out, stream=st.handle)
    g.launch()
    g.destroy()
    st.destroy()
    wv = mx.dequantize(*mx.quantize(w), k)
    rows = capi.DeviceBuffer((48, n), "bf16")
    for r0 in (0, 32 * 1024, 65504):
        L.call("tt_memcpy_d2d", rows.ptr, out.ptr + r0 * n * 2, rows.nbytes)
        L.sync()
        xv = mx.dequantize(*mx.quantize(x[r0:r0 + 48]), k)
        ref = xv @ wv.T + bias
        assert (np.abs(rows.download() - ref) <= product_bound(xv, wv, k, "bf16", ref, 1.0, np.abs(bias))).all()


def test_product_of_one_row_by_more_than_2_27(capi):
    m, n, k = 1, (1 << 27) + 40, 32
    L = capi.lib()
    rng = np.random.default_rng(51)
    a, b = rng.standard_normal((m, k)), rng.standard_normal((64, k))
    ac, as_ = held(capi, a)
    bc, bs = capi.mxfp4_buffers((n, k))
    L.call("tt_memset", bc.ptr, 0x22, bc.nbytes)  # 1.0 everywhere
    L.call("tt_memset", bs.ptr, 127, bs.nbytes)
    tc, ts = held(capi, b)
    L.call("tt_memcpy_d2d", bc.ptr + (n - 64) * 16, tc.ptr, 64 * 16)
    L.call("tt_memcpy_d2d", bs.ptr + (n - 64), ts.ptr, 64)
    c = capi.DeviceBuffer((m, n), "bf16")
    L.call("tt_memset", c.ptr, 0, c.nbytes)
    capi.gemm_mxfp4(k, 1.0, ac, as_, bc, bs, 0.0, c)
    L.sync()
    got = c.download()
    av, bv = mx.dequantize(*mx.quantize(a), k), mx.dequantize(*mx.quantize(b), k)
    ref = av @ bv.T
    assert (np.abs(got[:, -64:] - ref) <= product_bound(av, bv, k, "bf16", ref)).all()
    one = av.sum()
    assert (np.abs(got[:, :-64] - one) <= (k + 4) * U * np.abs(av).sum() + 2.0 ** -8 * abs(one)).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(70000, 10, 64), (20000, 10, 784), (9000, 1, 100), (5, 70000, 64), (40000, 17, 33), (8192, 128, 1024)])
def test_narrow_products(capi, m, n, k, dtype):
    """Many rows and few columns, as a classifier's last layer has: the product and the layer."""
    rng = np.random.default_rng(m + n)
    x, b, bias = normal(rng, (m, k), dtype), rng.standard_normal((n, k)), normal(rng, (n,), dtype)
    (ac, as_), (bc, bs) = held(capi, x), held(capi, b)
    f, c = capi.DeviceBuffer.from_numpy, capi.DeviceBuffer((m, n), dtype)
    capi.gemm_mxfp4(k, 1.0, ac, as_, bc, bs, 0.0, c)
    capi.lib().sync()
    av, bv = mx.dequantize(*mx.quantize(x), k), mx.dequantize(*mx.quantize(b), k)
    ref = av @ bv.T
    assert (np.abs(c.download() - ref) <= product_bound(av, bv, k, dtype, ref)).all()
    capi.fc_forward_mxfp4(f(x, dtype), bc, bs, f(bias, dtype), c)
    capi.lib().sync()
    ref += bias
    assert (np.abs(c.download() - ref) <= product_bound(av, bv, k, dtype, ref, 1.0, np.abs(bias))).all()


@pytest.mark.parametrize("m,n", [(600, 1101), (2900, 3001)])
def test_tiles_of_no_k_are_beta_c(capi, m, n):
    c0 = normal(np.random.default_rng(52), (m, n), "f32")
    c = capi.DeviceBuffer.from_numpy(c0)
    capi.lib().call("tt_gemm_mxfp4", capi.TT_F32, m, n, 0, 1.0, None, None, None, None, 0.5, c.ptr, None)
    capi.lib().sync()
    assert np.array_equal(c.download(), c0 * 0.5)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(3, 50, 97), (30, 50, 3000), (600, 1101, 200)])
def test_layer_at_any_element_alignment(capi, m, n, k, dtype):
    """in, bias and out one element into their buffers; what lies around out stays."""
    rng = np.random.default_rng(m)
    x, w, bias = normal(rng, (m, k), dtype), rng.standard_normal((n, k)), normal(rng, (n,), dtype)
    wc, ws = held(capi, w)
    f, e = capi.DeviceBuffer.from_numpy, capi.DeviceBuffer.ITEM[dtype]
    xb, bb = f(np.concatenate(([9.0], x.ravel())).astype(np.float32), dtype), f(np.append(9.0, bias).astype(np.float32), dtype)
    out = f(np.full(m * n + 2, 77.0, np.float32), dtype)
    capi.lib().call("tt_fc_forward_mxfp4", capi.TT_BF16 if dtype == "bf16" else capi.TT_F32, m, k, n, xb.ptr + e, wc.ptr,
                    ws.ptr, bb.ptr + e, 0, out.ptr + e, None)
    capi.lib().sync()
    got = out.download()
    assert got[0] == got[-1] == 77.0
    xv, wv = mx.dequantize(*mx.quantize(x), k), mx.dequantize(*mx.quantize(w), k)
    ref = xv @ wv.T + bias
    assert (np.abs(got[1:-1].reshape(m, n) - ref) <= product_bound(xv, wv, k, dtype, ref, 1.0, np.abs(bias))).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_at_any_element_alignment(capi, dtype):
    """q, o and lse one element into their buffers, K and V one cache."""
    rng = np.random.default_rng(53)
    B, H, T, d = 2, 4, 2, 64
    c = Cache(capi, rng, B, 2, 300, d, [300, 41])
    c.vc, c.vs = c.kc, c.ks
    c.upload()
    q = normal(rng, (B, H, T, d), dtype)
    f, e = capi.DeviceBuffer.from_numpy, capi.DeviceBuffer.ITEM[dtype]
    qb, o = f(np.append(9.0, q.ravel()).astype(np.float32), dtype), f(np.full(q.size + 2, 77.0, np.float32), dtype)
    lse = f(np.full(B * H * T + 2, 77.0, np.float32))
    kc, ks = c.dev[:2]
    capi.lib().call("tt_attn_decode_mxfp4", capi.TT_BF16 if dtype == "bf16" else capi.TT_F32, qb.ptr + e, kc.ptr, ks.ptr, kc.ptr,
                    ks.ptr, c.len.ptr, o.ptr + e, lse.ptr + 4, B, H, 2, T, 300, d, 0.125, None)
    capi.lib().sync()
    o, lse = o.download(), lse.download()
    assert o[0] == o[-1] == lse[0] == lse[-1] == 77.0
    check_attention(c, q, dtype, 0.125, o[1:-1].reshape(q.shape), lse[1:-1].reshape(q.shape[:3]))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_calls_repeat_bit_for_bit(capi, dtype):
    """Split attention and products of every kind of tile, the same in every call."""
    rng = np.random.default_rng(54)
    c = Cache(capi, rng, 2, 4, 3000, 128, [3000, 1700]).upload()
    q = normal(rng, (2, 8, 2, 128), dtype)
    first = attend(capi, c, q, dtype, 0.1)
    for _ in range(3):
        again = attend(capi, c, q, dtype, 0.1)
        assert np.array_equal(again[0], first[0]) and np.array_equal(again[1], first[1])
    for m, n, k in ((3, 500, 2000), (300, 300, 1056), (700, 1025, 2049), (2900, 3001, 544)):
        (ac, as_), (bc, bs) = held(capi, rng.standard_normal((m, k))), held(capi, rng.standard_normal((n, k)))
        outs = []
        for _ in range(3):
            y = capi.DeviceBuffer((m, n), dtype)
            capi.gemm_mxfp4(k, 1.0, ac, as_, bc, bs, 0.0, y)
            capi.lib().sync()
            outs.append(y.download())
        assert np.array_equal(outs[1], outs[0]) and np.array_equal(outs[2], outs[0])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(3, 50, 97), (100, 70, 300), (30, 50, 3000), (600, 1101, 200)])
def test_layer_of_nan_and_infinite_inputs(capi, m, n, k, dtype):
    """Quantised in the product or before it: such an input makes its own row NaN, and an infinite bias its column infinite."""
    rng = np.random.default_rng(m + 1)
    x, w, bias = normal(rng, (m, k), dtype), rng.standard_normal((n, k)), normal(rng, (n,), dtype)
    x[0, k - 1], x[m - 1, 0], bias[3] = np.nan, -np.inf, np.inf
    wc, ws = held(capi, w)
    f, out = capi.DeviceBuffer.from_numpy, capi.DeviceBuffer((m, n), dtype)
    capi.fc_forward_mxfp4(f(x, dtype), wc, ws, f(bias, dtype), out)
    capi.lib().sync()
    got = out.download()
    assert np.isnan(got[[0, m - 1]]).all() and np.isposinf(got[1:-1, 3]).all()
    assert np.isfinite(np.delete(got[1:-1], 3, 1)).all()
