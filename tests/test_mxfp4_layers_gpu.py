"""GPU tests of the 4-bit layer functions and of Tensor_byte against the oracle.

Codes and scales are exact.  FcForwardMxfp4 and AttentionDecodeMxfp4 keep the
bounds of the calls that they make: k 2^-24 of the sum of magnitudes and the
store's half step for a product with its bias; for attention the error of a
score, (d + 4) 2^-24 sum |q| |k| scale, twice over in the weights, the weights'
two bf16 terms (2^-16) or three (2^-24), 2 (n + 4) 2^-24 for exp2 and the sums,
all of sum p |v|, and the store's half step."""
import numpy as np
import pytest

from oracle import attn_oracle as orc
from oracle import mxfp4_oracle as mx

pytestmark = pytest.mark.gpu
HALF = {"float": 2.0 ** -24, "bf16": 2.0 ** -8}
TERMS = {"float": 2.0 ** -24, "bf16": 2.0 ** -16}
U = 2.0 ** -24


@pytest.fixture(scope="module")
def mods():
    import myLayer
    import myTensor

    assert myTensor.device_count() >= 1, "no HIP device visible"
    return myTensor, myLayer


def normal(rng, shape, name):
    x = rng.standard_normal(shape).astype(np.float32)
    return orc.bf16_round(x) if name == "bf16" else x


def new(mt, *shape):
    return mt.Tensor_byte(list(shape), "gpu").zeros()


def test_bytes_move_between_devices(mods):
    mt, _ = mods
    x = np.random.default_rng(1).integers(0, 256, (3, 5, 7), dtype=np.uint8)
    t = mt.Tensor_byte(x, "gpu")
    assert np.array_equal(t.numpy(), x) and np.array_equal(t[2].numpy(), x[2])
    assert np.array_equal(mt.Tensor_byte(t).cpu().numpy(), x)
    assert np.array_equal(mt.Tensor_byte(x, "cpu").gpu().numpy(), x)
    assert t.resize([2, 3]).get_data() == x.reshape(-1)[:6].tolist()
    assert t.zeros().get_data() == [0] * 6
    with pytest.raises(ValueError, match="no arithmetic"):
        t + t


@pytest.mark.parametrize("name", ["float", "bf16"])
@pytest.mark.parametrize("shape", [(5,), (3, 64), (2, 3, 33), (0, 40), (4, 0)])
def test_quantize_and_back(mods, shape, name):
    mt, ml = mods
    T = getattr(mt, "Tensor_" + name)
    x = normal(np.random.default_rng(2), shape, name)
    codes, scales, y = mt.Tensor_byte([1], "gpu"), mt.Tensor_byte([1], "gpu"), T([1], "gpu")
    ml.QuantizeMxfp4(T(x.reshape(-1), "gpu").resize(list(shape)) if x.size else T(list(shape), "gpu"), codes, scales)
    rc, rs = mx.quantize(x) if x.size else (np.zeros((*shape[:-1], 16 * mx.blocks(shape[-1])), np.uint8),
                                            np.zeros((*shape[:-1], mx.blocks(shape[-1])), np.uint8))
    assert codes.get_shape() == list(rc.shape) and scales.get_shape() == list(rs.shape)
    ml.DequantizeMxfp4(codes, scales, y, shape[-1])
    assert y.get_shape() == list(shape)
    if x.size:
        assert np.array_equal(codes.numpy(), rc) and np.array_equal(scales.numpy(), rs)
        assert np.array_equal(y.numpy().astype(np.float64), mx.dequantize(rc, rs, shape[-1]))


@pytest.mark.parametrize("name", ["float", "bf16"])
@pytest.mark.parametrize("batch,fin,fout,scalar", [((1,), 96, 40, False), ((2, 11), 70, 33, True), ((), 784, 100, False),
                                                   ((0,), 64, 8, False), ((3,), 64, 0, False), ((3,), 0, 8, False)])
def test_fc_with_its_weight_laid_out_once(mods, batch, fin, fout, scalar, name):
    mt, ml = mods
    T = getattr(mt, "Tensor_" + name)
    rng = np.random.default_rng(fin + fout)
    x, w = normal(rng, (*batch, fin), name), normal(rng, (fin, fout), name)
    b = normal(rng, (1 if scalar else fout,), name)

    def held(a):
        return T(list(a.shape), "gpu", a.reshape(-1).tolist())

    wc, ws, out = mt.Tensor_byte([1], "gpu"), mt.Tensor_byte([1], "gpu"), T([1], "gpu")
    ml.QuantizeMxfp4(held(w), wc, ws, transposed=True)
    assert wc.get_shape() == [fout, 16 * mx.blocks(fin)]
    ml.FcForwardMxfp4(held(x), out, wc, ws, held(b))
    assert out.get_shape() == [*batch, fout]
    if out.Size() == 0:
        return
    if fin:
        xv = mx.dequantize(*mx.quantize(x), fin)
        wv = mx.dequantize(*mx.quantize(np.ascontiguousarray(w.T)), fin)
        ref, mag = xv @ wv.T, np.abs(xv) @ np.abs(wv.T)
    else:
        ref, mag = np.zeros((*batch, fout)), np.zeros((*batch, fout))
    ref, mag = ref + b, mag + np.abs(b)
    assert (np.abs(out.numpy() - ref) <= (fin + 1) * U * mag * (1 + HALF[name]) + HALF[name] * np.abs(ref)).all()


@pytest.mark.parametrize("name", ["float", "bf16"])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_a_prompt_and_its_tokens(mods, d, name):
    """A layer's weights in 4 bits give q, k and v of a padded batch of prompts and
    of the tokens after them; the cache takes each step's keys and its attention
    is followed by an output projection."""
    mt, ml = mods
    T = getattr(mt, "Tensor_" + name)
    rng = np.random.default_rng(d)
    B, H, Hkv, cap, E, first = 3, 4, 2, 40, 48, 9
    scale = float(np.float32(d ** -0.5))
    w = {n: normal(rng, (E if n != "o" else H * d, (H if n == "q" else Hkv) * d if n != "o" else E), name) * 0.25
         for n in "qkvo"}
    held = {}
    for n in "qkvo":
        held[n] = (mt.Tensor_byte([1], "gpu"), mt.Tensor_byte([1], "gpu"))
        ml.QuantizeMxfp4(T(w[n], "gpu"), *held[n], transposed=True)
    zero = T([1], "gpu").zeros()
    kc, ks, vc, vs = new(mt, B, Hkv, cap, d // 2), new(mt, B, Hkv, cap, d // 32), \
        new(mt, B, Hkv, cap, d // 2), new(mt, B, Hkv, cap, d // 32)
    ref = {n: (np.zeros((B, Hkv, cap, d // 2), np.uint8), np.zeros((B, Hkv, cap, d // 32), np.uint8)) for n in "kv"}
    lengths = np.array([first, 4, 0], np.int32)
    for step, tokens in enumerate((first, 1, 1, 2)):
        if step:
            lengths = np.where(lengths > 0, lengths + tokens, 0).astype(np.int32)
        x = T(normal(rng, (B, tokens, E), name), "gpu")
        proj = {}
        for n in "qkv":
            y = T([1], "gpu")
            ml.FcForwardMxfp4(x, y, *held[n], zero)
            heads = H if n == "q" else Hkv
            proj[n] = np.ascontiguousarray(y.numpy().reshape(B, tokens, heads, d).transpose(0, 2, 1, 3))
        n = mt.Tensor_int([B], "gpu", lengths.tolist())
        ml.KvAppendMxfp4(T(proj["k"], "gpu"), T(proj["v"], "gpu"), kc, ks, vc, vs, n)
        for i in "kv":
            ref[i] = mx.append(*ref[i], proj[i], lengths)
        for t, r in zip((kc, ks, vc, vs), (*ref["k"], *ref["v"])):
            assert np.array_equal(t.numpy(), r)
        out = T([1], "gpu")
        ml.AttentionDecodeMxfp4(T(proj["q"], "gpu"), kc, ks, vc, vs, n, out, scale)
        assert out.get_shape() == [B, H, tokens, d]
        k, v = (mx.dequantize(*ref[i], d) for i in "kv")
        o, _, mag, smax = mx.decode(proj["q"], k, v, lengths, scale)
        e = (d + 4) * U * smax[..., None]
        tol = (2 * e + TERMS[name] + 2 * (cap + 4) * U) * mag
        assert (np.abs(out.numpy() - o) <= tol * (1 + HALF[name]) + HALF[name] * np.abs(o)).all()
        assert (out.numpy()[2] == 0).all()
        y, flat = T([1], "gpu"), np.ascontiguousarray(out.numpy().transpose(0, 2, 1, 3)).reshape(B, tokens, H * d)
        ml.FcForwardMxfp4(T(flat, "gpu"), y, *held["o"], zero)
        fv = mx.dequantize(*mx.quantize(flat), H * d)
        wv = mx.dequantize(*mx.quantize(np.ascontiguousarray(w["o"].T)), H * d)
        r, m = fv @ wv.T, np.abs(fv) @ np.abs(wv.T)
        assert (np.abs(y.numpy() - r) <= (H * d + 1) * U * m * (1 + HALF[name]) + HALF[name] * np.abs(r)).all()


def test_refusals(mods):
    mt, ml = mods
    F = mt.Tensor_float
    x, y = F([2, 64], "gpu").zeros(), F([1], "gpu")
    c, s = new(mt, 8, 32), new(mt, 8, 2)
    b = F([8], "gpu").zeros()
    n = mt.Tensor_int([1], "gpu").zeros()

    def refused(match, f):
        with pytest.raises(ValueError, match=match):
            f()

    refused("rank 2", lambda: ml.QuantizeMxfp4(F([2, 3, 4], "gpu"), c, s, transposed=True))
    refused("same tensor", lambda: ml.QuantizeMxfp4(x, c, c))
    refused("16 bytes", lambda: ml.DequantizeMxfp4(new(mt, 8, 31), s, y, 64))
    refused("blocks of 32", lambda: ml.DequantizeMxfp4(c, s, y, 65))
    refused("blocks of 32", lambda: ml.DequantizeMxfp4(c, s, y, 32))
    refused("blocks of 32", lambda: ml.DequantizeMxfp4(c, s, y, -1))
    refused("last axis", lambda: ml.FcForwardMxfp4(F([2, 65], "gpu"), y, c, s, b))
    refused("bias", lambda: ml.FcForwardMxfp4(x, y, c, s, F([7], "gpu")))
    refused("rank 2", lambda: ml.FcForwardMxfp4(x, y, new(mt, 32), new(mt, 2), b))
    refused("same tensor", lambda: ml.FcForwardMxfp4(x, x, c, s, b))
    refused("same tensor", lambda: ml.FcForwardMxfp4(x, b, c, s, b))
    kc, ks, vc, vs = new(mt, 1, 2, 4, 32), new(mt, 1, 2, 4, 2), new(mt, 1, 2, 4, 32), new(mt, 1, 2, 4, 2)
    k, q = F([1, 2, 1, 64], "gpu").zeros(), F([1, 4, 1, 64], "gpu").zeros()
    refused("lengths", lambda: ml.KvAppendMxfp4(k, k, kc, ks, vc, vs, mt.Tensor_int([2], "gpu")))
    refused("B, Hkv or d", lambda: ml.KvAppendMxfp4(q, q, kc, ks, vc, vs, n))
    refused("same shape", lambda: ml.KvAppendMxfp4(k, q, kc, ks, vc, vs, n))
    refused("same shape", lambda: ml.KvAppendMxfp4(k, k, kc, ks, new(mt, 1, 2, 5, 32), new(mt, 1, 2, 5, 2), n))
    refused("same tensor", lambda: ml.KvAppendMxfp4(k, k, kc, ks, kc, vs, n))
    refused("rank 4", lambda: ml.KvAppendMxfp4(x, x, kc, ks, vc, vs, n))
    refused("head dim", lambda: ml.AttentionDecodeMxfp4(F([1, 2, 1, 256], "gpu"), new(mt, 1, 2, 4, 128),
                                                        new(mt, 1, 2, 4, 8), new(mt, 1, 2, 4, 128),
                                                        new(mt, 1, 2, 4, 8), n, y, 0.1))
    refused("head dim", lambda: ml.AttentionDecodeMxfp4(F([1, 2, 1, 96], "gpu"), new(mt, 1, 2, 4, 48),
                                                        new(mt, 1, 2, 4, 3), new(mt, 1, 2, 4, 48),
                                                        new(mt, 1, 2, 4, 3), n, y, 0.1))
    refused("B or d", lambda: ml.AttentionDecodeMxfp4(F([1, 4, 1, 32], "gpu"), kc, ks, vc, vs, n, y, 0.1))
    refused("multiple", lambda: ml.AttentionDecodeMxfp4(F([1, 3, 1, 64], "gpu"), kc, ks, vc, vs, n, y, 0.1))
    refused("same tensor", lambda: ml.AttentionDecodeMxfp4(q, kc, ks, vc, vs, n, q, 0.1))
    assert all((t.numpy() == 0).all() for t in (x, k, q, c, s, kc, ks, vc, vs))
