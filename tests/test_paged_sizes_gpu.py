"""GPU tests of the paged cache at the sizes where its kernels change: appends of many
sequences, whose workgroups take several heads one after another, and reads back of
more than the caches hold.  A sample of the sequences goes against the float64 oracle;
all of them have the bits that appends of a few sequences, a head a workgroup, give.
Then every code of an 8-bit cache through a decode, and caches whose memory was NaN.

The bounds are those of test_paged_gpu.py."""
import numpy as np
import pytest

from oracle import paged_oracle as po
from test_norm_rope_gpu import EPS, FREQ, HALF, U, normal, pairs
from test_paged_gpu import KINDS, Cache, capi  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu
CUS = 256


def heads_of_a_workgroup(B, T, page, Hkv):
    """The rule of the 8-bit append: eight heads, fewer where there would be fewer than four workgroups a CU."""
    pages, heads = B * ((T + page - 2) // page + 1), min(Hkv, 8)
    while heads > 1 and 2 * pages * -(-Hkv // heads) < 4 * CUS:
        heads = (heads + 1) // 2
    return heads


def dirty(c):
    """All bits of the pools set: NaN in every type, and the largest byte of a scale."""
    for b in (*c.dev.values(), *(s for s in c.scale.values() if s)):
        b.L.call("tt_memset", b.ptr, 255, b.nbytes)


def raw(b):
    return b.download_bytes().view(np.uint8)


@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("d,page,rot,inter,Hkv", [(64, 64, 64, False, 11), (64, 128, 32, True, 5), (128, 64, 96, True, 11),
                                                  (128, 128, 128, False, 9)])
def test_appends_of_many_sequences(capi, d, page, rot, inter, Hkv, dtype, cache):  # noqa: F811
    """Prompts, then tokens into pages that they filled in part, whose values grow, then one token each."""
    rng = np.random.default_rng(d + page + rot)
    B, first = 260 if Hkv < 8 else 136, page - 12
    c, few = (Cache(capi, dtype, cache, B, Hkv, page, 2, d, np.random.default_rng(1)) for _ in range(2))
    dirty(c), dirty(few)
    sample = [0, 1, B // 3, B - 2, B - 1]
    ref = po.Cache(c.npages, Hkv, page, d, c.table[sample], cache == "u8")
    lengths = rng.integers(1, first + 1, B).astype(np.int32)
    lengths[[1, 7]], lengths[[0, B - 1]] = 0, first  # idle slots, and the longest
    freq = FREQ[rot]
    put = lambda a, t=dtype: capi.DeviceBuffer.from_numpy(np.ascontiguousarray(a), t)  # noqa: E731
    assert np.array_equal(c.table, few.table)
    mag = {}
    for step, T in enumerate((first, 31, 1)):
        if step:
            lengths = np.where(lengths > 0, lengths + T, 0).astype(np.int32)
        # several heads a workgroup; the last of them fewer, in the last step at least
        want = heads_of_a_workgroup(B, T, page, Hkv)
        assert want > (3 if step < 2 else 1) and (Hkv % want != 0 or step < 2)
        w = ((1 + 0.1 * normal(rng, (d,), "f32")) * 3.0 ** step).astype(np.float32)
        k, v = normal(rng, (B, T, Hkv, d), dtype), normal(rng, (B, T, Hkv, d), dtype, 4.0 ** step)
        W, F = put(w, "f32"), put(freq, "f32")
        capi.kv_append_paged(put(k), put(v), c.dev["k"], c.dev["v"], c.tab, put(lengths, "i32"), W, F, EPS, None, inter, True,
                             **c.scales())
        for at in range(0, B, 4):
            assert heads_of_a_workgroup(4, T, page, Hkv) == 1
            capi.kv_append_paged(put(k[at:at + 4]), put(v[at:at + 4]), few.dev["k"], few.dev["v"], put(c.table[at:at + 4], "i32"),
                                 put(lengths[at:at + 4], "i32"), W, F, EPS, None, inter, True, **few.scales())
        capi.lib().sync()
        ks, vs, ls = (np.swapaxes(k[sample], 1, 2), np.swapaxes(v[sample], 1, 2), lengths[sample])
        ref.append("k", po.norm_rope(ks, w, EPS, po.positions(len(sample), T, lengths=ls), freq, inter), ls)
        ref.append("v", vs.astype(np.float64), ls)
        m = pairs(po.norm(ks, w, EPS), rot, inter)
        for i in range(len(sample)):
            for t in range(T):
                if ls[i] - T + t >= 0:
                    mag[i, int(ls[i]) - T + t] = m[i, :, t]
        for n in "kv":  # whole pools: the rows that no token went to among them
            assert np.array_equal(raw(c.dev[n]), raw(few.dev[n]))
            if cache == "u8":
                assert np.array_equal(c.scale[n].download(), few.scale[n].download())
    for n in "kv":
        got = c.dev[n].download_bytes() if cache == "u8" else c.dev[n].download()
        for i, b in enumerate(sample):
            for j in range(2 * page):
                p, row = c.table[b, j // page], j % page
                if j >= lengths[b]:  # as it was
                    assert (got[p, :, row] == 255).all() if cache == "u8" else np.isnan(got[p, :, row]).all()
                elif cache == "u8" or n == "v":
                    assert np.array_equal(got[p, :, row], ref.pool[n][p, :, row])
                else:
                    x = ref.pool[n][p, :, row]
                    assert (np.abs(got[p, :, row] - x) <= (d / 2 + 16) * U * mag[i, j] * (1 + HALF[dtype]) + HALF[dtype] * np.abs(x)).all()
            if cache == "u8":
                at = c.table[b, :-(-int(lengths[b]) // page)]
                assert np.array_equal(c.scale[n].download()[at], ref.scale[n][at])


@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("d", [32, 64, 128])
def test_reads_back_past_the_caches(capi, d, dtype, cache):  # noqa: F811
    """More than 64 MiB of rows, of sequences of several lengths, one of them with a page that is not there."""
    rng = np.random.default_rng(d)
    B, Hkv, page, L = 3, 7, 32, 3210 * (128 // d) * (1 if dtype == "f32" else 2)
    assert 2 * B * Hkv * L * d * (4 if dtype == "f32" else 2) > 2 ** 26
    width = -(-L // page)
    c = Cache(capi, dtype, cache, B, Hkv, page, width, d, rng)
    t = c.table.copy()
    t[1, 3] = -1
    c.set(t)
    lengths = [L, L - 1000, 1]
    shape = (c.npages, Hkv, page, d)
    host = {}
    for n in "kv":
        if cache == "u8":
            x, byte = rng.integers(0, 127, shape, dtype=np.uint8), rng.integers(60, 200, shape[:2], dtype=np.uint8)
            c.dev[n].upload(x), c.scale[n].upload(byte)
            host[n] = po.E4_GRID.astype(np.float32)[x] * np.ldexp(np.float32(1), byte.astype(np.int32) - 127)[:, :, None, None]
        else:
            host[n] = normal(rng, shape, dtype)
            c.dev[n].upload(host[n])
    c.lengths.upload(np.asarray(lengths, np.int32))
    out = {n: capi.DeviceBuffer((B, Hkv, L, d), dtype) for n in "kv"}
    for b in out.values():
        b.L.call("tt_memset", b.ptr, 255, b.nbytes)
    capi.kv_gather_paged(c.dev["k"], c.dev["v"], c.tab, c.lengths, out["k"], out["v"], **c.scales())
    capi.lib().sync()
    for n in "kv":
        got = out[n].download()
        for b, size in enumerate(lengths):
            j = np.arange(size)
            j = j[t[b, j // page] >= 0]
            ref = np.full((Hkv, L, d), np.nan, np.float32)
            ref[:, j] = host[n][t[b, j // page], :, j % page].swapaxes(0, 1)
            assert np.array_equal(got[b], ref, equal_nan=True)


# ------------------------------------------------------------------ every code through a decode

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_every_code_of_v_through_a_decode(capi, d, dtype):  # noqa: F811
    """One key a sequence: o is its row of V, of all 256 codes under all scales, values that are subnormal in
    bf16 among them, exactly."""
    per, page = 256 // d, 16
    npages = 244 * per
    codes = np.zeros((npages, 1, page, d), np.uint8)
    codes[:, 0, 0] = np.tile(np.arange(256, dtype=np.uint8).reshape(per, d), (244, 1))
    codes[:, 0, 1:] = 127  # rows that no token sees
    byte = np.repeat(np.arange(3, 247, dtype=np.uint8), per)[:, None]
    f = capi.DeviceBuffer.from_numpy
    K, KS, V, VS = f(np.zeros_like(codes), "u8"), f(np.full_like(byte, 127), "u8"), f(codes, "u8"), f(byte, "u8")
    tab, n = f(np.arange(npages, dtype=np.int32)[:, None], "i32"), f(np.ones(npages, np.int32), "i32")
    q = f(np.ones((npages, 1, 1, d), np.float32), dtype)
    o, lse = capi.DeviceBuffer((npages, 1, 1, d), dtype), capi.DeviceBuffer((npages, 1, 1))
    capi.attn_decode_paged(q, K, V, tab, n, o, lse, 0.25, k_scales=KS, v_scales=VS)
    capi.lib().sync()
    ref = po.decode(codes[:, 0, 0], byte.astype(int))
    assert np.array_equal(o.download()[:, 0, 0], ref, equal_nan=True)
    assert (lse.download() == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_every_code_of_k_through_a_decode(capi, d, dtype):  # noqa: F811
    """One key a sequence, of one code that is not zero, and q a power of two there: lse is their product."""
    byte, code = (a.reshape(-1) for a in np.meshgrid(np.arange(3, 247), np.r_[0:127, 128:255], indexing="ij"))
    B, page = len(byte), 16
    at = (7 * code + byte) % d
    row = np.arange(B)
    codes = np.zeros((B, 1, page, d), np.uint8)
    codes[row, 0, 0, at] = code
    e = np.clip(127 - byte, -100, 120)  # so that the product is of fp32's normal range
    q = np.zeros((B, 1, 1, d), np.float32)
    q[row, 0, 0, at] = np.ldexp(np.float32(1), e)
    f = capi.DeviceBuffer.from_numpy
    K, KS = f(codes, "u8"), f(byte.astype(np.uint8)[:, None], "u8")
    tab, n = f(np.arange(B, dtype=np.int32)[:, None], "i32"), f(np.ones(B, np.int32), "i32")
    V = f(np.full_like(codes, 0x38), "u8")  # ones
    VS, Q = f(np.full((B, 1), 127, np.uint8), "u8"), f(q, dtype)
    o, lse = capi.DeviceBuffer((B, 1, 1, d), dtype), capi.DeviceBuffer((B, 1, 1))
    capi.attn_decode_paged(Q, K, V, tab, n, o, lse, 1.0, k_scales=KS, v_scales=VS)
    capi.lib().sync()
    ref = po.decode(code.astype(np.uint8), byte) * np.ldexp(1.0, e)
    # the product is exact; log2 e, the product with it, ln 2 and the product with that are half a step each
    assert (np.abs(lse.download()[:, 0, 0] - ref) <= 4.5 * U * np.abs(ref)).all()
    assert (o.download() == 1).all()


# ------------------------------------------------------------------ memory that was NaN

@pytest.mark.parametrize("dtype,cache", [("f32", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("page,d", [(16, 32), (32, 128), (128, 64)])
def test_pools_that_held_nan(capi, page, d, dtype, cache):  # noqa: F811
    """Prompts and tokens into 16- and 32-bit pools of NaN: rows without a token stay, and attention uses none."""
    rng = np.random.default_rng(page)
    B, Hkv, H = 3, 2, 4
    c = Cache(capi, dtype, cache, B, Hkv, page, 3, d, rng)
    dirty(c)
    lengths = np.array([page + 5, page // 2, 0], np.int32)
    for n in "kv":
        c.ref.pool[n][:] = np.nan
    for step, T in enumerate((page + 5, 1, 4)):
        if step:
            lengths = np.where(lengths > 0, lengths + T, 0).astype(np.int32)
        k, v = normal(rng, (B, Hkv, T, d), dtype), normal(rng, (B, Hkv, T, d), dtype)
        c.append(k, v, lengths, tokens_first=step == 1)
        for n in "kv":
            assert np.array_equal(c.dev[n].download(), c.ref.pool[n], equal_nan=True)
        c.check_attention(normal(rng, (B, H, T, d), dtype), lengths, 0.2)
