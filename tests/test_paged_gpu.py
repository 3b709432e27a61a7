"""GPU tests of the paged cache against the float64 oracle: append, read back and
attention, in 32, 16 and 8 bits.

Codes, scales and V are exact.  K in 32 or 16 bits keeps the bound of the rotation:
(d / 2 + 16) u (|a| + |b|) over a turned pair and the store's half step, u = 2^-24.
Attention: a score is off by (d + 8) u sum |q| |k| scale, twice over in the weights;
the weights keep 2^-17 (bf16 calls) or 2^-24 of themselves where they meet V; exp2
and the sums of n keys add 2 (n + 8) u; all of sum p |v|, and the store's half step.
lse: the scores' bound, (n + 8) u for the sum, and 4 u (|lse| + 1) for the logarithm."""
import os
import subprocess
import sys

import numpy as np
import pytest

from oracle import attn_oracle as orc
from oracle import paged_oracle as po
from test_capture_gpu import Capture
from test_norm_rope_gpu import EPS, FREQ, HALF, U, normal, pairs

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TERMS = {"f32": 2.0 ** -24, "bf16": 2.0 ** -17}
KINDS = [("f32", "f32"), ("bf16", "bf16"), ("f32", "u8"), ("bf16", "u8")]


@pytest.fixture(scope="module")
def capi():
    import tt_capi

    assert tt_capi.lib().device_count() >= 1, "no HIP device visible"
    tt_capi.lib().call("tt_init", 0)
    return tt_capi


class Cache:
    """Pools on the device beside the oracle's."""

    def __init__(self, capi, dtype, cache, B, Hkv, page, width, d, rng, spare=2, fill=0):
        self.T, self.dtype, self.cache, self.d, self.Hkv = capi, dtype, cache, d, Hkv
        self.npages = B * width + spare
        self.table = rng.permutation(self.npages)[:B * width].reshape(B, width).astype(np.int32)
        self.dev = {n: capi.DeviceBuffer((self.npages, Hkv, page, d), cache) for n in "kv"}
        self.scale = {n: capi.DeviceBuffer((self.npages, Hkv), "u8") for n in "kv"} if cache == "u8" else {"k": None, "v": None}
        for b in (*self.dev.values(), *(s for s in self.scale.values() if s)):
            b.L.call("tt_memset", b.ptr, fill, b.nbytes)
        self.lengths = capi.DeviceBuffer((B,), "i32")
        self.set(self.table)
        self.ref = po.Cache(self.npages, Hkv, page, d, self.table, cache == "u8")
        if fill and cache == "u8":
            for n in "kv":
                self.ref.pool[n][:] = fill
                self.ref.scale[n][:] = fill

    def set(self, table):
        self.table = table
        self.tab = self.T.DeviceBuffer.from_numpy(table, "i32")
        if hasattr(self, "ref"):
            self.ref.table = np.asarray(table, np.int32)

    def scales(self):
        return dict(k_scales=self.scale["k"], v_scales=self.scale["v"])

    def append(self, k, v, lengths, w=None, freq=None, positions=None, inter=False, tokens_first=False, stream=None):
        """Into both; k and v [B, Hkv, T, d]."""
        put = lambda a: self.T.DeviceBuffer.from_numpy(np.ascontiguousarray(np.swapaxes(a, 1, 2)) if tokens_first else a, self.dtype)  # noqa: E731
        some = lambda a, t: None if a is None else self.T.DeviceBuffer.from_numpy(a, t)  # noqa: E731
        self.lengths.upload(np.asarray(lengths, np.int32))
        self.T.kv_append_paged(put(k), put(v), self.dev["k"], self.dev["v"], self.tab, self.lengths, some(w, "f32"),
                               some(freq, "f32"), EPS, some(positions, "i32"), inter, tokens_first, stream=stream,
                               **self.scales())
        self.T.lib().sync()
        pos = po.positions(k.shape[0], k.shape[2], given=positions, lengths=lengths)
        self.ref.append("k", po.norm_rope(k, w, EPS, pos, freq, inter), lengths)
        self.ref.append("v", v.astype(np.float64), lengths)

    def check(self, w=None, freq=None):
        """Codes and scales are the oracle's where it has tokens; values within the rotation's bound."""
        for n in "kv":
            got = self.dev[n].download_bytes() if self.cache == "u8" else self.dev[n].download()
            ref = self.ref.pool[n]
            if self.cache == "u8":
                got, ref = (np.where(a & 127 == 127, 127, a) for a in (got, ref))  # NaN has two codes
                assert np.array_equal(got, ref), np.argwhere(got != ref)[:5]
                assert np.array_equal(self.scale[n].download(), self.ref.scale[n])
            elif n == "v" or (w is None and freq is None):
                assert np.array_equal(got, ref)
            else:  # |a| + |b| of a turned pair is at most sqrt 2 of the pair it came from, as of the one it became
                mag = np.sqrt(2.0) * pairs(ref, self.d, False)
                if freq is not None and 2 * len(freq) != self.d:
                    mag = np.abs(ref).max(-1, keepdims=True) * 2 + 0 * ref
                bound = (self.d / 2 + 16) * U * mag * (1 + HALF[self.dtype]) + HALF[self.dtype] * np.abs(ref)
                assert (np.abs(got - ref) <= bound).all()

    def adopt(self):
        """The oracle's pools as the device's (16- and 32-bit K is rounded there)."""
        if self.cache != "u8":
            for n in "kv":
                self.ref.pool[n][:] = self.dev[n].download()

    def attend(self, q, lengths, scale, lse=True, stream=None):
        B, H, T, d = q.shape
        self.lengths.upload(np.asarray(lengths, np.int32))
        o = self.T.DeviceBuffer.from_numpy(np.full(q.shape, 7.0, np.float32), self.dtype)
        L = self.T.DeviceBuffer.from_numpy(np.full((B, H, T), 7.0, np.float32)) if lse else None
        self.T.attn_decode_paged(self.T.DeviceBuffer.from_numpy(q, self.dtype), self.dev["k"], self.dev["v"], self.tab,
                                 self.lengths, o, L, scale, stream=stream, **self.scales())
        self.T.lib().sync()
        if stream:
            self.T.lib().call("tt_stream_sync", stream)
        return o.download(), L.download() if lse else None

    def check_attention(self, q, lengths, scale, got=None):
        d, n = q.shape[-1], max(1, max(int(x) for x in lengths))
        o, lse = got or self.attend(q, lengths, scale)
        ro, rl, mag, score = self.ref.attend(q, lengths, scale)
        rel = 2 * (d + 8) * U * score + TERMS[self.dtype] + 2 * (n + 8) * U
        bound = rel[..., None] * mag * (1 + HALF[self.dtype]) + HALF[self.dtype] * np.abs(ro)
        assert (np.abs(o - ro) <= bound).all(), np.max(np.abs(o - ro) - bound)
        none = rl == -np.inf
        assert (lse[none] == -np.inf).all() and (o[none] == 0).all()
        off = np.abs(lse[~none] - rl[~none])
        assert (off <= (d + 8) * U * score[~none] + (n + 8) * U + 4 * U * (np.abs(rl[~none]) + 1)).all()


def filled(capi, dtype, cache, B, Hkv, page, d, lengths, rng, width=None, **kw):
    """A cache that holds `lengths` normal keys of each sequence."""
    width = width or -(-max(max(lengths), 1) // page)
    c = Cache(capi, dtype, cache, B, Hkv, page, width, d, rng, **kw)
    n = max(max(lengths), 1)
    c.append(normal(rng, (B, Hkv, n, d), dtype), normal(rng, (B, Hkv, n, d), dtype), lengths)
    c.adopt()
    return c


# ------------------------------------------------------------------ append

@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_prompts_and_tokens(capi, d, page, dtype, cache):
    """Prompts padded on the left, then tokens one, two and more at a time, each norm, rotated and growing;
    the pools hold 0xff before, which is NaN in every type."""
    rng = np.random.default_rng(d + page)
    B, Hkv, width = 3, 2, 3
    c = Cache(capi, dtype, cache, B, Hkv, page, width, d, rng, fill=255 if cache == "u8" else 0)
    w, freq = 1 + 0.1 * normal(rng, (d,), "f32"), FREQ[d]
    lengths = np.array([page + 5, page // 2, 0], np.int32)
    for step, T in enumerate((page + 5, 1, 1, 2, page - 3)):
        if step:
            lengths = np.where(lengths > 0, lengths + T, 0).astype(np.int32)
        # V grows, so that pages are scaled again; K is normed
        k, v = normal(rng, (B, Hkv, T, d), dtype), normal(rng, (B, Hkv, T, d), dtype, 4.0 ** step)
        c.append(k, v, lengths, w, freq, tokens_first=step % 2 == 1)
    c.check(w, freq)


@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("weight,rot", [(True, 32), (False, 64), (True, 0), (False, 0)])
def test_append_norm_and_rotation(capi, weight, rot, inter, dtype, cache):
    """Each with and without, at positions that are not the keys' own."""
    rng = np.random.default_rng(rot + inter)
    B, Hkv, T, page, d = 2, 3, 21, 16, 64
    c = Cache(capi, dtype, cache, B, Hkv, page, 2, d, rng)
    w, freq = normal(rng, (d,), "f32") if weight else None, FREQ[rot] if rot else None
    given = rng.integers(0, 200000, (B, T)).astype(np.int32)
    k, v = normal(rng, (B, Hkv, T, d), dtype), normal(rng, (B, Hkv, T, d), dtype)
    c.append(k, v, [21, 17], w, freq, given, inter)
    if cache != "u8" and (weight or rot):
        pos = po.positions(B, T, given=given)
        mag = pairs(po.norm(k, w, EPS), rot, inter)
        got, bound = c.dev["k"].download(), np.zeros((c.npages, Hkv, page, d))
        for b, n in enumerate((21, 17)):
            for j in range(n):
                bound[c.table[b, j // page], :, j % page] = mag[b, :, T - n + j]
        ref = c.ref.pool["k"]
        assert pos is not None
        assert (np.abs(got - ref) <= (d / 2 + 16) * U * bound * (1 + HALF[dtype]) + HALF[dtype] * np.abs(ref)).all()
        c.ref.pool["k"][:] = got
    c.check()


@pytest.mark.parametrize("dtype,cache", KINDS)
def test_tokens_without_a_place(capi, dtype, cache):
    """Keys past the table, before its start and in pages that the pool does not have are not stored;
    all other rows stay as they are."""
    rng = np.random.default_rng(3)
    B, Hkv, T, page, d = 5, 2, 40, 16, 32
    c = Cache(capi, dtype, cache, B, Hkv, page, 2, d, rng)
    c.set(np.array([[0, 3], [-1, 5], [2, c.npages], [2 ** 31 - 1, 7], [1, -2 ** 31]], np.int32))
    k, v = normal(rng, (B, Hkv, T, d), dtype), normal(rng, (B, Hkv, T, d), dtype)
    for lengths in ([40, 40, 40, 40, 40], [32, 20, 70, 5, 2 ** 31 - 1], [-5, -2 ** 31, 0, 1, 33]):
        c.append(k, v, lengths)
        c.check()


def test_scales_of_pages(capi):
    """Largest values next to 448, all zero, subnormal, largest, and not finite."""
    rng = np.random.default_rng(4)
    B, Hkv, T, page, d = 1, 8, 16, 16, 32
    c = Cache(capi, "f32", "u8", B, Hkv, page, 1, d, rng, fill=255)
    k = normal(rng, (B, Hkv, T, d), "f32")
    k[0, 0] *= 448.0 / np.abs(k[0, 0]).max()
    k[0, 0].flat[np.abs(k[0, 0]).argmax()] = 448.0
    k[0, 1].flat[3] = np.nextafter(np.float32(448.0), np.float32(449.0))
    k[0, 2] = 0.0
    k[0, 3] = (rng.integers(1, 2 ** 20, (T, d)).astype(np.uint32)).view(np.float32)  # subnormal
    k[0, 4] = np.finfo(np.float32).max
    k[0, 4, 3] = -np.finfo(np.float32).max
    k[0, 5, 2, 7], k[0, 5, 9, 1], k[0, 5, 11, 30] = np.inf, -np.inf, np.nan
    k[0, 6] = np.nan
    k[0, 7] = -0.0
    c.append(k, k[:, ::-1].copy(), [16])
    c.check()
    assert list(c.scale["k"].download()[c.table[0, 0]][[0, 1, 2, 3, 4, 6]]) == [127, 128, 3, 3, 246, 3]


def test_ties_of_codes(capi):
    """Every value between two codes, and its neighbours, under a scale that the page's 448 fixes."""
    grid = po.E4_GRID
    mid = ((grid[:-1] + grid[1:]) / 2).astype(np.float32)
    x = np.concatenate([mid, np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(500)), grid.astype(np.float32)])
    x = np.concatenate([x, -x])
    T, d = 64, 32
    k = np.zeros((1, 1, T, d), np.float32)
    k.reshape(-1)[:len(x)] = x
    c = Cache(capi, "f32", "u8", 1, 1, 64, 1, d, np.random.default_rng(0))
    c.append(k, k * np.float32(2.0 ** 30), [T])
    c.check()
    assert c.scale["k"].download()[c.table[0, 0], 0] == 127 and c.scale["v"].download()[c.table[0, 0], 0] == 157


def test_pages_that_grow_far(capi):
    """Old tokens under a scale up to 2^243 smaller than the new one; a scale never shrinks with old tokens there."""
    rng = np.random.default_rng(5)
    c = Cache(capi, "f32", "u8", 1, 1, 32, 1, 64, rng)
    n = 0
    for std in (2.0 ** -120, 2.0 ** -110, 2.0 ** -100, 2.0 ** -99, 1.0, 0.5, 2.0, 2.0 ** 100, 1.0, 2.0 ** 120):
        n += 2
        x = normal(rng, (1, 1, 2, 64), "f32") * np.float32(std)
        c.append(x, -x, [n])
        c.check()
    c.append(x, x, [2])  # a sequence that begins again takes its page's scale from its own tokens
    c.check()


# ------------------------------------------------------------------ read back

@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("page,L", [(16, 50), (64, 33), (128, 200)])
def test_gather(capi, page, L, dtype, cache):
    rng = np.random.default_rng(page)
    B, Hkv, d = 4, 2, 64
    lengths = [50, 0, 33, 1]
    c = filled(capi, dtype, cache, B, Hkv, page, d, lengths, rng)
    t = c.table.copy()
    t[2, 0] = -1 if page == 16 else t[2, 0]
    c.set(t)
    c.lengths.upload(np.asarray([50, -3, 60, 1], np.int32))
    k, v = (capi.DeviceBuffer.from_numpy(np.full((B, Hkv, L, d), 3.0, np.float32), dtype) for _ in range(2))
    capi.kv_gather_paged(c.dev["k"], c.dev["v"], c.tab, c.lengths, k, v, **c.scales())
    capi.lib().sync()
    for n, out in (("k", k.download()), ("v", v.download())):
        for b, size in enumerate((50, 0, 60, 1)):
            end = min(size, L, c.table.shape[1] * page)
            rows, has = c.ref.rows(n, b, end)
            ref = np.full((Hkv, L, d), 3.0)
            ref[:, :end][:, has] = rows[:, has]
            assert np.array_equal(out[b], ref)


def test_every_code_reads_back(capi):
    """All 256 codes under all scales, into both types and through a decode of one key."""
    rng = np.random.default_rng(0)
    npages, d, page = 244, 64, 16
    codes = np.tile(np.arange(256, dtype=np.uint8), (npages, 1, 4)).reshape(npages, 1, page, d)
    byte = np.arange(3, 247, dtype=np.uint8)[:, None]
    K, S = capi.DeviceBuffer.from_numpy(codes, "u8"), capi.DeviceBuffer.from_numpy(byte, "u8")
    tab = capi.DeviceBuffer.from_numpy(rng.permutation(npages).astype(np.int32)[None], "i32")
    n = capi.DeviceBuffer.from_numpy(np.array([npages * page], np.int32), "i32")
    order = tab.download()[0]
    ref = po.decode(codes[order, 0].reshape(1, 1, -1, d), np.repeat(byte[order, 0].astype(int), page)[None, None, :, None])
    for dtype in ("f32", "bf16"):
        k, v = (capi.DeviceBuffer((1, 1, npages * page, d), dtype) for _ in range(2))
        capi.kv_gather_paged(K, K, tab, n, k, v, k_scales=S, v_scales=S)
        capi.lib().sync()
        for out in (k, v):
            assert np.array_equal(out.download(), ref, equal_nan=True)


# ------------------------------------------------------------------ attention

@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("H,Hkv,T", [(2, 2, 1), (8, 2, 3), (5, 1, 7)])
def test_decode(capi, H, Hkv, T, d, page, dtype, cache):
    """Lengths of none, one, fewer than the tokens, a page less and more, and several steps of every wave."""
    rng = np.random.default_rng(H + d + page)
    lengths = [0, 1, 5, page - 1, page, page + 1, 301]
    c = filled(capi, dtype, cache, len(lengths), Hkv, page, d, lengths, rng)
    q = normal(rng, (len(lengths), H, T, d), dtype)
    c.check_attention(q, lengths, float(np.float32(d ** -0.5)))
    c.check_attention(q, [x // 2 for x in lengths], -0.3)
    c.check_attention(q, [x + 2 for x in lengths[:-1]] + [2 ** 31 - 1] if page == 16 else lengths, 0.0)


@pytest.mark.parametrize("dtype,cache", KINDS)
def test_long_sequences_are_split(capi, dtype, cache):
    """Few heads: the keys go over many workgroups, more than a wave's 128 pages each; ragged, with an idle slot."""
    rng = np.random.default_rng(1)
    lengths, page, d = [9001, 0, 4500], 16, 64
    c = filled(capi, dtype, cache, 3, 1, page, d, lengths, rng)
    q = normal(rng, (3, 2, 2, d), dtype, 2.0)
    c.check_attention(q, lengths, 0.25)
    c.check_attention(q, [3, 9008, 100], 0.25)


@pytest.mark.parametrize("dtype,cache", KINDS)
def test_unsplit_sequences_of_many_pages(capi, dtype, cache):
    """Many heads, so that a wave goes through hundreds of pages of 16 itself."""
    rng = np.random.default_rng(2)
    B, Hkv, page, d, n = 64, 32, 16, 32, 2100
    width = -(-n // page)
    tab = np.stack([rng.permutation(width) for _ in range(B)]).astype(np.int32)  # sequences share their pages
    c = Cache(capi, dtype, cache, 1, Hkv, page, width, d, rng, spare=0)
    c.set(tab[:1])
    c.append(normal(rng, (1, Hkv, n, d), dtype), normal(rng, (1, Hkv, n, d), dtype), [n])
    c.adopt()
    c.lengths = capi.DeviceBuffer((B,), "i32")
    c.set(tab)
    lengths = [n - 13 * b for b in range(B)]
    q = normal(rng, (B, Hkv, 1, d), dtype)
    o, lse = c.attend(q, lengths, 0.2)
    for b in (0, 17, 63):  # each by itself in the oracle
        c.ref.table = tab[b:b + 1]
        c.check_attention(q[b:b + 1], lengths[b:b + 1], 0.2, (o[b:b + 1], lse[b:b + 1]))


@pytest.mark.parametrize("dtype,cache", KINDS)
def test_pages_that_the_pool_does_not_have(capi, dtype, cache):
    """Their keys are not seen, nor are those past the table."""
    rng = np.random.default_rng(3)
    B, Hkv, page, d = 4, 2, 16, 64
    c = filled(capi, dtype, cache, B, Hkv, page, d, [80] * B, rng)
    t = c.table.copy()
    t[0, 1], t[1, 0], t[1, 4], t[2] = -1, c.npages, 2 ** 31 - 1, -2 ** 31
    c.set(t)
    q = normal(rng, (B, 4, 3, d), dtype)
    for lengths in ([80, 80, 80, 80], [17, 16, 40, 81], [90, 1000, 2 ** 31 - 1, -1]):
        c.check_attention(q, lengths, 0.125)


@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("d", [32, 64, 128])
def test_values_that_are_not_finite(capi, d, dtype, cache):
    """NaN and infinities behind the sequence, in keys that some tokens do not see, and in seen keys: they
    reach the tokens that see them and no others."""
    rng = np.random.default_rng(d)
    page, T, n, H = 16, 4, 70, 2
    c = filled(capi, dtype, cache, 1, 1, page, d, [80], rng)
    q = normal(rng, (1, H, T, d), dtype)
    clean, _ = c.attend(q, [n], 0.2)
    at = lambda j: (c.table[0, j // page], 0, j % page)  # noqa: E731
    bad = {"u8": [127, 255], "f32": [np.nan, np.inf], "bf16": [np.nan, -np.inf]}[cache]

    def poison(keys, column=slice(None)):
        for m in "kv":
            host = c.dev[m].download_bytes() if cache == "u8" else c.dev[m].download()
            for i, j in enumerate(keys):
                host[at(j)][column] = bad[i % 2]
            c.dev[m].upload(host)

    keep = {m: c.dev[m].download_bytes() if cache == "u8" else c.dev[m].download() for m in "kv"}
    poison([70, 71, 75, 79])
    o, _ = c.attend(q, [n], 0.2)
    assert np.array_equal(o, clean)
    # V alone, one column of the two newest keys: tokens 0 and 1 do not see them
    for m in "kv":
        c.dev[m].upload(keep[m])
    host = keep["v"].copy()
    host[at(68)][3], host[at(69)][d - 1] = bad
    c.dev["v"].upload(host)
    o, _ = c.attend(q, [n], 0.2)
    assert np.array_equal(o[:, :, :2], clean[:, :, :2])
    rest = [i for i in range(d) if i not in (3, d - 1)]
    assert np.array_equal(o[:, :, 2:, rest], clean[:, :, 2:, rest])
    assert not np.isfinite(o[:, :, 2:, 3]).any() and np.isfinite(o[:, :, 2, d - 1]).all()
    assert not np.isfinite(o[:, :, 3, d - 1]).any()
    # a key far from the edge, which all see: that column alone
    host = keep["v"].copy()
    host[at(9)][7] = bad[1]
    c.dev["v"].upload(host)
    o, _ = c.attend(q, [n], 0.2)
    assert not np.isfinite(o[..., 7]).any()
    if cache != "u8":
        assert (o[..., 7] == bad[1]).all()
    assert np.array_equal(np.delete(o, 7, -1), np.delete(clean, 7, -1))
    # NaN keys in sight of the last token alone
    for m in "kv":
        c.dev[m].upload(keep[m])
    host = keep["k"].copy()
    host[at(69)] = bad[0]
    c.dev["k"].upload(host)
    o, _ = c.attend(q, [n], 0.2)
    assert np.array_equal(o[:, :, :3], clean[:, :, :3]) and np.isnan(o[:, :, 3]).all()



@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("n,H,T", [(77, 9, 5), (1500, 1, 3), (1500, 9, 5)])
def test_infinite_values_over_tiles_and_splits(capi, n, H, T, dtype, cache):
    """One column of a key that the last token alone sees, with several tiles of rows, splits, and splits merged by
    their last workgroup: the other tokens and columns keep their bits."""
    rng = np.random.default_rng(n + H)
    page, d = 32, 64
    c = filled(capi, dtype, cache, 2, 1, page, d, [n, n], rng)
    q = normal(rng, (2, H, T, d), dtype)
    clean, lse = c.attend(q, [n, n - 40], 0.2)
    host = c.dev["v"].download_bytes() if cache == "u8" else c.dev["v"].download()
    host[c.table[0, (n - 1) // page], 0, (n - 1) % page, 5] = 127 if cache == "u8" else np.inf
    c.dev["v"].upload(host)
    o, again = c.attend(q, [n, n - 40], 0.2)
    assert np.array_equal(again, lse) and np.array_equal(o[1], clean[1]) and np.array_equal(o[0, :, :-1], clean[0, :, :-1])
    assert not np.isfinite(o[0, :, -1, 5]).any()
    assert np.array_equal(np.delete(o[0, :, -1], 5, -1), np.delete(clean[0, :, -1], 5, -1))


@pytest.mark.parametrize("dtype,cache", KINDS)
def test_scores_of_minus_infinity(capi, dtype, cache):
    """A row all of whose keys score -inf has nothing to weigh: o = 0, lse = -inf; one key above it has all the weight."""
    rng = np.random.default_rng(11)
    c = filled(capi, dtype, cache, 1, 1, 32, 32, [40], rng)
    if cache == "u8":
        host = np.full(c.dev["k"].shape, 126, np.uint8)  # 448 under 2^119
        c.dev["k"].upload(host)
        c.scale["k"].upload(np.full(c.scale["k"].shape, 246, np.uint8))
    else:
        c.dev["k"].upload(np.full(c.dev["k"].shape, 2.0 ** 127, np.float32))
    q = np.full((1, 1, 1, 32), -4.0, np.float32)
    o, lse = c.attend(q, [40], 1.0)
    assert (o == 0).all() and lse[0, 0, 0] == -np.inf


@pytest.mark.parametrize("dtype,cache", [("f32", "f32"), ("bf16", "bf16")])
def test_a_pool_past_4_gib(capi, dtype, cache):
    """Pages at both ends of a pool of more than 2^32 bytes, on both sides of 2^31 and 2^32."""
    page, d, Hkv = 128, 128, 8
    item = 4 if dtype == "f32" else 2
    npages = 2 ** 32 // (Hkv * page * d * item) + 3
    K, V = (capi.DeviceBuffer((npages, Hkv, page, d), dtype) for _ in range(2))
    rng = np.random.default_rng(6)
    half = 2 ** 31 // (Hkv * page * d * item)
    tab = np.array([[0, half - 1, half, npages - 4, npages - 3, npages - 1]], np.int32)
    n, T = 6 * page - 9, 6 * page - 9
    k, v = (normal(rng, (1, Hkv, T, d), dtype) for _ in range(2))
    table, lengths = capi.DeviceBuffer.from_numpy(tab, "i32"), capi.DeviceBuffer.from_numpy(np.array([n], np.int32), "i32")
    dev = lambda a: capi.DeviceBuffer.from_numpy(a, dtype)  # noqa: E731
    capi.kv_append_paged(dev(k), dev(v), K, V, table, lengths)
    ko, vo = (capi.DeviceBuffer((1, Hkv, T, d), dtype) for _ in range(2))
    capi.kv_gather_paged(K, V, table, lengths, ko, vo)
    q = normal(rng, (1, 2 * Hkv, 1, d), dtype)
    o = capi.DeviceBuffer(q.shape, dtype)
    capi.attn_decode_paged(dev(q), K, V, table, lengths, o, None, 0.1)
    capi.lib().sync()
    assert np.array_equal(ko.download(), k) and np.array_equal(vo.download(), v)
    ref = po.Cache(6, Hkv, page, d, [[0, 1, 2, 3, 4, 5]])
    ref.append("k", k.astype(np.float64), [n])
    ref.append("v", v.astype(np.float64), [n])
    ro, _, mag, score = ref.attend(q, [n], float(np.float32(0.1)))
    rel = 2 * (d + 8) * U * score + TERMS[dtype] + 2 * (n + 8) * U
    assert (np.abs(o.download() - ro) <= rel[..., None] * mag * (1 + HALF[dtype]) + HALF[dtype] * np.abs(ro)).all()


# ------------------------------------------------------------------ splits and their merge

@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("H,T", [(1, 1), (3, 1), (2, 2)])
@pytest.mark.parametrize("d,n", [(32, 5117), (64, 1291), (128, 257)])
def test_splits_of_a_few_rows(capi, d, n, H, T, dtype, cache):
    """Three to forty splits that their last workgroup merges, call after call: the same bits each time."""
    rng = np.random.default_rng(d + H)
    lengths = [n, 1, 0, n // 3]
    c = filled(capi, dtype, cache, 4, 1, 64, d, lengths, rng)
    q = normal(rng, (4, H, T, d), dtype)
    first = c.attend(q, lengths, 0.2)
    c.check_attention(q, lengths, 0.2, first)
    for i in range(5):
        c.attend(normal(rng, (4, H, T, d), dtype), [n - 7 * i, n, 3, 0], 0.1)  # others in between
        o, lse = c.attend(q, lengths, 0.2, lse=i % 2 == 0)
        assert np.array_equal(o, first[0]) and (lse is None or np.array_equal(lse, first[1]))


@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f32", "u8")])
def test_a_sequence_over_hundreds_of_splits(capi, dtype, cache):
    rng = np.random.default_rng(21)
    n, page, d = 200003, 128, 32
    c = Cache(capi, dtype, cache, 1, 1, page, -(-n // page), d, rng)
    k, v = (normal(rng, (1, 1, n, d), dtype) for _ in range(2))
    c.append(k, v, [n])
    c.adopt()
    c.check_attention(normal(rng, (1, 2, 3, d), dtype), [n], 0.3)


@pytest.mark.parametrize("dtype,cache", KINDS)
def test_many_rows_of_a_head(capi, dtype, cache):
    """A prompt's chunk: seventeen tiles of query rows, the last one of four, most of whose tokens one sequence lacks."""
    rng = np.random.default_rng(22)
    lengths, T = [300, 26], 65
    c = filled(capi, dtype, cache, 2, 2, 32, 64, lengths, rng)
    c.check_attention(normal(rng, (2, 8, T, 64), dtype), lengths, 0.125)


def test_threads_and_streams(capi):
    """Four host threads, two to a stream: norms' gradients, appends, reads back and split attention, each as alone."""
    import threading

    f, d, B, Hkv, page = capi.DeviceBuffer.from_numpy, 64, 2, 2, 32
    streams, jobs = [capi.Stream(), capi.Stream()], []
    for i in range(4):
        rng = np.random.default_rng(30 + i)
        dtype, cache = KINDS[i]
        n = 700 + 300 * i
        c = filled(capi, dtype, cache, B, Hkv, page, d, [n, n // 2], rng, width=80)
        T = 40 + i
        x, dy = normal(rng, (B, 4, T, d), dtype), normal(rng, (B, 4, T, d), dtype)
        k, v, q = (normal(rng, (B, h, 1, d), dtype) for h in (Hkv, Hkv, 4))
        jobs.append(dict(c=c, st=streams[i % 2].handle, x=f(x, dtype), dy=f(dy, dtype), w=f(normal(rng, (d,), "f32")),
                         F=f(FREQ[64]), k=f(k, dtype), v=f(v, dtype), q=f(q, dtype), error=None, got=[],
                         out=lambda shape, t=dtype: capi.DeviceBuffer(shape, t), T=T, L=n))

    def work(j, times):
        try:
            c, s = j["c"], dict(stream=j["st"])
            for _ in range(times):
                dx, dw, o, lse = j["out"]((B, 4, j["T"], d)), j["out"]((d,), "f32"), j["out"]((B, 4, 1, d)), j["out"]((B, 4, 1), "f32")
                ko, vo = (j["out"]((B, Hkv, j["L"], d)) for _ in range(2))
                for b in (ko, vo):
                    b.zero()
                capi.lib().sync()
                capi.norm_rope_backward(j["x"], j["dy"], dx, j["w"], dw, j["F"], eps=EPS, **s)
                capi.kv_append_paged(j["k"], j["v"], c.dev["k"], c.dev["v"], c.tab, c.lengths, j["w"], j["F"], **c.scales(), **s)
                capi.attn_decode_paged(j["q"], c.dev["k"], c.dev["v"], c.tab, c.lengths, o, lse, 0.2, **c.scales(), **s)
                capi.kv_gather_paged(c.dev["k"], c.dev["v"], c.tab, c.lengths, ko, vo, **c.scales(), **s)
                j["got"].append((dx, dw, o, lse, ko, vo))
        except Exception as e:  # reported by the test's own thread
            j["error"] = e

    alone = []
    for j in jobs:
        work(j, 1)
        capi.lib().call("tt_stream_sync", j["st"])
        assert j["error"] is None
        alone.append([b.download() for b in j["got"].pop()])
    threads = [threading.Thread(target=work, args=(j, 12)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for st in streams:
        st.sync()
    for j, ref in zip(jobs, alone):
        assert j["error"] is None
        for got in j["got"]:
            for a, b in zip(got, ref):
                assert np.array_equal(a.download(), b)


def test_graphs_that_share_scratch(capi):
    """Two graphs of one stream, of other types and numbers of splits, replayed in turn with eager calls between."""
    rng, st, jobs = np.random.default_rng(40), capi.Stream(), []
    for dtype, cache, d, n, H, T in (("bf16", "bf16", 64, 5000, 2, 2), ("f32", "u8", 128, 700, 3, 1)):
        c = filled(capi, dtype, cache, 2, 1, 64, d, [n, n - 90], rng)
        q, x, dy = (capi.DeviceBuffer((2, H, t, d), dtype) for t in (T, 50, 50))
        o, lse, dx = capi.DeviceBuffer(q.shape, dtype), capi.DeviceBuffer((2, H, T)), capi.DeviceBuffer(x.shape, dtype)
        w, dw, F = capi.DeviceBuffer.from_numpy(normal(rng, (d,), "f32")), capi.DeviceBuffer((d,)), capi.DeviceBuffer.from_numpy(FREQ[d])

        def step(c=c, q=q, x=x, dy=dy, o=o, lse=lse, dx=dx, w=w, dw=dw, F=F):
            capi.attn_decode_paged(q, c.dev["k"], c.dev["v"], c.tab, c.lengths, o, lse, 0.2, stream=st.handle, **c.scales())
            capi.norm_rope_backward(x, dy, dx, w, dw, F, eps=EPS, stream=st.handle)

        c.lengths.upload(np.array([n, n - 90], np.int32))
        for b in (q, x, dy):
            b.fill_normal(1)
        capi.lib().sync()
        step()
        st.sync()
        with Capture(capi, st.handle, 1) as g:
            step()
        jobs.append(dict(step=step, g=g, inputs=(q, x, dy), out=(o, lse, dx, dw), dtype=dtype))
    for i in range(6):
        for j in jobs:
            for b in j["inputs"]:
                b.upload(normal(rng, b.shape, j["dtype"]))
        capi.lib().sync()
        ref = []
        for j in jobs:
            j["step"]()
            st.sync()
            ref.append([b.download() for b in j["out"]])
        for j, r in list(zip(jobs, ref))[::1 if i % 2 else -1] * 2:
            for b in j["out"]:
                b.zero()
            capi.lib().sync()
            j["g"].launch()
            assert all(np.array_equal(b.download(), a) for b, a in zip(j["out"], r))


REFUSED = r"""
import ctypes as C, numpy as np, tt_capi as T
from oracle import paged_oracle as po
from test_paged_gpu import Cache, filled, normal
def in_use():
    a = C.c_size_t()
    T.lib().call("tt_mem_stats", C.byref(a), None)
    return a.value
class Counted(T.DeviceBuffer):
    n = 0
    def __init__(self, *a, **k):
        Counted.n += 1
        super().__init__(*a, **k)
f, T.DeviceBuffer = T.DeviceBuffer, Counted
rng = np.random.default_rng(1)
c = filled(T, "f32", "f32", 1, 1, 64, 64, [2000], rng)
q = normal(rng, (1, 2, 1, 64), "f32")
o, lse, Q = T.DeviceBuffer(q.shape), T.DeviceBuffer((1, 2, 1)), T.DeviceBuffer.from_numpy(q)
x, w, dx, dw = (T.DeviceBuffer.from_numpy(np.full(s, 7.0, np.float32)) for s in ((1, 2, 5, 64), (64,), (1, 2, 5, 64), (64,)))
c.lengths.upload(np.array([2000], np.int32))
T.lib().sync()
print("COUNT", Counted.n, flush=True)
before = in_use()
T.attn_decode_paged(Q, c.dev["k"], c.dev["v"], c.tab, c.lengths, o, lse, 0.125)
T.lib().sync()
if %d:
    assert in_use() == before, "the scratch was not refused"
    try:
        T.norm_rope_backward(x, x, dx, w, dw)
        print("NOT REFUSED")
    except T.TTError as e:
        T.lib().sync()
        assert e.code == T.TT_ERR_NOMEM and (dx.download() == 7).all() and (dw.download() == 7).all()
        T.norm_rope_backward(x, x, dx, w, None)  # needs none
        T.lib().sync()
        assert not (dx.download() == 7).all()
        print("REFUSED True")
c.check_attention(q, [2000], 0.125, (o.download(), lse.download()))
print("DONE")
"""


def test_refused_scratch(capi):
    """Without its scratch the attention runs unsplit; weights' gradients are refused before anything is written."""
    def run(after, refuse):
        env = dict(os.environ, PYTHONPATH=os.pathsep.join([ROOT, os.path.join(ROOT, "pku-aiprogramming_amd"),
                                                           os.path.join(ROOT, "tests"), os.environ.get("PYTHONPATH", "")]))
        if refuse:
            env["TT_FAIL_ALLOC_AFTER"] = str(after)
        return subprocess.run([sys.executable, "-c", REFUSED % refuse], env=env, capture_output=True, text=True, timeout=100)

    r = run(0, 0)
    assert r.returncode == 0 and "DONE" in r.stdout, r.stdout + r.stderr
    r = run(int(r.stdout.split("COUNT")[1].split()[0]), 1)
    assert r.returncode == 0 and "REFUSED True" in r.stdout and "DONE" in r.stdout, r.stdout + r.stderr


# ------------------------------------------------------------------ together, streams, graphs

@pytest.mark.parametrize("dtype,cache", KINDS)
def test_a_model_goes_on(capi, dtype, cache):
    """A fused projection's rows normed, rotated, appended and attended to, a padded batch of prompts and then
    tokens; in 16 and 32 bits the prompt's attention is that of tt_attn_fwd on the rows read back."""
    rng = np.random.default_rng(12)
    B, H, Hkv, page, d, first = 2, 4, 2, 16, 64, 30
    c = Cache(capi, dtype, cache, B, Hkv, page, 4, d, rng)
    wq, wk = (1 + 0.1 * normal(rng, (d,), "f32") for _ in range(2))
    dev = lambda a, t=dtype: capi.DeviceBuffer.from_numpy(a, t)  # noqa: E731
    lengths, scale = np.array([first, 11], np.int32), float(np.float32(d ** -0.5))
    for step, T in enumerate((first, 1, 1, 3)):
        if step:
            lengths = (lengths + T).astype(np.int32)
        x = normal(rng, (B, T, H + 2 * Hkv, d), dtype)
        n = dev(lengths, "i32")
        q, kk, vv = (capi.DeviceBuffer((B, h, T, d), dtype) for h in (H, Hkv, Hkv))
        # the rotation on the way into the cache is the one of the queries
        rest = dict(q_weight=dev(wq, "f32"), k_weight=dev(wk, "f32"), inv_freq=dev(FREQ[64], "f32"), eps=EPS, lengths=n)
        capi.qkv_norm_rope(dev(x), q, kk, vv, **rest)
        k, v = (np.ascontiguousarray(np.swapaxes(x[:, :, a:a + Hkv], 1, 2)) for a in (H, H + Hkv))
        c.append(k, v, lengths, wk, FREQ[64], tokens_first=step % 2 == 0)
        if cache != "u8":
            got, mine = c.dev["k"].download(), kk.download()
            for b in range(B):
                for t in range(T):
                    j = lengths[b] - T + t
                    if j >= 0:
                        assert np.array_equal(got[c.table[b, j // page], :, j % page], mine[b, :, t])
        c.check(wk, FREQ[64]) if cache == "u8" else c.adopt()
        c.check_attention(q.download(), lengths, scale)
    if cache != "u8":
        L = int(lengths[0])
        k, v = (capi.DeviceBuffer((B, Hkv, L, d), dtype) for _ in range(2))
        capi.kv_gather_paged(c.dev["k"], c.dev["v"], c.tab, n, k, v)
        capi.lib().sync()
        kh, vh = (np.repeat(a.download()[:1], H // Hkv, 1) for a in (k, v))
        qh = normal(rng, (1, H, L, d), dtype)
        o = capi.DeviceBuffer(qh.shape, dtype)
        capi.attn_fwd(dev(qh), dev(kh), dev(vh), o, None, scale, True)
        capi.lib().sync()
        paged, _ = c.attend(np.concatenate([qh, qh]), [L, 0], scale)
        assert orc.max_rel_err(paged[:1], o.download()) <= (1e-4 if dtype == "f32" else 2e-2)


@pytest.mark.parametrize("dtype,cache", KINDS)
def test_captured_steps(capi, dtype, cache):
    """A token's step captured before its scratch is there (unsplit) and after; replayed as lengths go on, with eager
    work on the stream and on another between the replays."""
    rng = np.random.default_rng(13)
    B, H, Hkv, page, d, n0 = 2, 4, 2, 16, 64, 900
    c = filled(capi, dtype, cache, B, Hkv, page, d, [n0, n0 - 7], rng, width=64)
    k, v, q = (capi.DeviceBuffer((B, h, 1, d), dtype) for h in (Hkv, Hkv, H))
    F = capi.DeviceBuffer.from_numpy(FREQ[64])
    o, lse = capi.DeviceBuffer((B, H, 1, d), dtype), capi.DeviceBuffer((B, H, 1), "f32")

    def step(stream):
        capi.kv_append_paged(k, v, c.dev["k"], c.dev["v"], c.tab, c.lengths, None, F, stream=stream, **c.scales())
        capi.attn_decode_paged(q, c.dev["k"], c.dev["v"], c.tab, c.lengths, o, lse, 0.125, stream=stream, **c.scales())

    st, graphs = capi.Stream(), []
    for warm in (False, True):
        if warm:
            c.attend(normal(rng, (B, H, 1, d), dtype), [n0, n0], 0.125, stream=st.handle)
        with Capture(capi, st.handle, 1) as g:
            step(st.handle)
        graphs.append(g)
    lengths = np.array([n0, n0 - 7], np.int32)
    for i in range(6):
        lengths = (lengths + 1).astype(np.int32)
        x = [normal(rng, b.shape, dtype) for b in (k, v, q)]
        for b, a in zip((k, v, q), x):
            b.upload(a)
        c.lengths.upload(lengths)
        capi.lib().sync()
        graphs[i % 2].launch()
        got = o.download(), lse.download()
        pos = po.positions(B, 1, lengths=lengths)
        c.ref.append("k", po.norm_rope(x[0], None, EPS, pos, FREQ[64], False), lengths)
        c.ref.append("v", x[1].astype(np.float64), lengths)
        c.check() if cache == "u8" else c.adopt()
        c.check_attention(x[2], lengths, 0.125, got)
        c.check_attention(x[2], lengths, 0.125, c.attend(x[2], lengths, 0.125, stream=st.handle if i % 3 else None))


@pytest.mark.parametrize("name", ["float", "bf16"])
@pytest.mark.parametrize("small", [False, True])
def test_layer_functions(name, small):
    """myLayer's functions over a fused projection from FcForward, and their refusals."""
    import myLayer as ml
    import myTensor as mt

    rng = np.random.default_rng(14)
    dtype = "f32" if name == "float" else "bf16"
    T_ = getattr(mt, "Tensor_" + name)
    B, H, Hkv, page, d, E, T = 2, 4, 2, 16, 32, 24, 20
    n = H + 2 * Hkv
    x = T_(normal(rng, (B, T, E), dtype), "gpu")
    w, zero = T_(normal(rng, (E, n * d), dtype, 0.3), "gpu"), T_([1], "gpu").zeros()
    qkv, q, k, v = (T_([1], "gpu") for _ in range(4))
    ml.FcForward(x, qkv, w, zero)
    qkv.resize([B, T, n, d])
    host = qkv.numpy().reshape(B, T, n, d)
    wq, wk = (1 + 0.1 * normal(rng, (d,), "f32") for _ in range(2))
    tq, tk, tf = mt.Tensor_float(wq, "gpu"), mt.Tensor_float(wk, "gpu"), mt.Tensor_float(FREQ[32], "gpu")
    lengths = np.array([20, 13], np.int32)
    tn = mt.Tensor_int([B], "gpu", lengths.tolist())  # a flat array of whole numbers would be a shape
    ml.QkvNormRopeForward(qkv, q, k, v, Hkv, tq, tk, tf, EPS, lengths=tn)
    assert q.get_shape() == [B, H, T, d] and k.get_shape() == v.get_shape() == [B, Hkv, T, d]
    pos = po.positions(B, T, lengths=lengths)
    sides = [np.ascontiguousarray(np.swapaxes(p, 1, 2)) for p in np.split(host, [H, H + Hkv], 2)]
    from test_norm_rope_gpu import check_backward, check_forward

    check_forward(q.numpy().reshape(B, H, T, d), sides[0], wq, pos, FREQ[32], False, dtype)
    check_forward(k.numpy().reshape(B, Hkv, T, d), sides[1], wk, pos, FREQ[32], False, dtype)
    dy = [normal(rng, s.shape, dtype) for s in sides]
    gx, gq, gk = T_([1], "gpu"), mt.Tensor_float([1], "gpu"), mt.Tensor_float([1], "gpu")
    ml.QkvNormRopeBackward(qkv, *(T_(a, "gpu") for a in dy), gx, tq, tk, gq, gk, tf, EPS, lengths=tn)
    back = [np.swapaxes(p, 1, 2) for p in np.split(gx.numpy().reshape(B, T, n, d), [H, H + Hkv], 2)]
    check_backward(back[0], gq.numpy(), sides[0], wq, dy[0], pos, FREQ[32], False, dtype, B * T * H)
    check_backward(back[1], gk.numpy(), sides[1], wk, dy[1], pos, FREQ[32], False, dtype, B * T * Hkv)
    assert np.array_equal(back[2], dy[2])

    npages, width = 5, 2
    shape = [npages, Hkv, page, d]
    pools = [(mt.Tensor_byte if small else T_)(shape, "gpu").zeros() for _ in range(2)]
    extra = dict(k_scales=mt.Tensor_byte([npages, Hkv], "gpu"), v_scales=mt.Tensor_byte([npages, Hkv], "gpu")) if small else {}
    table = np.array([[4, 0], [2, 3]], np.int32)
    tt = mt.Tensor_int(table, "gpu")
    ml.KvAppendPaged(T_(sides[1], "gpu"), v, *pools, tt, tn, k_weight=tk, inv_freq=tf, eps=EPS, **extra)
    ref = po.Cache(npages, Hkv, page, d, table, small)
    ref.append("k", po.norm_rope(sides[1], wk, EPS, pos, FREQ[32], False), lengths)
    ref.append("v", sides[2].astype(np.float64), lengths)
    ko, vo = T_([1], "gpu"), T_([1], "gpu")
    ml.KvGatherPaged(*pools, tt, tn, ko, vo, T, **extra)
    for b, size in enumerate(lengths):
        rows, _ = ref.rows("v", b, size)
        assert np.array_equal(vo.numpy().reshape(B, Hkv, T, d)[b, :, :size], rows)
        rows, _ = ref.rows("k", b, size)
        got = ko.numpy().reshape(B, Hkv, T, d)[b, :, :size]
        assert np.array_equal(got, rows) if small else np.abs(got - rows).max() <= 2 * HALF[dtype] * np.abs(rows).max() + 1e-5
    out = T_([1], "gpu")
    ml.AttentionDecodePaged(q, *pools, tt, tn, out, 0.2, **extra)
    if not small:
        for n_, p in zip("kv", pools):
            ref.pool[n_][:] = p.numpy().reshape(shape)
    ro, _, mag, score = ref.attend(q.numpy().reshape(B, H, T, d), lengths, float(np.float32(0.2)))
    rel = 2 * (d + 8) * U * score + TERMS[dtype] + 2 * (T + 8) * U
    got = out.numpy().reshape(B, H, T, d)
    assert (np.abs(got - ro) <= rel[..., None] * mag * (1 + HALF[dtype]) + HALF[dtype] * np.abs(ro)).all()

    one, f = T_([1], "gpu"), mt.Tensor_float([1], "gpu")
    bad = [lambda: ml.NormRopeForward(one, one), lambda: ml.NormRopeForward(q, q),
           lambda: ml.NormRopeForward(q, one, weight=f), lambda: ml.NormRopeForward(q, one, positions=tn),
           lambda: ml.NormRopeBackward(q, k, one), lambda: ml.NormRopeBackward(q, q, one, grad_weight=f),
           lambda: ml.QkvNormRopeForward(qkv, q, k, v, n), lambda: ml.QkvNormRopeForward(qkv, q, q, v, Hkv),
           lambda: ml.QkvNormRopeBackward(qkv, q, k, q, one), lambda: ml.QkvNormRopeBackward(qkv, q, k, v, one, tq, tk, gq, gq),
           lambda: ml.KvAppendPaged(q, v, *pools, tt, tn, **extra), lambda: ml.KvAppendPaged(q, q, *pools, tt, tn, **extra),
           lambda: ml.KvAppendPaged(v, v, *pools, tt, mt.Tensor_int([3], "gpu"), **extra),
           lambda: ml.KvAppendPaged(v, v, *pools, tn, tn, **extra), lambda: ml.KvAppendPaged(v, v, pools[0], pools[0], tt, tn, **extra),
           lambda: ml.KvGatherPaged(*pools, tt, tn, ko, ko, T, **extra), lambda: ml.KvGatherPaged(*pools, tt, tn, ko, vo, -1, **extra),
           lambda: ml.AttentionDecodePaged(T_([B, 3, 1, d], "gpu"), *pools, tt, tn, out, 0.2, **extra),
           lambda: ml.AttentionDecodePaged(q, *pools, tt, tn, q, 0.2, **extra),
           lambda: ml.AttentionDecodePaged(q, *pools, tt, tn, out, 0.2,
                                           **({} if small else dict(k_scales=mt.Tensor_byte([npages, Hkv], "gpu"),
                                                                    v_scales=mt.Tensor_byte([npages, Hkv], "gpu"))))]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")
