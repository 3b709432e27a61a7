"""GPU tests of norms and rotation at the sizes where their kernels change: two and four
heads a workgroup, with heads that these do not divide, and gradients that go past the
caches.  The bounds are those of test_norm_rope_gpu.py, where a weight's gradient is a
chain of fewer than 80 additions: four heads of two tiles a thread, nine steps over lanes
and waves, and of the workgroups' sums 48 and 8 (up to 12288 / d in groups of 256 / d) or
32 and 6 (up to 2048 in groups of 64)."""
import numpy as np
import pytest

from oracle import paged_oracle as po
from test_norm_rope_gpu import EPS, FREQ, U, capi, check_backward, check_forward, normal, pairs  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu
CUS = 256


def heads_of_a_workgroup(tokens, heads, d, dtype):
    """The rule: four heads, two or one where more would leave fewer than two workgroups a CU."""
    tiles = -(-tokens // (256 // (d // (8 if dtype == "f32" else 16))))
    count = 4
    while count > 1 and tiles * heads < 2 * count * CUS:
        count //= 2
    return count


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d,rot,inter", [(32, 32, True), (64, 64, False), (64, 32, True), (128, 128, False), (128, 96, True)])
@pytest.mark.parametrize("count", [2, 4])
def test_heads_of_a_workgroup(capi, count, d, rot, inter, dtype):  # noqa: F811
    """A fused projection, forward and back, of 7 and 3 heads."""
    rng = np.random.default_rng(d + rot + count)
    B, H, Hkv = 3, 7, 3
    T = (256 // (d // (8 if dtype == "f32" else 16)) * (94 if count == 2 else 165)) // B - 3
    assert heads_of_a_workgroup(B * T, H + 2 * Hkv, d, dtype) == count
    x = normal(rng, (B, T, H + 2 * Hkv, d), dtype)
    dy = [normal(rng, (B, h, T, d), dtype) for h in (H, Hkv, Hkv)]
    wq, wk = (1 + 0.2 * normal(rng, (d,), "f32") for _ in range(2))
    dev = lambda a, t=dtype: capi.DeviceBuffer.from_numpy(a, t)  # noqa: E731
    lengths = np.array([T, 131072, 70000], np.int32)
    X, DY, n = dev(x), [dev(a) for a in dy], dev(lengths, "i32")
    rest = dict(q_weight=dev(wq, "f32"), k_weight=dev(wk, "f32"), inv_freq=dev(FREQ[rot], "f32"), eps=EPS, lengths=n, interleaved=inter)
    out = [capi.DeviceBuffer((B, h, T, d), dtype) for h in (H, Hkv, Hkv)]
    capi.qkv_norm_rope(X, *out, **rest)
    dx, dw = capi.DeviceBuffer(x.shape, dtype), [capi.DeviceBuffer((d,)) for _ in range(2)]
    capi.qkv_norm_rope_backward(X, *DY, dx, dq_weight=dw[0], dk_weight=dw[1], **rest)
    capi.lib().sync()
    pos = po.positions(B, T, lengths=lengths)
    sides = [np.ascontiguousarray(np.swapaxes(p, 1, 2)) for p in np.split(x, [H, H + Hkv], 2)]
    back = [np.swapaxes(p, 1, 2) for p in np.split(dx.download(), [H, H + Hkv], 2)]
    for i, w in enumerate((wq, wk)):
        check_forward(out[i].download(), sides[i], w, pos, FREQ[rot], inter, dtype)
        check_backward(back[i], dw[i].download(), sides[i], w, dy[i], pos, FREQ[rot], inter, dtype, 80)
    assert np.array_equal(out[2].download(), sides[2]) and np.array_equal(back[2], dy[2])
    # head-major, q alone, rotated alone: other loops over the same heads
    if H * B * T * d < 2 ** 23:
        y = capi.DeviceBuffer((B, H, T, d), dtype)
        capi.norm_rope(dev(sides[0]), y, None, rest["inv_freq"], interleaved=inter, lengths=n)
        gx = capi.DeviceBuffer((B, H, T, d), dtype)
        capi.norm_rope_backward(None, DY[0], gx, None, None, rest["inv_freq"], interleaved=inter, lengths=n)
        capi.lib().sync()
        check_forward(y.download(), sides[0], None, pos, FREQ[rot], inter, dtype)
        check_backward(gx.download(), None, None, None, dy[0], pos, FREQ[rot], inter, dtype, 0)


@pytest.mark.parametrize("dtype,d,T", [("bf16", 128, 8500), ("f32", 128, 4300), ("bf16", 64, 17000), ("f32", 32, 17100)])
def test_gradients_past_the_caches(capi, d, T, dtype):  # noqa: F811
    """More than 256 MiB: every row has the bits that it has in a call of its own sequence, and the weights'
    gradients are their sum."""
    B, H, Hkv, e = 2, 9, 8, 4 if dtype == "f32" else 2
    total = B * T * d * (3 * (H + Hkv) + 2 * Hkv) * e
    assert total > 2 ** 28 > total // 2 and heads_of_a_workgroup(T, H + 2 * Hkv, d, dtype) == 4
    n = H + 2 * Hkv
    buf = lambda *s, t=dtype: capi.DeviceBuffer(s, t)  # noqa: E731
    x, dx, dy = buf(B, T, n, d), buf(B, T, n, d), [buf(B, h, T, d) for h in (H, Hkv, Hkv)]
    for i, b in enumerate((x, *dy)):
        b.fill_normal(5 + i)
    rng = np.random.default_rng(d)
    w = [1 + 0.2 * normal(rng, (d,), "f32") for _ in range(2)]
    dev = lambda a, t="f32": capi.DeviceBuffer.from_numpy(a, t)  # noqa: E731
    rest = dict(q_weight=dev(w[0]), k_weight=dev(w[1]), inv_freq=dev(FREQ[d // 2]), eps=EPS)
    dw = [buf(d, t="f32") for _ in range(2)]
    capi.qkv_norm_rope_backward(x, *dy, dx, dq_weight=dw[0], dk_weight=dw[1], **rest)
    capi.lib().sync()
    hx, hdx, hdy = x.download(), dx.download(), [b.download() for b in dy]
    sums = np.zeros((2, d))
    for b in range(B):
        part, pw = buf(1, T, n, d), [buf(d, t="f32") for _ in range(2)]
        capi.qkv_norm_rope_backward(dev(hx[b:b + 1], dtype), *(dev(a[b:b + 1], dtype) for a in hdy), part, dq_weight=pw[0],
                                    dk_weight=pw[1], **rest)
        capi.lib().sync()
        assert np.array_equal(part.download()[0], hdx[b])
        sums += [p.download().astype(np.float64) for p in pw]
    for i, (lo, hi) in enumerate(((0, H), (H, H + Hkv))):
        rows = np.swapaxes(hx[:, :, lo:hi], 1, 2)
        normed = np.abs(rows) / np.sqrt(np.mean(rows * rows, -1, keepdims=True) + np.float32(EPS))
        top = (pairs(hdy[i], d // 2, False) * normed).sum((0, 1, 2), dtype=np.float64)
        assert -(-B * T // (256 // (d // (8 if dtype == "f32" else 16)))) <= 2 * (2048 // 5)  # two tiles: 5 chunks of heads
        assert (np.abs(dw[i].download() - sums[i]) <= 2 * (80 + d / 2 + 40) * U * top * (1 + 2.0 ** -20)).all()
    # rows of the first and the last tokens against the formula
    for b, t0 in ((0, 0), (B - 1, T - 40)):
        at = np.s_[t0:t0 + 40]
        for i, (lo, hi) in enumerate(((0, H), (H, H + Hkv))):
            xs = np.swapaxes(hx[b:b + 1, at, lo:hi], 1, 2)
            check_backward(np.swapaxes(hdx[b:b + 1, at, lo:hi], 1, 2), None, xs, w[i], hdy[i][b:b + 1, :, at],
                           np.arange(T, dtype=np.float64)[None, at], FREQ[d // 2], False, dtype, 0)
        assert np.array_equal(hdx[b, at, H + Hkv:], np.swapaxes(hdy[2][b, :, at], 0, 1))
