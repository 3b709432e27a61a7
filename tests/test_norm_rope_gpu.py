"""GPU tests of norms and rotation of heads against the float64 oracle.

Bounds, u = 2^-24.  A row's scale 1 / sqrt(mean x^2 + eps) is off by at most (d / 2 +
4) u of itself (the sum of d squares, halved by the root, and the root), so a normed
value by (d / 2 + 7) u; cos and sin by 4 u (the reduced angle's rounding, the
series); a turned pair by those, two products and a sum, all of |a| + |b|: (d / 2 +
16) u (|a| + |b|).  Backwards the gradient's pairs are off by 7 u (|a| + |b|), and
dx = r (g w - n mean(g w n)) by (3 d / 2 + 40) u of r (|g w| + |n| mean |g w n|); dw, a
sum of R rows, by (R + d / 2 + 40) u of the sum of |g n|.  The store adds half a step."""
import numpy as np
import pytest

from oracle import attn_oracle as orc
from oracle import paged_oracle as po
from test_capture_gpu import Capture

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}
EPS = 1e-5


@pytest.fixture(scope="module")
def capi():
    import tt_capi

    assert tt_capi.lib().device_count() >= 1, "no HIP device visible"
    tt_capi.lib().call("tt_init", 0)
    return tt_capi


def normal(rng, shape, dtype, std=1.0):
    x = (rng.standard_normal(shape) * std).astype(np.float32)
    return orc.bf16_round(x) if dtype == "bf16" else x


def pairs(x, rot, interleaved):
    """|a| + |b| at both places of each pair, |x| elsewhere."""
    y = np.abs(x)
    i, j = (np.s_[..., 0:rot:2], np.s_[..., 1:rot:2]) if interleaved else (np.s_[..., :rot // 2], np.s_[..., rot // 2:rot])
    s = y[i] + y[j]
    y = y.copy()
    y[i], y[j] = s, s
    return y


def check_forward(got, x, w, pos, freq, inter, dtype, eps=EPS):
    d, rot = x.shape[-1], 0 if freq is None else 2 * len(freq)
    ref = po.norm_rope(x, w, eps, pos, freq, inter)
    bound = (d / 2 + 16) * U * pairs(po.norm(x, w, eps), rot, inter) * (1 + HALF[dtype]) + HALF[dtype] * np.abs(ref)
    bound = np.where(np.abs(ref) < 2.0 ** -100, bound + 2.0 ** -130, bound)  # fp32's own steps next to zero
    worst = np.max(np.abs(got - ref) - bound)
    assert worst <= 0, worst


def check_backward(dx, dw, x, w, dy, pos, freq, inter, dtype, rows):
    d, rot = dy.shape[-1], 0 if freq is None else 2 * len(freq)
    rx, rw = po.norm_rope_backward(x, w, EPS, pos, freq, inter, dy)
    back = po.rotate(dy, pos, freq, inter, back=True)
    g = pairs(back, rot, inter)
    if w is None:
        bound = 7 * U * g
    else:
        x64 = np.asarray(x, np.float64)
        r = 1 / np.sqrt(np.mean(x64 * x64, -1, keepdims=True) + np.float64(np.float32(EPS)))
        n, gw = np.abs(x64 * r), g * np.abs(w)
        bound = (1.5 * d + 40) * U * r * (gw + n * np.mean(gw * n, -1, keepdims=True))
        if dw is not None:
            assert (np.abs(dw - rw) <= (rows + d / 2 + 40) * U * (g * n).sum((0, 1, 2)) + U * np.abs(rw)).all()
    assert (np.abs(dx - rx) <= bound * (1 + HALF[dtype]) + HALF[dtype] * np.abs(rx)).all()


FREQ = {rot: (10000.0 ** (-2.0 * np.arange(rot // 2) / rot)).astype(np.float32) for rot in (0, 16, 32, 48, 64, 96, 128)}


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("d,rot", [(32, 32), (32, 16), (64, 64), (64, 48), (128, 128), (128, 96), (128, 16), (128, 0)])
@pytest.mark.parametrize("B,H,Hkv,T", [(1, 1, 1, 1), (3, 5, 2, 37)])
def test_fused_projection(capi, B, H, Hkv, T, d, rot, inter, dtype):
    """Out of one projection's rows, forward and back, at positions that lengths give."""
    rng = np.random.default_rng(d + rot + T)
    n = H + 2 * Hkv
    x = normal(rng, (B, T, n, d), dtype)
    wq, wk = (normal(rng, (d,), "f32") + 1 for _ in range(2))
    lengths = rng.integers(0, 3 * T + 1, B).astype(np.int32)  # the first tokens of some before position 0
    pos, freq = po.positions(B, T, lengths=lengths), FREQ[rot]
    dev = lambda a, t=dtype: capi.DeviceBuffer.from_numpy(a, t)  # noqa: E731
    out = [capi.DeviceBuffer((B, h, T, d), dtype) for h in (H, Hkv, Hkv)]
    rest = dict(q_weight=dev(wq, "f32"), k_weight=dev(wk, "f32"), inv_freq=dev(freq, "f32") if rot else None, eps=EPS,
                lengths=dev(lengths, "i32"), interleaved=inter)
    capi.qkv_norm_rope(dev(x), *out, **rest)
    capi.lib().sync()
    parts = [np.ascontiguousarray(np.swapaxes(p, 1, 2)) for p in np.split(x, [H, H + Hkv], 2)]
    check_forward(out[0].download(), parts[0], wq, pos, freq, inter, dtype)
    check_forward(out[1].download(), parts[1], wk, pos, freq, inter, dtype)
    assert np.array_equal(out[2].download(), parts[2])

    dy = [normal(rng, (B, h, T, d), dtype) for h in (H, Hkv, Hkv)]
    dx = capi.DeviceBuffer((B, T, n, d), dtype)
    dw = [capi.DeviceBuffer((d,), "f32") for _ in range(2)]
    capi.qkv_norm_rope_backward(dev(x), *(dev(a) for a in dy), dx, dq_weight=dw[0], dk_weight=dw[1], **rest)
    capi.lib().sync()
    got = [np.swapaxes(p, 1, 2) for p in np.split(dx.download(), [H, H + Hkv], 2)]
    check_backward(got[0], dw[0].download(), parts[0], wq, dy[0], pos, freq, inter, dtype, B * T * H)
    check_backward(got[1], dw[1].download(), parts[1], wk, dy[1], pos, freq, inter, dtype, B * T * Hkv)
    assert np.array_equal(got[2], dy[2])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens_first", [False, True])
@pytest.mark.parametrize("weight,rot", [(True, 64), (True, 0), (False, 64), (False, 0)])
def test_one_tensor(capi, weight, rot, tokens_first, dtype):
    """With and without the norm, the rotation and both, at given positions, in both layouts."""
    rng = np.random.default_rng(rot + weight)
    B, H, T, d = 2, 3, 70, 64
    x, dy = normal(rng, (B, H, T, d), dtype, 3.0), normal(rng, (B, H, T, d), dtype)
    w = normal(rng, (d,), "f32") if weight else None
    given = rng.integers(-50, 2 ** 20, (B, T)).astype(np.int32)
    freq = FREQ[rot] if rot else None
    pos = po.positions(B, T, given=given)
    put = lambda a: capi.DeviceBuffer.from_numpy(np.ascontiguousarray(np.swapaxes(a, 1, 2)) if tokens_first else a, dtype)  # noqa: E731
    y, dx = capi.DeviceBuffer((B, H, T, d), dtype), put(np.zeros_like(x))
    dw = capi.DeviceBuffer((d,), "f32") if weight else None
    rest = dict(weight=capi.DeviceBuffer.from_numpy(w) if weight else None,
                inv_freq=capi.DeviceBuffer.from_numpy(freq) if rot else None, eps=EPS,
                positions=capi.DeviceBuffer.from_numpy(given, "i32"), tokens_first=tokens_first)
    capi.norm_rope(put(x), y, **rest)
    capi.norm_rope_backward(put(x) if weight else None, capi.DeviceBuffer.from_numpy(dy, dtype), dx, dweight=dw, **rest)
    capi.lib().sync()
    check_forward(y.download(), x, w, pos, freq, False, dtype)
    gx = dx.download()
    check_backward(np.swapaxes(gx, 1, 2) if tokens_first else gx, dw.download() if weight else None, x, w, dy, pos, freq, False,
                   dtype, B * H * T)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("far", [131071, 2 ** 24 + 1, 2 ** 31 - 1])
def test_far_positions(capi, far, dtype):
    """Angles of millions of turns are as exact as those next to zero."""
    rng = np.random.default_rng(far % 97)
    d = 128
    x = normal(rng, (1, 2, 64, d), dtype)
    given = (far - rng.integers(0, 1000, (1, 64))).astype(np.int32)
    y = capi.DeviceBuffer(x.shape, dtype)
    capi.norm_rope(capi.DeviceBuffer.from_numpy(x, dtype), y, inv_freq=capi.DeviceBuffer.from_numpy(FREQ[128]),
                   positions=capi.DeviceBuffer.from_numpy(given, "i32"))
    capi.lib().sync()
    check_forward(y.download(), x, None, po.positions(1, 64, given=given), FREQ[128], False, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_keep_to_themselves(capi, dtype):
    """Rows of zeros, infinities and NaN change no other row, forward or back, nor the other weight's gradient."""
    rng = np.random.default_rng(5)
    B, H, Hkv, T, d = 1, 4, 2, 50, 128
    x, w = normal(rng, (B, T, H + 2 * Hkv, d), dtype), normal(rng, (d,), "f32")
    dy = [normal(rng, (B, h, T, d), dtype) for h in (H, Hkv, Hkv)]
    dev = lambda a, t=dtype: capi.DeviceBuffer.from_numpy(a, t)  # noqa: E731

    def run(x):
        out = [capi.DeviceBuffer((B, h, T, d), dtype) for h in (H, Hkv, Hkv)]
        dx, dw = capi.DeviceBuffer(x.shape, dtype), [capi.DeviceBuffer((d,), "f32") for _ in range(2)]
        rest = dict(q_weight=dev(w, "f32"), k_weight=dev(w, "f32"), inv_freq=dev(FREQ[128], "f32"), eps=EPS)
        capi.qkv_norm_rope(dev(x), *out, **rest)
        capi.qkv_norm_rope_backward(dev(x), *(dev(a) for a in dy), dx, dq_weight=dw[0], dk_weight=dw[1], **rest)
        capi.lib().sync()
        return [b.download() for b in out], dx.download(), [b.download() for b in dw]

    plain, pdx, pdw = run(x)
    odd = x.copy()
    odd[0, 7, 1] = 0.0
    odd[0, 20, 2, 5] = np.inf
    odd[0, 21, 0, 9] = np.nan
    got, gdx, gdw = run(odd)
    same = np.ones((T, H), bool)
    same[[7, 20, 21], [1, 2, 0]] = False
    assert np.array_equal(got[0][0].swapaxes(0, 1)[same], plain[0][0].swapaxes(0, 1)[same])
    assert (got[0][0, 1, 7] == 0).all() and not np.isfinite(got[0][0, 2, 20]).all() and np.isnan(got[0][0, 0, 21]).all()
    assert np.array_equal(got[1], plain[1]) and np.array_equal(got[2], plain[2])
    assert np.array_equal(gdx[0, :, :H][same], pdx[0, :, :H][same]) and np.array_equal(gdx[:, :, H:], pdx[:, :, H:])
    assert np.isfinite(gdx[0, 7, 1]).all()
    assert np.array_equal(gdw[1], pdw[1]) and np.isnan(gdw[0]).any()


def test_strided_rows_between_others(capi):
    """q, k and v in a wider matrix: what lies between the parts is neither read nor written."""
    rng = np.random.default_rng(6)
    B, T, H, Hkv, d, ld, at = 2, 19, 3, 1, 64, 64 * 9, (64, 64 * 5, 64 * 7)
    x = np.full((B, T, ld), np.nan, np.float32)
    for a, h in zip(at, (H, Hkv, Hkv)):
        x[:, :, a:a + h * d] = rng.standard_normal((B, T, h * d))
    w = (rng.standard_normal(d)).astype(np.float32)
    dy = [rng.standard_normal((B, h, T, d)).astype(np.float32) for h in (H, Hkv, Hkv)]
    X, W, F = capi.DeviceBuffer.from_numpy(x), capi.DeviceBuffer.from_numpy(w), capi.DeviceBuffer.from_numpy(FREQ[64])
    out = [capi.DeviceBuffer(a.shape) for a in dy]
    dx, dw = capi.DeviceBuffer.from_numpy(np.full(x.shape, 7.0, np.float32)), [capi.DeviceBuffer((d,)) for _ in range(2)]
    p, g = [X.ptr + 4 * a for a in at], [dx.ptr + 4 * a for a in at]
    rope = (W.ptr, W.ptr, EPS, F.ptr, 64, 1, None, None)
    capi.lib().call("tt_qkv_norm_rope", capi.TT_F32, *p, ld, ld, ld, *rope, *(b.ptr for b in out), B, H, Hkv, T, d, None)
    D = [capi.DeviceBuffer.from_numpy(a) for a in dy]
    capi.lib().call("tt_qkv_norm_rope_backward", capi.TT_F32, p[0], p[1], ld, ld, *rope, *(b.ptr for b in D), *g, ld, ld, ld,
                    dw[0].ptr, dw[1].ptr, B, H, Hkv, T, d, None)
    capi.lib().sync()
    pos, got = po.positions(B, T), dx.download()
    for i, (a, h) in enumerate(zip(at, (H, Hkv, Hkv))):
        part = x[:, :, a:a + h * d].reshape(B, T, h, d).swapaxes(1, 2)
        back = got[:, :, a:a + h * d].reshape(B, T, h, d).swapaxes(1, 2)
        if i == 2:
            assert np.array_equal(out[2].download(), part) and np.array_equal(back, dy[2])
        else:
            check_forward(out[i].download(), part, w, pos, FREQ[64], True, "f32")
            check_backward(back, dw[i].download(), part, w, dy[i], pos, FREQ[64], True, "f32", B * T * h)
        got[:, :, a:a + h * d] = 7.0
    assert (got == 7.0).all()


@pytest.mark.parametrize("parts", ["q", "k", "v", "kv", "qv"])
def test_some_of_the_parts(capi, parts):
    """q, k and v given or not, head-major: what is not given is neither read nor written; frequencies of no pair."""
    rng = np.random.default_rng(10)
    B, T, H, Hkv, d = 2, 21, 3, 2, 64
    heads, w, F = dict(q=H, k=Hkv, v=Hkv), normal(rng, (d,), "f32"), capi.DeviceBuffer.from_numpy(FREQ[32])
    x = {n: normal(rng, (B, h, T, d), "f32") for n, h in heads.items()}
    dy = {n: normal(rng, (B, h, T, d), "f32") for n, h in heads.items()}
    X, DY, W = ({n: capi.DeviceBuffer.from_numpy(a) for n, a in g.items()} for g in (x, dy, dict(q=w, k=w)))
    out, dx = ({n: capi.DeviceBuffer.from_numpy(np.full(a.shape, 7.0, np.float32)) for n, a in x.items()} for _ in range(2))
    dw = {n: capi.DeviceBuffer.from_numpy(np.full(d, 7.0, np.float32)) for n in "qk"}
    ptr = lambda g, n: g[n].ptr if n in parts else None  # noqa: E731
    for rot in (32, 0):
        rope = (EPS, F.ptr, rot, 0, None, None)
        capi.lib().call("tt_qkv_norm_rope", capi.TT_F32, *(ptr(X, n) for n in "qkv"), 0, 0, 0, W["q"].ptr, W["k"].ptr, *rope,
                        *(ptr(out, n) for n in "qkv"), B, H, Hkv, T, d, None)
        capi.lib().call("tt_qkv_norm_rope_backward", capi.TT_F32, ptr(X, "q"), ptr(X, "k"), 0, 0, W["q"].ptr, W["k"].ptr, *rope,
                        *(ptr(DY, n) for n in "qkv"), *(ptr(dx, n) for n in "qkv"), 0, 0, 0, ptr(dw, "q"), ptr(dw, "k"),
                        B, H, Hkv, T, d, None)
        capi.lib().sync()
        pos, freq = po.positions(B, T), FREQ[rot] if rot else None
        for n in "qkv":
            if n not in parts:
                assert (out[n].download() == 7.0).all() and (dx[n].download() == 7.0).all()
                assert n == "v" or (dw[n].download() == 7.0).all()
            elif n == "v":
                assert np.array_equal(out[n].download(), x[n]) and np.array_equal(dx[n].download(), dy[n])
            else:
                check_forward(out[n].download(), x[n], w, pos, freq, False, "f32")
                check_backward(dx[n].download(), dw[n].download(), x[n], w, dy[n], pos, freq, False, "f32", B * T * heads[n])


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_few_and_many_sums_in_turn(capi, dtype, d):
    """Sums that the last workgroup adds up and sums that a launch does, of one weight and of both, call after call."""
    rng = np.random.default_rng(11)
    w = capi.DeviceBuffer.from_numpy(1 + normal(rng, (d,), "f32"))
    jobs = []
    for B, T, H, Hkv, both in ((1, 1, 1, 1, True), (3, 50, 4, 2, True), (2, 33, 5, 1, False), (2, 700, 6, 2, True)):
        x, dy = normal(rng, (B, T, H + 2 * Hkv, d), dtype), [normal(rng, (B, h, T, d), dtype) for h in (H, Hkv, Hkv)]
        jobs.append((B, T, H, Hkv, both, x, dy, capi.DeviceBuffer.from_numpy(x, dtype), [capi.DeviceBuffer.from_numpy(a, dtype) for a in dy]))
    first = {}
    for turn in range(4):
        for i, (B, T, H, Hkv, both, x, dy, X, DY) in enumerate(jobs):
            dx, dw = capi.DeviceBuffer(x.shape, dtype), [capi.DeviceBuffer((d,)) for _ in range(2)]
            capi.qkv_norm_rope_backward(X, *DY, dx, w, w, dw[0] if both else None, dw[1], eps=EPS)
            capi.lib().sync()
            got = [dx.download(), dw[1].download()] + ([dw[0].download()] if both else [])
            if turn:
                assert all(np.array_equal(a, b) for a, b in zip(got, first[i]))
                continue
            first[i] = got
            sides = [np.ascontiguousarray(np.swapaxes(p, 1, 2)) for p in np.split(x, [H, H + Hkv], 2)]
            back = [np.swapaxes(p, 1, 2) for p in np.split(got[0], [H, H + Hkv], 2)]
            W, pos = w.download(), po.positions(B, T)
            check_backward(back[0], got[2] if both else None, sides[0], W, dy[0], pos, None, False, dtype, B * T * H)
            check_backward(back[1], got[1], sides[1], W, dy[1], pos, None, False, dtype, B * T * Hkv)
            assert np.array_equal(back[2], dy[2])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_long_sums(capi, dtype):
    """More rows than workgroups that leave sums, of gradients that do not cancel."""
    rng = np.random.default_rng(7)
    B, H, T, d = 2, 3, 40000, 32
    x, dy = normal(rng, (B, H, T, d), dtype), np.abs(normal(rng, (B, H, T, d), dtype))
    w = normal(rng, (d,), "f32")
    dx, dw = capi.DeviceBuffer(x.shape, dtype), capi.DeviceBuffer((d,), "f32")
    X, Y, W = (capi.DeviceBuffer.from_numpy(a, t) for a, t in ((x, dtype), (dy, dtype), (w, "f32")))
    got = []
    for _ in range(3):
        capi.norm_rope_backward(X, Y, dx, W, dw, eps=EPS)
        capi.lib().sync()
        got.append(dw.download())
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])  # the order is fixed
    # R here: what one thread adds up (its tiles, three heads) and the 1024 sums
    check_backward(dx.download(), got[0], x, w, dy, po.positions(B, T), None, False, dtype, 2048)


@pytest.mark.parametrize("B,H,T", [(0, 3, 5), (2, 0, 5), (2, 3, 0)])
def test_no_rows_have_no_gradient(capi, B, H, T):
    d = 64
    W, dw = capi.DeviceBuffer.from_numpy(np.ones(d, np.float32)), capi.DeviceBuffer.from_numpy(np.full(d, 3.0, np.float32))
    x = capi.DeviceBuffer((B, H, T, d))
    capi.norm_rope_backward(x, capi.DeviceBuffer((B, H, T, d)), capi.DeviceBuffer((B, H, T, d)), W, dw)
    capi.norm_rope(x, capi.DeviceBuffer((B, H, T, d)), W)
    capi.lib().sync()
    assert (dw.download() == 0).all()


def test_most_heads(capi):
    """As many heads as the weights' gradients may have, and more without them."""
    rng = np.random.default_rng(9)
    B, T, d, w = 1, 3, 32, normal(rng, (32,), "f32")
    W, F, pos = capi.DeviceBuffer.from_numpy(w), capi.DeviceBuffer.from_numpy(FREQ[32]), po.positions(B, T)
    for H, weight in ((2048, True), (5000, False)):
        x, dy = normal(rng, (B, H, T, d), "bf16"), normal(rng, (B, H, T, d), "bf16")
        X, Y, out = capi.DeviceBuffer.from_numpy(x, "bf16"), capi.DeviceBuffer.from_numpy(dy, "bf16"), capi.DeviceBuffer(x.shape, "bf16")
        dw = capi.DeviceBuffer((d,)) if weight else None
        capi.norm_rope(X, out, W, F, eps=EPS)
        capi.lib().sync()
        check_forward(out.download(), x, w, pos, FREQ[32], False, "bf16")
        capi.norm_rope_backward(X, Y, out, W, dw, F, eps=EPS)
        capi.lib().sync()
        check_backward(out.download(), dw.download() if weight else None, x, w, dy, pos, FREQ[32], False, "bf16", B * T * H)


def test_captured_and_on_another_stream(capi):
    """A step captured once its scratch is there, replayed on new inputs beside eager calls on two streams."""
    rng = np.random.default_rng(8)
    B, H, T, d = 2, 4, 90, 128
    w = normal(rng, (d,), "f32")
    W, F, x = capi.DeviceBuffer.from_numpy(w), capi.DeviceBuffer.from_numpy(FREQ[128]), capi.DeviceBuffer((B, H, T, d))
    dy, y, dx = (capi.DeviceBuffer((B, H, T, d)) for _ in range(3))
    dw = capi.DeviceBuffer((d,))
    st, other = capi.Stream(), capi.Stream()
    mine = [capi.DeviceBuffer((B, H, T, d)) for _ in range(2)] + [capi.DeviceBuffer((d,))]

    def step(s, y, dx, dw):
        capi.norm_rope(x, y, W, F, eps=EPS, stream=s)
        capi.norm_rope_backward(x, dy, dx, W, dw, F, eps=EPS, stream=s)

    def fill():
        a, b = normal(rng, (B, H, T, d), "f32"), normal(rng, (B, H, T, d), "f32")
        x.upload(a)
        dy.upload(b)
        capi.lib().sync()
        return a, b

    def check(a, b, y, dx, dw):
        check_forward(y.download(), a, w, po.positions(B, T), FREQ[128], False, "f32")
        check_backward(dx.download(), dw.download(), a, w, b, po.positions(B, T), FREQ[128], False, "f32", B * H * T)

    fresh = capi.Stream()
    with pytest.raises(capi.TTError, match="scratch"):
        with Capture(capi, fresh.handle, 1):
            step(fresh.handle, y, dx, dw)
    fill()
    step(st.handle, y, dx, dw)
    st.sync()
    with Capture(capi, st.handle, 1) as c:
        step(st.handle, y, dx, dw)
    for _ in range(4):
        a, b = fill()
        c.launch()
        step(other.handle, *mine)
        st.sync()
        other.sync()
        check(a, b, y, dx, dw)
        check(a, b, *mine)
        a, b = fill()
        step(st.handle, *mine)
        st.sync()
        check(a, b, *mine)


def test_rotated_heads_train(capi):
    """norm_rope, attention and their gradients through the graph, against differences of the composition."""
    import operators as ops

    rng = np.random.default_rng(9)
    B, L, H, d = 1, 6, 2, 32
    q, k, v = (rng.standard_normal((B, L, H, d)).astype(np.float32) for _ in range(3))
    wq, wk = (1 + 0.1 * rng.standard_normal(d).astype(np.float32) for _ in range(2))
    go = rng.standard_normal((B, H, L, d)).astype(np.float32)
    freq = ops.rope_frequencies(16)

    def loss(q, k, v, wq, wk):
        pos = po.positions(B, L)
        a = po.norm_rope(q.swapaxes(1, 2), wq, 1e-6, pos, freq, False)
        b = po.norm_rope(k.swapaxes(1, 2), wk, 1e-6, pos, freq, False)
        o, _ = orc.attn_fwd_f64(a, b, v.swapaxes(1, 2).astype(np.float64), float(np.float32(d ** -0.5)), True)
        return (o * go).sum()

    t = [ops.Tensor(a) for a in (q, k, v, wq, wk)]
    a = ops.norm_rope(t[0], t[3], freq, tokens_first=True)
    b = ops.norm_rope(t[1], t[4], freq, tokens_first=True)
    c = ops.norm_rope(t[2], tokens_first=True)  # moved alone
    out = ops.attention(a, b, c, causal=True)
    out.backward(ops.Tensor(go, requires_grad=False))
    assert abs((out.numpy() * go).sum() - loss(q, k, v, wq, wk)) < 1e-4 * np.abs(go).sum()
    h = 1e-4
    data = [x.astype(np.float64) for x in (q, k, v, wq, wk)]
    for n, x in enumerate(data):
        grad = t[n].grad.numpy()
        assert grad.shape == x.shape
        for at in rng.integers(0, x.size, 6):
            i = np.unravel_index(at, x.shape)
            both = []
            for sign in (h, -h):
                moved = [y.copy() for y in data]
                moved[n][i] += sign
                both.append(loss(*moved))
            # a difference is h^2 f''' / 6 off; the fp32 gradient some 1e-5 of the largest
            assert abs((both[0] - both[1]) / (2 * h) - grad[i]) <= 1e-4 * max(1.0, np.abs(grad).max())
