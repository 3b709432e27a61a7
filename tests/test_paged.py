"""CPU tests of norms and rotation of heads and of the paged cache: the oracle
against brute force and differences, and every refusal of the C-ABI and of its
Python binding, none of which needs a device."""

import numpy as np
import pytest

from oracle import paged_oracle as po


@pytest.fixture(scope="module")
def capi():
    import tt_capi

    return tt_capi


# ------------------------------------------------------------------ the oracle

@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_is_a_complex_product(interleaved):
    rng = np.random.default_rng(1)
    x, pos, f = rng.standard_normal((2, 3, 5, 32)), np.array([[0, 1, 7, 100, 9999]] * 2), np.float32([1.0, 0.1, 0.01, 0.5] * 2)
    y = po.rotate(x, pos, f, interleaved)
    for i in range(8):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + 8)
        z = (x[..., a] + 1j * x[..., b]) * np.exp(1j * pos[:, None] * float(f[i]))
        assert np.allclose(y[..., a], z.real, atol=1e-12) and np.allclose(y[..., b], z.imag, atol=1e-12)
    assert np.array_equal(y[..., 16:], x[..., 16:])
    assert np.allclose(po.rotate(y, pos, f, interleaved, back=True), x, atol=1e-12)


@pytest.mark.parametrize("weight", [True, False])
def test_gradients_by_differences(weight):
    rng = np.random.default_rng(2)
    x, dy = rng.standard_normal((2, 2, 3, 32)), rng.standard_normal((2, 2, 3, 32))
    w = 1 + 0.1 * rng.standard_normal(32) if weight else None
    pos, f = po.positions(2, 3, lengths=[9, 4]), np.float32(10000.0 ** (-np.arange(8) / 8))

    def loss(x, w):
        return (po.norm_rope(x, w, 1e-3, pos, f, False) * dy).sum()

    dx, dw = po.norm_rope_backward(x, w, 1e-3, pos, f, False, dy)
    h = 1e-6
    for at in [(0, 0, 0, 0), (1, 1, 2, 9), (0, 1, 1, 20), (1, 0, 0, 31)]:
        up, down = x.copy(), x.copy()
        up[at] += h
        down[at] -= h
        assert abs((loss(up, w) - loss(down, w)) / (2 * h) - dx[at]) < 1e-7
    for i in range(0, 32, 5) if weight else ():
        e = np.eye(32)[i] * h
        assert abs((loss(x, w + e) - loss(x, w - e)) / (2 * h) - dw[i]) < 1e-6


def test_e4m3_by_brute_force():
    every = po.decode(np.arange(256, dtype=np.uint8), 127)
    assert np.isnan(every[[127, 255]]).all() and every[126] == 448 and every[1] == 2.0 ** -9 and every[56] == 1.0
    rng = np.random.default_rng(3)
    x = np.concatenate([rng.standard_normal(300) * 2.0 ** rng.integers(-12, 9, 300), (every[:126] + every[1:127]) / 2])
    c = po.encode(x, 127)
    for v, code in zip(x, c):
        d = np.abs(po.E4_GRID - min(abs(v), 448.0))
        near = np.flatnonzero(d == d.min())
        want = near[0] if len(near) == 1 else near[near % 2 == 0][0]
        assert code == want + 128 * (v < 0)
    assert np.array_equal(po.decode(po.encode(every[:127], 127), 127), every[:127])
    assert po.scale_byte(np.array([448.0])) == 127 and po.scale_byte(np.array([448.5])) == 128
    assert po.scale_byte(np.array([0.0])) == 3 and po.scale_byte(np.array([3.4e38])) == 246
    assert po.scale_byte(np.array([1.0, np.inf, np.nan])) == po.scale_byte(np.array([1.0])) == 119
    assert list(po.encode(np.array([np.inf, -np.inf, np.nan, -0.0, 1e30]), 127)) == [127, 127, 127, 128, 126]


def test_cache_by_definition():
    """One token at a time gives the rows of a prompt at once, and pages scale up as values grow."""
    rng = np.random.default_rng(4)
    x = rng.standard_normal((2, 1, 40, 32)) * np.exp(0.1 * np.arange(40))[:, None]
    table = [[5, 0, 3], [1, -1, 4]]
    a, b = po.Cache(6, 1, 16, 32, table), po.Cache(6, 1, 16, 32, table)
    a.append("k", x, [40, 38])
    for j in range(40):
        b.append("k", x[:, :, j:j + 1], [j + 1, j - 1])
    assert np.array_equal(a.pool["k"], b.pool["k"])
    rows, has = a.rows("k", 1, 38)
    assert np.array_equal(has, (np.arange(38) < 16) | (np.arange(38) >= 32))
    assert np.array_equal(rows[:, has], x[1][:, 2:][:, has])
    e = po.Cache(6, 1, 16, 32, table, e4m3=True)
    for j in range(40):
        e.append("k", x[:1, :, j:j + 1].repeat(2, 0), [j + 1, 0])
    got, _ = e.rows("k", 0, 40)
    for i in range(3):
        rows = x[0, :, 16 * i:16 * (i + 1)]
        byte = po.scale_byte(rows)
        assert e.scale["k"][table[0][i], 0] == byte
        assert np.abs(got[:, 16 * i:16 * (i + 1)] - rows).max() <= 2.0 ** -4 * np.abs(rows).max()


# ------------------------------------------------------------------ refusals

P = 1 << 20  # an address: nothing is read or written before the checks


def rope(capi, **kw):
    a = dict(dtype=capi.TT_F32, q=P, k=2 * P, v=3 * P, ldq=0, ldk=0, ldv=0, wq=4 * P, wk=5 * P, eps=1e-6, freq=6 * P, rot=32,
             inter=0, pos=None, len=None, qo=7 * P, ko=8 * P, vo=9 * P, B=2, H=4, Hkv=2, T=3, d=64)
    assert set(kw) <= set(a)
    return "tt_qkv_norm_rope", [*{**a, **kw}.values(), None]


def rope_back(capi, **kw):
    a = dict(dtype=capi.TT_F32, q=P, k=2 * P, ldq=0, ldk=0, wq=4 * P, wk=5 * P, eps=1e-6, freq=6 * P, rot=32, inter=0, pos=None,
             len=None, dqo=7 * P, dko=8 * P, dvo=9 * P, dq=10 * P, dk=11 * P, dv=12 * P, lddq=0, lddk=0, lddv=0, dwq=13 * P,
             dwk=14 * P, B=2, H=4, Hkv=2, T=3, d=64)
    assert set(kw) <= set(a)
    return "tt_qkv_norm_rope_backward", [*{**a, **kw}.values(), None]


def append(capi, **kw):
    a = dict(dtype=capi.TT_F32, cache=capi.TT_F32, k=P, v=2 * P, ldk=0, ldv=0, wk=3 * P, eps=1e-6, freq=4 * P, rot=32, inter=0,
             pos=None, kp=5 * P, vp=6 * P, ks=7 * P, vs=8 * P, table=9 * P, len=10 * P, B=2, Hkv=2, T=3, d=64, npages=7, page=16,
             width=3)
    assert set(kw) <= set(a)
    return "tt_kv_append_paged", [*{**a, **kw}.values(), None]


def gather(capi, **kw):
    a = dict(dtype=capi.TT_F32, cache=capi.TT_F32, kp=5 * P, vp=6 * P, ks=7 * P, vs=8 * P, table=9 * P, len=10 * P, k=P, v=2 * P,
             B=2, Hkv=2, L=30, d=64, npages=7, page=16, width=3)
    assert set(kw) <= set(a)
    return "tt_kv_gather_paged", [*{**a, **kw}.values(), None]


def decode(capi, **kw):
    a = dict(dtype=capi.TT_F32, cache=capi.TT_F32, q=P, kp=5 * P, vp=6 * P, ks=7 * P, vs=8 * P, table=9 * P, len=10 * P, o=2 * P,
             lse=3 * P, B=2, H=4, Hkv=2, T=3, d=64, npages=7, page=16, width=3, scale=0.125)
    assert set(kw) <= set(a)
    return "tt_attn_decode_paged", [*{**a, **kw}.values(), None]


def refused(capi, what, code, words):
    name, args = what
    rc = getattr(capi.lib().lib, name)(*args)
    assert rc == code, (rc, capi.lib().last_error())
    assert words in capi.lib().last_error() and name in capi.lib().last_error()


ARG, UNSUPPORTED = 1, 3


@pytest.mark.parametrize("kw,words", [
    (dict(dtype=1), "dtype"), (dict(B=-1), "negative"), (dict(T=-1), "negative"), (dict(H=-1), "negative"),
    (dict(H=1 << 21), "too many heads"), (dict(B=1 << 16, T=1 << 15), "too many tokens"), (dict(rot=24), "rot"),
    (dict(rot=80), "rot"), (dict(rot=-16), "rot"), (dict(inter=2), "interleaved"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(q=None), "both"), (dict(vo=None), "both"), (dict(k=2 * P + 4), "aligned"),
    (dict(qo=7 * P + 8), "aligned"), (dict(ldq=128), "leading"), (dict(ldk=130), "leading"), (dict(ldv=-128), "leading"),
    (dict(ldq=(1 << 31) + 4), "leading"), (dict(qo=P), "overlaps"), (dict(ko=7 * P + 64), "overlaps"),
    (dict(vo=4 * P - 64), "overlaps"), (dict(ko=6 * P), "overlaps"), (dict(qo=1 << 22, pos=(1 << 22) + 16), "overlaps")])
def test_rotation_refusals(capi, kw, words):
    refused(capi, rope(capi, **kw), ARG, words)


def test_head_dim_refusals(capi):
    for call in (rope, rope_back, append, gather, decode):
        refused(capi, call(capi, d=96), UNSUPPORTED, "head dim")


@pytest.mark.parametrize("kw,words", [
    (dict(dtype=2), "dtype"), (dict(Hkv=-1), "negative"), (dict(rot=8), "rot"), (dict(dq=None), "both"), (dict(dvo=None), "both"),
    (dict(wq=None), "not given"), (dict(dq=None, dqo=None), "comes with"), (dict(q=None), "normed"), (dict(k=None), "normed"),
    (dict(lddq=64), "leading"), (dict(lddq=(1 << 31) + 256), "leading"), (dict(dqo=7 * P + 4), "aligned"),
    (dict(q=P + 2), "aligned"), (dict(dv=12 * P + 8), "aligned"), (dict(dq=P), "overlaps"), (dict(dk=10 * P + 64), "overlaps"),
    (dict(dwq=13 * P, dwk=13 * P + 64), "overlaps"), (dict(dwq=10 * P + 4), "overlaps"), (dict(dwk=P), "overlaps"),
    # parts of one fused gradient whose columns meet, or whose rows are of other lengths
    (dict(lddq=512, lddk=512, lddv=512, dk=10 * P + 4 * 192, dv=10 * P + 4 * 384), "overlaps"),
    (dict(lddq=512, lddk=516, lddv=512, dk=10 * P + 4 * 256, dv=10 * P + 4 * 384), "overlaps"),
    (dict(lddq=448, lddk=448, lddv=448, dk=10 * P + 4 * 256, dv=10 * P + 4 * 384), "overlaps")])
def test_rotation_gradient_refusals(capi, kw, words):
    refused(capi, rope_back(capi, **kw), ARG, words)


def test_heads_of_weight_gradients(capi):
    big = dict(H=2047, Hkv=2, T=1, B=1, d=32, dq=1 << 26, dqo=1 << 27, q=1 << 28)
    refused(capi, rope_back(capi, **big), ARG, "too many heads for the weights")


CACHE = [(dict(dtype=4), "dtype"), (dict(cache=3), "cache"), (dict(cache=1), "cache"), (dict(B=-1), "negative"),
         (dict(npages=-1), "negative"), (dict(width=-1), "negative"), (dict(width=1 << 27), "too long"),
         (dict(B=1 << 25), "too many heads"), (dict(B=1 << 13, Hkv=1 << 12, **{}), "too many heads"),
         (dict(npages=1 << 31), "too many pages"), (dict(Hkv=1 << 23, B=1, npages=1 << 30), "too many pages"),
         (dict(kp=None), "null"), (dict(table=None), "null"), (dict(len=None), "null"), (dict(kp=5 * P + 8), "aligned"),
         (dict(cache=4, ks=None), "scales")]


@pytest.mark.parametrize("call", [append, gather, decode])
@pytest.mark.parametrize("kw,words", CACHE)
def test_paged_refusals(capi, call, kw, words):
    if call is decode and "Hkv" in kw:
        kw = {**kw, "H": kw["Hkv"]}
    refused(capi, call(capi, **kw), ARG, words)


@pytest.mark.parametrize("call", [append, gather, decode])
@pytest.mark.parametrize("page", [0, 8, 24, 256, -16])
def test_page_refusals(capi, call, page):
    refused(capi, call(capi, page=page), UNSUPPORTED, "pages hold")


@pytest.mark.parametrize("kw,words", [
    (dict(rot=72), "rot"), (dict(inter=-1), "interleaved"), (dict(eps=-0.5), "eps"), (dict(ldk=64), "leading"),
    (dict(ldv=131), "leading"), (dict(k=None), "null"), (dict(v=2 * P + 4), "aligned"), (dict(kp=P), "overlaps"),
    (dict(vp=5 * P + 64), "overlap"), (dict(cache=4, vs=7 * P + 4), "overlap"), (dict(kp=9 * P), "overlaps"),
    (dict(T=(1 << 30) + 1), "too long"), (dict(B=2, T=1 << 30), "too many tokens")])
def test_append_refusals(capi, kw, words):
    refused(capi, append(capi, **kw), ARG, words)


@pytest.mark.parametrize("kw,words", [(dict(k=None), "null"), (dict(v=2 * P + 4), "aligned"), (dict(k=5 * P), "overlaps"),
                                      (dict(v=P + 64), "overlap"), (dict(L=(1 << 30) + 1), "too long")])
def test_gather_refusals(capi, kw, words):
    refused(capi, gather(capi, **kw), ARG, words)


@pytest.mark.parametrize("kw,words", [
    (dict(H=5), "multiple"), (dict(H=-2), "multiple"), (dict(Hkv=0), "multiple"), (dict(q=None), "null"), (dict(o=None), "null"),
    (dict(q=P + 4), "aligned"), (dict(o=P), "overlaps"), (dict(o=5 * P), "overlaps"), (dict(lse=2 * P), "overlap"),
    (dict(H=1 << 25, Hkv=1), "too many heads"), (dict(B=1 << 10, H=1 << 10, T=1 << 12), "too many rows"),
    (dict(B=1 << 23, H=4, Hkv=2, T=16), "too many"), (dict(B=1 << 11, Hkv=1, H=1 << 12, T=128), "too large")])
def test_decode_refusals(capi, kw, words):
    refused(capi, decode(capi, **kw), ARG, words)


def test_fused_parts_are_accepted_by_the_overlap_check(capi):
    """Parts side by side in one matrix pass the checks: what fails, if anything, is the missing device."""
    if capi.lib().device_count():
        pytest.skip("would run on the device")
    name, args = rope_back(capi, lddq=512, lddk=512, lddv=512, dk=10 * P + 4 * 256, dv=10 * P + 4 * 384)
    assert getattr(capi.lib().lib, name)(*args) == 2, capi.lib().last_error()
    name, args = rope(capi, ldq=512, ldk=512, ldv=512, k=P + 4 * 256, v=P + 4 * 384)
    assert getattr(capi.lib().lib, name)(*args) == 2, capi.lib().last_error()


@pytest.mark.parametrize("call,kw", [
    *((rope, dict([kw])) for kw in (("B", 0), ("T", 0))), (rope, dict(H=0, Hkv=0)),
    *((append, {n: 0}) for n in ("B", "T", "Hkv", "npages", "width")),
    *((gather, {n: 0}) for n in ("B", "L", "Hkv", "npages", "width")),
    *((decode, {n: 0}) for n in ("B", "T", "H")), (decode, dict(H=0, Hkv=0))])
def test_empty_calls(capi, call, kw):
    name, args = call(capi, **kw)
    assert getattr(capi.lib().lib, name)(*args) == 0, capi.lib().last_error()


class Fake:
    def __init__(self, shape, dtype):
        self.shape, self.dtype, self.ptr = tuple(shape), dtype, P
        self.nbytes = int(np.prod(shape)) * {"f32": 4, "bf16": 2, "i32": 4, "u8": 1}[dtype]
        self.ITEM = {"f32": 4, "bf16": 2, "i32": 4, "u8": 1}


def test_binding_refusals(capi):
    f = lambda *s: Fake(s, "f32")  # noqa: E731
    i = lambda *s: Fake(s, "i32")  # noqa: E731
    u = lambda *s: Fake(s, "u8")  # noqa: E731
    bad = [lambda: capi.norm_rope(f(2, 3, 4, 64), f(2, 4, 3, 64)),
           lambda: capi.norm_rope(f(2, 3, 4, 64), f(2, 3, 4, 64), tokens_first=True),
           lambda: capi.norm_rope(f(2, 3, 4, 64), Fake((2, 3, 4, 64), "bf16")),
           lambda: capi.norm_rope(f(2, 3, 4, 64), f(2, 3, 4, 64), weight=f(32)),
           lambda: capi.norm_rope(f(2, 3, 4, 64), f(2, 3, 4, 64), positions=i(2, 3)),
           lambda: capi.norm_rope(f(2, 3, 4, 64), f(2, 3, 4, 64), lengths=f(2)),
           lambda: capi.norm_rope(f(2, 3, 4, 64), f(2, 3, 4, 64), inv_freq=i(32)),
           lambda: capi.norm_rope_backward(f(2, 3, 4, 64), f(2, 3, 4, 64), f(2, 3, 4, 32)),
           lambda: capi.norm_rope_backward(None, f(2, 3, 4, 64), f(2, 3, 4, 64), weight=f(64), dweight=f(65)),
           lambda: capi.qkv_norm_rope(f(2, 4, 6, 64), f(2, 3, 4, 64), f(2, 2, 4, 64), f(2, 2, 4, 64)),
           lambda: capi.qkv_norm_rope(f(2, 4, 7, 64), f(2, 3, 4, 64), f(2, 2, 4, 64), f(2, 1, 4, 64)),
           lambda: capi.qkv_norm_rope_backward(f(2, 4, 7, 64), f(2, 3, 4, 64), f(2, 2, 4, 64), f(2, 2, 4, 64), f(2, 4, 8, 64)),
           lambda: capi.kv_append_paged(f(2, 2, 3, 64), f(2, 2, 3, 64), f(7, 2, 16, 64), f(7, 2, 16, 32), i(2, 3), i(2)),
           lambda: capi.kv_append_paged(f(2, 3, 3, 64), f(2, 3, 3, 64), f(7, 2, 16, 64), f(7, 2, 16, 64), i(2, 3), i(2)),
           lambda: capi.kv_append_paged(f(2, 2, 3, 64), f(2, 2, 3, 64), u(7, 2, 16, 64), u(7, 2, 16, 64), i(2, 3), i(2)),
           lambda: capi.kv_append_paged(f(2, 2, 3, 64), f(2, 2, 3, 64), f(7, 2, 16, 64), f(7, 2, 16, 64), i(2, 3), i(2),
                                        k_scales=u(7, 2), v_scales=u(7, 2)),
           lambda: capi.kv_append_paged(f(2, 2, 3, 64), f(2, 2, 3, 64), f(7, 2, 16, 64), f(7, 2, 16, 64), f(2, 3), i(2)),
           lambda: capi.kv_gather_paged(f(7, 2, 16, 64), f(7, 2, 16, 64), i(2, 3), i(3), f(2, 2, 9, 64), f(2, 2, 9, 64)),
           lambda: capi.kv_gather_paged(f(7, 2, 16, 64), f(7, 2, 16, 64), i(2, 3), i(2), f(2, 2, 9, 64), f(2, 2, 8, 64)),
           lambda: capi.attn_decode_paged(f(2, 4, 1, 64), f(7, 2, 16, 64), f(7, 2, 16, 64), i(2, 3), i(2), f(2, 4, 2, 64), None, 1.0),
           lambda: capi.attn_decode_paged(f(2, 4, 1, 64), f(7, 2, 16, 64), f(7, 2, 16, 64), i(2, 3), i(2), f(2, 4, 1, 64), f(2, 4), 1.0),
           lambda: capi.attn_decode_paged(f(2, 4, 1, 64), u(7, 2, 16, 64), u(7, 2, 16, 64), i(2, 3), i(2), f(2, 4, 1, 64), None, 1.0,
                                          k_scales=u(7, 2), v_scales=u(7, 3))]
    for n, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {n} was accepted")


def test_graph_op_refusals():
    import operators as ops

    for kw, words in ((dict(positions=np.arange(5)), "positions"), (dict(inv_freq=np.ones((2, 8))), "frequency"),
                      (dict(dtype="float64"), "dtype")):
        with pytest.raises(ValueError, match=words):
            ops.NormRope(**kw)


def test_frequencies():
    import operators as ops

    f = ops.rope_frequencies(64, 500000.0)
    assert f.dtype == np.float32 and f.shape == (32,) and f[0] == 1.0
    assert np.allclose(f, 500000.0 ** (-np.arange(32) / 32), rtol=1e-6)
