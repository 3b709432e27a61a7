"""GPU tests of calls of the paged cache that its C interface allows beyond what the
wrappers make: K and V as parts of one fused projection or laid out apart, attention
without its log sums, and calls that repeat."""
import numpy as np
import pytest

from oracle import paged_oracle as po
from test_norm_rope_gpu import EPS, FREQ, normal
from test_paged_gpu import KINDS, Cache, capi, filled  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu
CODE = {"f32": 0, "bf16": 3, "u8": 4}


@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("B,T,Hkv", [(2, 21, 3), (140, 60, 5)])
def test_parts_of_a_projection(capi, B, T, Hkv, dtype, cache):  # noqa: F811
    """k and v as columns of [B, T, H + 2 Hkv, d], and k so with v head-major: the bits of separate rows."""
    rng = np.random.default_rng(B)
    H, d, page = 4, 64, 32
    lengths = rng.integers(0, T + 1, B).astype(np.int32)
    f = capi.DeviceBuffer.from_numpy
    x = normal(rng, (B, T, H + 2 * Hkv, d), dtype)
    k, v = x[:, :, H:H + Hkv], x[:, :, H + Hkv:]
    X, F, W = f(x, dtype), f(FREQ[64]), f(1 + normal(rng, (d,), "f32"))
    V = f(np.ascontiguousarray(np.swapaxes(v, 1, 2)), dtype)
    n, item, ld = f(lengths, "i32"), X.ITEM[dtype], (H + 2 * Hkv) * d
    got = []
    for way in range(3):
        c = Cache(capi, dtype, cache, B, Hkv, page, 2, d, np.random.default_rng(5))
        if way == 0:
            capi.kv_append_paged(f(np.ascontiguousarray(k), dtype), f(np.ascontiguousarray(v), dtype), c.dev["k"], c.dev["v"], c.tab, n, W,
                                 F, EPS, None, False, True, **c.scales())
        else:
            at = (X.ptr + item * (H + Hkv) * d, ld) if way == 1 else (V.ptr, 0)
            scales = [s.ptr if s else None for s in c.scale.values()]
            capi.lib().call("tt_kv_append_paged", CODE[dtype], CODE[cache], X.ptr + item * H * d, at[0], ld, at[1], W.ptr, EPS, F.ptr, 64,
                            0, None, c.dev["k"].ptr, c.dev["v"].ptr, *scales, c.tab.ptr, n.ptr, B, Hkv, T, d, c.npages, page, 2, None)
        capi.lib().sync()
        got.append([c.dev[s].download_bytes() for s in "kv"] + [s.download() for s in c.scale.values() if s])
    for other in got[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(other, got[0]))
    ref = po.Cache(c.npages, Hkv, page, d, c.table[:2], cache == "u8")
    ref.append("v", np.swapaxes(v[:2], 1, 2).astype(np.float64), lengths[:2])
    out = got[2][1] if cache == "u8" else c.dev["v"].download()
    pages = np.unique(c.table[:2])
    assert np.array_equal(out[pages], ref.pool["v"][pages])


@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("B,H,Hkv,T,n", [(1, 4, 2, 1, 1500), (1, 6, 1, 3, 1500), (64, 32, 32, 1, 90)])
def test_without_log_sums_and_again(capi, B, H, Hkv, T, n, dtype, cache):  # noqa: F811
    """Splits merged by the last workgroup, by a launch, and none: o has the same bits in every call, with and
    without lse."""
    rng = np.random.default_rng(n + T)
    c = filled(capi, dtype, cache, B, Hkv, 32, 64, [n - (b % 7) for b in range(B)], rng)
    q = normal(rng, (B, H, T, 64), dtype)
    first, lse = c.attend(q, [n - (b % 7) for b in range(B)], 0.125)
    for i in range(6):
        o, again = c.attend(q, [n - (b % 7) for b in range(B)], 0.125, lse=i % 2 == 0)
        assert np.array_equal(o, first) and (again is None or np.array_equal(again, lse))
