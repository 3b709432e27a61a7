"""GPU tests of a new workspace whose clearing is reported as failed: the call says
so, gives the buffer back, and the next one on the stream is right."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def capi():
    import tt_capi

    assert tt_capi.lib().device_count() >= 1, "no HIP device visible"
    tt_capi.lib().call("tt_init", 0)
    return tt_capi


def _in_use(capi):
    n = ctypes.c_size_t()
    capi.lib().call("tt_mem_stats", ctypes.byref(n), None)
    return n.value


def _stale_error(capi):
    """A HIP call of this thread that fails on the host, whose error the next launch check finds."""
    hip = ctypes.CDLL(None)
    fn = getattr(hip, "hipSetDevice", None) or ctypes.CDLL("libamdhip64.so").hipSetDevice
    assert fn(1 << 20) != 0


@pytest.mark.parametrize("what", ["decode", "gradients"])
def test_an_error_at_the_clearing(capi, what):
    rng, st, d = np.random.default_rng(1), capi.Stream(), 64
    f = capi.DeviceBuffer.from_numpy
    if what == "decode":
        n, page = 1500, 64
        k, v = (rng.standard_normal((1, 1, n, d)).astype(np.float32) for _ in range(2))
        kp, vp = (capi.DeviceBuffer((24, 1, page, d)) for _ in range(2))
        tab, lengths = f(np.arange(24, dtype=np.int32)[None], "i32"), f(np.array([n], np.int32), "i32")
        capi.kv_append_paged(f(k), f(v), kp, vp, tab, lengths)
        q = rng.standard_normal((1, 1, 1, d)).astype(np.float32)
        Q, o, lse = f(q), capi.DeviceBuffer((1, 1, 1, d)), capi.DeviceBuffer((1, 1, 1))
        call = lambda: capi.attn_decode_paged(Q, kp, vp, tab, lengths, o, lse, 0.125, stream=st.handle)  # noqa: E731
        s = k[0, 0].astype(np.float64) @ q[0, 0, 0] * 0.125
        p = np.exp(s - s.max())
        ref, out = (p[:, None] / p.sum() * v[0, 0]).sum(0), o
    else:
        x, dy = (rng.standard_normal((1, 2, 50, d)).astype(np.float32) for _ in range(2))
        X, DY, dx, w, dw = f(x), f(dy), capi.DeviceBuffer(x.shape), f(np.ones(d, np.float32)), capi.DeviceBuffer((d,))
        call = lambda: capi.norm_rope_backward(X, DY, dx, w, dw, stream=st.handle)  # noqa: E731
        x64 = x.astype(np.float64)
        ref, out = (dy * x64 / np.sqrt((x64 * x64).mean(-1, keepdims=True) + 1e-6)).sum((0, 1, 2)), dw
    capi.lib().sync()
    before = _in_use(capi)
    _stale_error(capi)
    with pytest.raises(capi.TTError):
        call()
    assert _in_use(capi) == before  # given back
    for _ in range(3):
        out.zero()
        capi.lib().sync()
        call()
        st.sync()
        # 1500 keys or 100 rows in fp32: (n + 100) 2^-24 of sums of magnitude below 50
        assert np.abs(out.download().reshape(-1) - ref).max() < 1600 * 2.0 ** -24 * 50
    assert _in_use(capi) > before
