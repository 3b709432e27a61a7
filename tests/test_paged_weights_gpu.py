"""GPU test of the attention's weights where they meet V: keys of almost equal scores, whose
values cancel, so that the last bits of the weights are what is left of the sums.

q is 1 in one column and K holds the scores there, -0.03 to 0, so that they are exact.
A weight is off by 3 u 0.03 (log2 e, the product, the maximum's) and by one unit of exp2,
2 u; products are exact in their bf16 terms, their sums over six keys and three terms
round nine times, the sum of the weights six and the quotient once, with u = 2^-24: 19 u
of sum p |v| / sum p, and the store's half step."""
import numpy as np
import pytest

from oracle import attn_oracle as orc
from oracle import paged_oracle as po
from test_norm_rope_gpu import HALF, U
from test_paged_gpu import KINDS, capi  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("d", [32, 64, 128])
def test_weights_of_values_that_cancel(capi, d, dtype, cache):  # noqa: F811
    rng = np.random.default_rng(d)
    B, page, n = 4096, 16, 6
    if cache == "u8":  # multiples of 2^-9 under a scale of one
        kc = rng.integers(0, 16, (B, n)).astype(np.uint8)
        kc[:, 0] = 0
        k = -po.E4_GRID[kc]
    else:
        k = -(rng.random((B, n)) * 0.03).astype(np.float32)
        k = (orc.bf16_round(k) if cache == "bf16" else k).astype(np.float64)
        k[:, 0] = 0.0
    p = np.exp(k)  # the largest score is 0
    # each key's row takes back what the ones before it have left, as far as its type goes
    v, left = np.zeros((B, n, d)), np.zeros((B, d))
    byte, codes = 127 - 8, np.zeros((B, 1, page, d), np.uint8)
    for j in range(n):
        x = rng.uniform(0.5, 1.0, (B, d)) if j == 0 else -left / p[:, j:j + 1]
        if cache == "u8":
            if j == 0:
                x[:, 0] = 1.0
            codes[:, 0, j] = po.encode(x, byte)
            x = po.decode(codes[:, 0, j], byte)
        else:
            x = (orc.bf16_round(x.astype(np.float32)) if cache == "bf16" else x.astype(np.float32)).astype(np.float64)
        v[:, j] = x
        left += p[:, j:j + 1] * x
    f = capi.DeviceBuffer.from_numpy
    q = np.zeros((B, 1, 1, d), np.float32)
    q[..., 5] = 1.0
    more = {}
    if cache == "u8":
        kp = np.zeros((B, 1, page, d), np.uint8)
        kp[:, 0, :n, 5] = kc | 128
        K, V = f(kp, "u8"), f(codes, "u8")
        more = dict(k_scales=f(np.full((B, 1), 127, np.uint8), "u8"), v_scales=f(np.full((B, 1), byte, np.uint8), "u8"))
    else:
        kp, vp = np.zeros((B, 1, page, d), np.float32), np.zeros((B, 1, page, d), np.float32)
        kp[:, 0, :n, 5], vp[:, 0, :n] = k, v
        K, V = f(kp, cache), f(vp, cache)
    tab, lengths = f(np.arange(B, dtype=np.int32)[:, None], "i32"), f(np.full(B, n, np.int32), "i32")
    o = capi.DeviceBuffer(q.shape, dtype)
    capi.attn_decode_paged(f(q, dtype), K, V, tab, lengths, o, None, 1.0, **more)
    capi.lib().sync()
    total = p.sum(1)[:, None]
    ref, mag = left / total, (p[..., None] * np.abs(v)).sum(1) / total
    off = np.abs(o.download()[:, 0, 0] - ref) - HALF[dtype] * np.abs(ref)
    assert float(np.abs(ref).max()) < 2.0 ** -12  # they do cancel
    worst = float((off / mag).max() / U)
    assert worst <= 19, worst
