"""float64 / integer oracle of the microscaled 4-bit operators: the format, its
product, the cache append and the attention over such a cache.

TEST INFRASTRUCTURE ONLY, like ``attn_oracle``: numpy, written from the
definitions and pinned by brute force in ``tests/test_mxfp4.py``.
"""
from __future__ import annotations

from typing import Tuple

import numpy as np

BLOCK = 32
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def blocks(n: int) -> int:
    return -(-n // BLOCK)


def quantize(x: np.ndarray) -> Tuple[np.ndarray, np.ndarray]:
    """x [.., n] -> codes uint8 [.., 16 nb], scales uint8 [.., nb]."""
    x = np.asarray(x, np.float64)
    n, nb = x.shape[-1], blocks(x.shape[-1])
    v = np.zeros((*x.shape[:-1], nb * BLOCK))
    v[..., :n] = x
    v = v.reshape(*x.shape[:-1], nb, BLOCK)
    bad = ~np.isfinite(v).all(-1)
    top = np.abs(np.where(np.isfinite(v), v, 0.0)).max(-1)
    e = np.where(top > 0, np.frexp(np.where(top > 0, top, 1.0))[1] - 1, -200)  # floor(log2 top)
    s = np.maximum(e - 2, -127)
    a = np.minimum(np.abs(np.where(bad[..., None], 0.0, v)) * np.ldexp(1.0, -s)[..., None], 6.0)
    # nearest grid value; a tie goes to the even code
    lo = np.searchsorted(GRID, a, side="right") - 1
    hi = np.minimum(lo + 1, 7)
    mid = (GRID[lo] + GRID[hi]) / 2
    code = np.where(a > mid, hi, np.where(a < mid, lo, np.where(lo % 2 == 0, lo, hi)))
    code = np.where(lo == hi, lo, code)
    code = np.where(bad[..., None], 0, code + 8 * np.signbit(v)).astype(np.uint8)
    codes = (code[..., 0::2] | (code[..., 1::2] << 4)).reshape(*x.shape[:-1], nb * BLOCK // 2)
    return codes, np.where(bad, 255, s + 127).astype(np.uint8)


def dequantize(codes: np.ndarray, scales: np.ndarray, n: int) -> np.ndarray:
    """The values [.., n] in float64."""
    c = np.stack((codes & 15, codes >> 4), -1).reshape(*scales.shape, BLOCK).astype(np.int64)
    v = np.where(c & 8, -1.0, 1.0) * GRID[c & 7] * np.ldexp(1.0, scales.astype(np.int64) - 127)[..., None]
    v[scales == 255] = np.nan
    return v.reshape(*scales.shape[:-1], -1)[..., :n]


def append(k_codes, k_scales, new, lengths):
    """The cache's codes and scales with the new rows [B, Hkv, T, d] in place."""
    codes, scales = k_codes.copy(), k_scales.copy()
    T, cap = new.shape[2], codes.shape[2]
    nc, ns = quantize(new)
    for b, n in enumerate(lengths):
        for t in range(T):
            at = int(n) - T + t
            if 0 <= at < cap:
                codes[b, :, at], scales[b, :, at] = nc[b, :, t], ns[b, :, t]
    return codes, scales


def decode(q, k, v, lengths, scale: float):
    """q [B, H, T, d] over the values k, v [B, Hkv, cap, d] -> o, lse, and the
    two magnitudes that an error bound needs: each row's sum p |v| [B, H, T, d]
    and its largest seen sum |q_i| |k_i| scale [B, H, T]."""
    q = np.asarray(q, np.float64)
    B, H, T, d = q.shape
    Hkv, cap = k.shape[1], k.shape[2]
    o, lse = np.zeros(q.shape), np.full(q.shape[:3], -np.inf)
    mag, smax = np.zeros(q.shape), np.zeros(q.shape[:3])
    for b in range(B):
        for h in range(H):
            kh, vh = k[b, h // (H // Hkv)], v[b, h // (H // Hkv)]
            for t in range(T):
                n = min(int(lengths[b]) - (T - 1 - t), cap)
                if n <= 0:
                    continue
                s = kh[:n] @ q[b, h, t] * scale
                m = s.max()
                p = np.exp(s - m)
                o[b, h, t] = p @ vh[:n] / p.sum()
                lse[b, h, t] = m + np.log(p.sum())
                mag[b, h, t] = p @ np.abs(vh[:n]) / p.sum()
                smax[b, h, t] = (np.abs(kh[:n]) @ np.abs(q[b, h, t])).max() * abs(scale)
    return o, lse, mag, smax
