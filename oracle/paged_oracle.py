"""float64 oracle of the operators on either side of attention: norms of heads
with the position rotation, their gradients, the e4m3 numbers and a paged cache.

TEST INFRASTRUCTURE ONLY, like ``attn_oracle``: numpy, written from the
definitions and pinned by brute force in ``tests/test_paged.py``.
"""
from __future__ import annotations

from typing import Optional, Tuple

import numpy as np

E4_MAX = 448.0
# the values of codes 0 .. 126 (127 is NaN): increasing
E4_GRID = np.array([(c & 7) * 2.0 ** -9 if c < 8 else 2.0 ** ((c >> 3) - 7) * (1 + (c & 7) / 8) for c in range(127)])


# ------------------------------------------------------------------ norms and rotation

def positions(B: int, T: int, given: Optional[np.ndarray] = None, lengths: Optional[np.ndarray] = None) -> np.ndarray:
    if given is not None:
        return np.asarray(given, np.float64)
    first = np.zeros(B) if lengths is None else np.asarray(lengths, np.float64) - T
    return first[:, None] + np.arange(T)


def rotate(x: np.ndarray, pos: np.ndarray, freq: Optional[np.ndarray], interleaved: bool, back: bool = False) -> np.ndarray:
    """x [B, H, T, d] with its pairs turned by pos [B, T] times freq (fp32 values), or back."""
    x = np.array(x, np.float64)
    if freq is None:
        return x
    n = len(freq)
    a = pos[:, None, :, None] * np.asarray(freq, np.float64)
    c, s = np.cos(a), -np.sin(a) if back else np.sin(a)
    i, j = (np.s_[..., 0:2 * n:2], np.s_[..., 1:2 * n:2]) if interleaved else (np.s_[..., :n], np.s_[..., n:2 * n])
    p, q = x[i].copy(), x[j].copy()
    x[i], x[j] = p * c - q * s, p * s + q * c
    return x


def norm(x: np.ndarray, w: Optional[np.ndarray], eps: float) -> np.ndarray:
    x = np.asarray(x, np.float64)
    if w is None:
        return x
    return x / np.sqrt(np.mean(x * x, -1, keepdims=True) + np.float64(np.float32(eps))) * np.asarray(w, np.float64)


def norm_rope(x, w, eps, pos, freq, interleaved):
    return rotate(norm(x, w, eps), pos, freq, interleaved)


def norm_rope_backward(x, w, eps, pos, freq, interleaved, dy) -> Tuple[np.ndarray, Optional[np.ndarray]]:
    """dx and dw (None without a weight) for dy [B, H, T, d]."""
    g = rotate(dy, pos, freq, interleaved, back=True)
    if w is None:
        return g, None
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    r = 1.0 / np.sqrt(np.mean(x * x, -1, keepdims=True) + np.float64(np.float32(eps)))
    n = x * r
    return r * (g * w - n * np.mean(g * w * n, -1, keepdims=True)), (g * n).sum((0, 1, 2))


# ------------------------------------------------------------------ e4m3 under one scale byte

def scale_byte(x: np.ndarray) -> int:
    """The byte of the smallest power of two of 2^-124 .. 2^119 that takes x's largest finite value to at most 448."""
    v = np.abs(x[np.isfinite(x)])
    top = v.max() if v.size else 0.0
    e = -124
    while e < 119 and top > np.ldexp(E4_MAX, e):
        e += 1
    return e + 127


def encode(x: np.ndarray, byte: int) -> np.ndarray:
    """Codes of x under a scale byte: nearest, ties to the even code, beyond 448 to 448, infinities and NaN to NaN."""
    x = np.asarray(x, np.float64)
    bad = ~np.isfinite(x)
    r = np.ldexp(np.where(bad, 0.0, x), 127 - int(byte))
    a = np.minimum(np.abs(r), E4_MAX)
    lo = np.searchsorted(E4_GRID, a, side="right") - 1
    hi = np.minimum(lo + 1, 126)
    mid = (E4_GRID[lo] + E4_GRID[hi]) / 2
    c = np.where(a > mid, hi, np.where(a < mid, lo, np.where(lo % 2 == 0, lo, hi)))
    return np.where(bad, 127, c + 128 * np.signbit(r)).astype(np.uint8)


def decode(codes: np.ndarray, byte) -> np.ndarray:
    c = codes.astype(np.int64)
    v = np.where((c & 127) == 127, np.nan, E4_GRID[np.minimum(c & 127, 126)])
    return np.where(c >= 128, -v, v) * np.ldexp(1.0, np.asarray(byte, np.int64) - 127)


# ------------------------------------------------------------------ the paged cache

class Cache:
    """Pools, table and lengths on the host; values of fp32 (of any type) or codes with scale bytes."""

    def __init__(self, npages, hkv, page, d, table, e4m3=False):
        self.page, self.e4m3, self.table = page, e4m3, np.asarray(table, np.int32)
        self.npages, self.hkv, self.d = npages, hkv, d
        shape = (npages, hkv, page, d)
        self.pool = {n: np.zeros(shape, np.uint8 if e4m3 else np.float64) for n in "kv"}
        self.scale = {n: np.zeros((npages, hkv), np.uint8) for n in "kv"}

    def at(self, b, j):
        """Page of key j of sequence b, or None."""
        i = j // self.page
        if j < 0 or i >= self.table.shape[1]:
            return None
        p = int(self.table[b, i])
        return p if 0 <= p < self.npages else None

    def append(self, n, x, lengths):
        """New rows x [B, Hkv, T, d] (float64, K rotated already) of side n."""
        B, hkv, T, _ = x.shape
        for b in range(B):
            tokens = [(int(lengths[b]) - T + t, t) for t in range(T)]
            tokens = [(j, t) for j, t in tokens if self.at(b, j) is not None]
            if not self.e4m3:
                for j, t in tokens:
                    self.pool[n][self.at(b, j), :, j % self.page] = x[b, :, t]
                continue
            for i in sorted({j // self.page for j, _ in tokens}):
                here = [(j % self.page, t) for j, t in tokens if j // self.page == i]
                p, old = self.at(b, i * self.page), here[0][0]
                for h in range(hkv):
                    rows = np.stack([x[b, h, t] for _, t in here])
                    byte, before = scale_byte(rows), int(self.scale[n][p, h])
                    if old:
                        byte = max(byte, before)
                        self.pool[n][p, h, :old] = encode(decode(self.pool[n][p, h, :old], before), byte)
                    self.pool[n][p, h, old:old + len(here)] = encode(rows, byte)
                    self.scale[n][p, h] = byte

    def rows(self, n, b, size):
        """(values [Hkv, size, d], which of them the table has)."""
        out, has = np.zeros((self.hkv, size, self.d)), np.zeros(size, bool)
        for j in range(size):
            p = self.at(b, j)
            if p is None:
                continue
            has[j] = True
            x = self.pool[n][p, :, j % self.page]
            out[:, j] = decode(x, self.scale[n][p][:, None].astype(int)) if self.e4m3 else x
        return out, has

    def attend(self, q, lengths, scale):
        """q [B, H, T, d] -> o, lse, and sum p |v| and the largest sum |q| |k| scale of each row for bounds."""
        B, H, T, d = q.shape
        group = H // self.hkv
        o, lse = np.zeros((B, H, T, d)), np.full((B, H, T), -np.inf)
        mag, score = np.zeros((B, H, T, d)), np.zeros((B, H, T))
        for b in range(B):
            end = min(max(int(lengths[b]), 0), self.table.shape[1] * self.page)
            k, has = self.rows("k", b, end)
            v, _ = self.rows("v", b, end)
            for h in range(H):
                for t in range(T):
                    see = has & (np.arange(end) < int(lengths[b]) - (T - 1 - t))
                    if not see.any():
                        continue
                    kk, vv, qq = k[h // group, see], v[h // group, see], np.asarray(q[b, h, t], np.float64)
                    with np.errstate(invalid="ignore", over="ignore"):
                        s = kk @ qq * scale
                        if (s == -np.inf).all():
                            continue
                        p = np.exp(s - s.max())
                        lse[b, h, t] = s.max() + np.log(p.sum())
                        p /= p.sum()
                        o[b, h, t] = (p[:, None] * vv).sum(0)
                        mag[b, h, t] = (p[:, None] * np.abs(vv)).sum(0)
                        score[b, h, t] = (np.abs(kk) @ np.abs(qq)).max() * abs(scale)
        return o, lse, mag, score
