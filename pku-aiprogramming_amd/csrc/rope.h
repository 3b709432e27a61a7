// Device-side building blocks of the kernels that norm and rotate heads.
//
// A head is a row of D values; rotating it by position p turns pair i (of
// rot / 2 pairs) by the angle p f_i: (a, b) -> (a c - b s, a s + b c).  Pair i is
// elements i and i + rot / 2, or 2 i and 2 i + 1 (INTER); elements from rot on
// stay.  A norm is x / sqrt(mean x^2 + eps) times a weight.
//
// A lane holds 16 bytes of each side of its pairs: two chunks of N values (8
// bf16, 4 fp32), so LPR = D / 2N lanes hold a row, no value crosses lanes for the
// rotation, and every load is 16 bytes wide.  Chunks p and p + rot / 2N belong to
// lane p (INTER: 2p and 2p + 1); lanes past the rotated part take the rest two
// by two.  rot is a multiple of 16, so a lane's values turn all or none.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "attn_common.h"

namespace tt {

// What both sides of a pair have in common, in a kernel's arguments.
struct Rope {
  const float* freq;     // [rot / 2]; null: nothing is rotated
  const int* positions;  // [B][T], or null
  const int* lengths;    // [B]: token t is at lengths[b] - T + t; null (and no positions): at t
  int rot, inter;
  float eps;
};

template <typename T> struct Chunk;  // 16 bytes of a row as floats
template <> struct Chunk<u16> {
  static constexpr int N = 8;
  __device__ static __forceinline__ void get(const uint4& v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ static __forceinline__ uint4 put(const float* f) {
    return uint4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
  }
};
template <> struct Chunk<float> {
  static constexpr int N = 4;
  __device__ static __forceinline__ void get(const uint4& v, float* f) { __builtin_memcpy(f, &v, 16); }
  __device__ static __forceinline__ uint4 put(const float* f) {
    uint4 v;
    __builtin_memcpy(&v, f, 16);
    return v;
  }
};

// Where lane p's two chunks lie in a row, in values, and its first pair.
template <int N>
struct Lay {
  int a, b, pair;
  bool turns;
  __device__ __forceinline__ Lay(int p, int rot, bool inter) {
    pair = p * N;
    turns = 2 * pair < rot;
    if (inter || !turns) {
      a = 2 * pair;
      b = a + N;
    } else {
      a = pair;
      b = pair + rot / 2;
    }
  }
};

// The angle p f in 64 bits less the nearest multiple of pi / 2, and that multiple
// modulo 4 (Cody and Waite's reduction: pi / 2 in two parts, each taken off by one
// fused multiply and add, so what is left is as exact as p f itself).
__device__ __forceinline__ double rope_reduce(double angle, int* quadrant) {
  constexpr double kTwoOverPi = 0.63661977236758134308, kHi = 1.57079632679489661923, kLo = 6.12323399573676603587e-17;
  const double k = __builtin_rint(angle * kTwoOverPi);
  *quadrant = (int)(k - 4.0 * __builtin_floor(0.25 * k));
  return __builtin_fma(-k, kLo, __builtin_fma(-k, kHi, angle));
}
// sin and cos of r in [-pi / 4, pi / 4] by their series, up to the first term below
// a last place (1.8e-9 and 1.2e-10 in 32 bits, 5e-17 and 2e-18 in 64).
template <typename F>
__device__ __forceinline__ void rope_series(F r, F* s, F* c) {
  const F x = r * r;
  if constexpr (sizeof(F) == 8) {
    F u = F(-1.0 / 1307674368000.0), v = F(1.0 / 20922789888000.0);
    v = __builtin_fma(v, x, F(-1.0 / 87178291200.0));
    u = __builtin_fma(u, x, F(1.0 / 6227020800.0));
    v = __builtin_fma(v, x, F(1.0 / 479001600.0));
    u = __builtin_fma(u, x, F(-1.0 / 39916800.0));
    v = __builtin_fma(v, x, F(-1.0 / 3628800.0));
    u = __builtin_fma(u, x, F(1.0 / 362880.0));
    v = __builtin_fma(v, x, F(1.0 / 40320.0));
    u = __builtin_fma(u, x, F(-1.0 / 5040.0));
    v = __builtin_fma(v, x, F(-1.0 / 720.0));
    u = __builtin_fma(u, x, F(1.0 / 120.0));
    v = __builtin_fma(v, x, F(1.0 / 24.0));
    u = __builtin_fma(u, x, F(-1.0 / 6.0));
    v = __builtin_fma(v, x, F(-0.5));
    *s = __builtin_fma(u * x, r, r);
    *c = __builtin_fma(v, x, F(1.0));
  } else {
    F u = F(1.0 / 362880.0), v = F(-1.0 / 3628800.0);
    v = __builtin_fmaf(v, x, F(1.0 / 40320.0));
    u = __builtin_fmaf(u, x, F(-1.0 / 5040.0));
    v = __builtin_fmaf(v, x, F(-1.0 / 720.0));
    u = __builtin_fmaf(u, x, F(1.0 / 120.0));
    v = __builtin_fmaf(v, x, F(1.0 / 24.0));
    u = __builtin_fmaf(u, x, F(-1.0 / 6.0));
    v = __builtin_fmaf(v, x, F(-0.5));
    *s = __builtin_fmaf(u * x, r, r);
    *c = __builtin_fmaf(v, x, F(1.0));
  }
}
// cos and sin of position pos times the N frequencies from `freq` on.  The angle
// is formed and reduced in 64 bits: at position 131072 the product alone, rounded
// to 32, would be 0.004 off.
template <int N, typename F>
__device__ __forceinline__ void rope_angles(const float* freq, int64_t pos, F (&c)[N], F (&s)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    int quadrant;
    const F r = (F)rope_reduce((double)pos * (double)freq[i], &quadrant);
    F x, y;
    rope_series(r, &x, &y);
    const F cc = (quadrant & 1) ? x : y, ss = (quadrant & 1) ? y : x;
    c[i] = (quadrant == 1 || quadrant == 2) ? -cc : cc;
    s[i] = (quadrant & 2) ? -ss : ss;
  }
}
// The position of token t of sequence b.
__device__ __forceinline__ int64_t rope_position(const Rope& rp, int64_t b, int64_t t, int64_t T) {
  if (rp.positions) return rp.positions[b * T + t];
  return (rp.lengths ? (int64_t)rp.lengths[b] - T : 0) + t;
}

__device__ __forceinline__ float rope_fma(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double rope_fma(double a, double b, double c) { return __builtin_fma(a, b, c); }

// Sum over the LPR neighbouring lanes that hold a row, the same in each.
template <int LPR, typename F>
__device__ __forceinline__ F row_sum(F x) {
#pragma unroll
  for (int off = 1; off < LPR; off <<= 1) x += __shfl_xor(x, off, 64);
  return x;
}

// The operations below are spelled out, so that every kernel gives a row the same bits.

// A lane's 2 N values with its pairs turned: pair j is values j and N + j, or INTER
// 2 j and 2 j + 1.
template <int N, typename F>
__device__ __forceinline__ void rope_turn(F (&x)[2 * N], const F (&c)[N], const F (&s)[N], bool inter) {
#pragma clang fp contract(off)
  if (inter) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const F a = x[2 * j], b = x[2 * j + 1];
      x[2 * j] = rope_fma(a, c[j], -(b * s[j]));
      x[2 * j + 1] = rope_fma(a, s[j], b * c[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const F a = x[j], b = x[N + j];
      x[j] = rope_fma(a, c[j], -(b * s[j]));
      x[N + j] = rope_fma(a, s[j], b * c[j]);
    }
  }
}

// 1 / sqrt(mean x^2 + eps) of the row that LPR lanes hold.
template <int N, int LPR, typename F>
__device__ __forceinline__ F rope_rms(const F (&x)[2 * N], float eps) {
#pragma clang fp contract(off)
  F ss = x[0] * x[0];
#pragma unroll
  for (int e = 1; e < 2 * N; ++e) ss = rope_fma(x[e], x[e], ss);
  ss = rope_fma(row_sum<LPR>(ss), F(1.0 / (2 * N * LPR)), F(eps));
  if constexpr (sizeof(F) == 8)
    return 1.0 / __builtin_sqrt(ss);
  else
    return __builtin_amdgcn_rsqf(ss);
}
// x times that and the weight.
template <int N, typename F>
__device__ __forceinline__ void rope_scale(F (&x)[2 * N], F r, const float (&w)[2 * N]) {
#pragma clang fp contract(off)
#pragma unroll
  for (int e = 0; e < 2 * N; ++e) x[e] = x[e] * (r * F(w[e]));
}

}  // namespace tt
