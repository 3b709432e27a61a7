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
  __device__ static __forceinline__ void get(const uint4& v, float* f) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  }
  __device__ static __forceinline__ uint4 put(const float* f) {
    return uint4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
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

// The angle p f in 64 bits less the nearest multiple of pi / 2, and that multiple's
// number, of which the last two bits count (Cody and Waite's reduction: pi / 2 in two
// parts, each taken off by one fused multiply and add, so what is left is as exact
// as p f itself).  Adding 1.5 2^52 rounds to a whole number and leaves it in the last bits.
__device__ __forceinline__ double rope_reduce(double angle, uint32_t* quadrant) {
#pragma clang fp contract(off)
  constexpr double kTwoOverPi = 0.63661977236758134308, kHi = 1.57079632679489661923, kLo = 6.12323399573676603587e-17;
  constexpr double kRound = 6755399441055744.0;
  const double at = __builtin_fma(angle, kTwoOverPi, kRound), k = at - kRound;
  *quadrant = (uint32_t)__double_as_longlong(at);
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
// x with its sign changed where the first bit of `by` is set.
__device__ __forceinline__ float rope_flip(float x, uint32_t by) {
  return __uint_as_float(__float_as_uint(x) ^ (by & 0x80000000u));
}
__device__ __forceinline__ double rope_flip(double x, uint32_t by) {
  return __longlong_as_double(__double_as_longlong(x) ^ (long long)((uint64_t)(by & 0x80000000u) << 32));
}
// cos and sin of position pos times the N frequencies from `freq` on.  The angle
// is formed and reduced in 64 bits: at position 131072 the product alone, rounded
// to 32, would be 0.004 off.
template <int N, typename F>
__device__ __forceinline__ void rope_angles(const float* freq, int64_t pos, F (&c)[N], F (&s)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    uint32_t quadrant;
    const F r = (F)rope_reduce((double)pos * (double)freq[i], &quadrant);
    F x, y;
    rope_series(r, &x, &y);
    const F cc = (quadrant & 1u) ? x : y, ss = (quadrant & 1u) ? y : x;
    c[i] = rope_flip(cc, (quadrant + 1u) << 30);  // negative in quadrants 1 and 2, 2 and 3
    s[i] = rope_flip(ss, quadrant << 30);
  }
}
// The position of token t of sequence b.
__device__ __forceinline__ int64_t rope_position(const Rope& rp, int64_t b, int64_t t, int64_t T) {
  if (rp.positions) return rp.positions[b * T + t];
  return (rp.lengths ? (int64_t)rp.lengths[b] - T : 0) + t;
}

__device__ __forceinline__ float rope_fma(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double rope_fma(double a, double b, double c) { return __builtin_fma(a, b, c); }

// x of the lane that a DPP control names.
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(x), CTRL, 0xf, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ double dpp(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)u, CTRL, 0xf, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, true);
  return __longlong_as_double((long long)((uint64_t)lo | ((uint64_t)hi << 32)));
}
// Sum over the LPR neighbouring lanes that hold a row (2 to 16), the same in each:
// with lanes 1 0 3 2 and 2 3 0 1 of a quad, then, its lanes being equal, with
// the mirror images of eight and of 16 lanes.
template <int LPR, typename F>
__device__ __forceinline__ F row_sum(F x) {
  static_assert(LPR >= 2 && LPR <= 16, "lanes of a row");
  x += dpp<0xB1>(x);
  if constexpr (LPR >= 4) x += dpp<0x4E>(x);
  if constexpr (LPR >= 8) x += dpp<0x141>(x);
  if constexpr (LPR >= 16) x += dpp<0x140>(x);
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

// A lane's rotation with the weights of its norm in it: pair (a, b) of a row times r
// becomes (a ca - b cb, a sa + b sb) of that, ca = w_a cos, cb = w_b sin, sa = w_a
// sin, sb = w_b cos; lanes that turn nothing keep their weights in ca and sb.
template <int N>
struct RopeTurn {
  float ca[N], cb[N], sa[N], sb[N];
  // w: the weights in the order of the lane's values.
  __device__ __forceinline__ void set(const float (&c)[N], const float (&s)[N], const float (&w)[2 * N], bool turns,
                                      bool inter) {
#pragma clang fp contract(off)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float wa = inter ? w[2 * j] : w[j], wb = inter ? w[2 * j + 1] : w[N + j];
      ca[j] = turns ? wa * c[j] : wa;
      sb[j] = turns ? wb * c[j] : wb;
      cb[j] = wb * s[j];
      sa[j] = wa * s[j];
    }
  }
  __device__ __forceinline__ void operator()(float (&x)[2 * N], float r, bool turns, bool inter) const {
#pragma clang fp contract(off)
    if (inter) {
      pairs<true>(x, r, turns);
    } else {
      pairs<false>(x, r, turns);
    }
  }
  template <bool INTER>
  __device__ __forceinline__ void pairs(float (&x)[2 * N], float r, bool turns) const {
#pragma clang fp contract(off)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      constexpr int A = INTER ? 2 : 1, B = INTER ? 1 : N;
      const float a = x[A * j] * r, b = x[A * j + B] * r;
      if (turns) {
        x[A * j] = rope_fma(a, ca[j], -(b * cb[j]));
        x[A * j + B] = rope_fma(a, sa[j], b * sb[j]);
      } else {
        x[A * j] = a * ca[j];
        x[A * j + B] = b * sb[j];
      }
    }
  }
};

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
