// Device-side building blocks that the decodes over quantised and over paged caches
// share: T newest tokens of a K / V head's query heads as a tile of 16 rows on the
// matrix unit, their bf16 terms, and the merge of splits.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "attn_common.h"

namespace tt {
namespace {

constexpr int kMdThreads = 256, kMdWaves = kMdThreads / 64;
constexpr int kMdRows = 16;  // query rows of a workgroup
constexpr int kMdKeys = 32;  // keys of a wave's step

__device__ __forceinline__ f32x4 mfma_bf16_16x16x32(const bf16x8& a, const bf16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// max and sum over lanes l, l ^ 16, l ^ 32, l ^ 48, in every one of them
__device__ __forceinline__ float max_rows(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return max_xor32(vmax(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float sum_rows(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return sum_xor32(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// x as a sum of N bf16 terms: each what the earlier ones leave, cut off, the last
// one rounded; three hold any fp32 value of 2^-110 and more exactly.  Of two (the
// 4-bit cache's weights) the first is rounded too: it leaves at most 2^-8 of the
// value, of which the second is 2^-17 off at most (cut off, it would leave 2^-7,
// and 2^-16 in the end).  ANY: x may be
// infinite or NaN, or meet infinities.  A term is then the largest bf16 below the
// value, so that none but zero's own are zero (1 is 255 / 2^8 + 255 / 2^16 + 1 /
// 2^16): times an infinity each has x's sign, where 0 inf would be NaN; an
// infinite x ends in an infinite term, NaN in NaN.
template <int N, bool ANY = false>
__device__ __forceinline__ void md_terms(const float (&x)[8], bf16x8 (&t)[N]) {
  float left[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) left[e] = x[e];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (N == 2 && n == 0) {
        w[i] = pack_bf16x2(left[2 * i], left[2 * i + 1]);
        left[2 * i] -= __uint_as_float(w[i] << 16);
        left[2 * i + 1] -= __uint_as_float(w[i] & 0xffff0000u);
      } else if (n + 1 < N) {
        uint32_t lo = __float_as_uint(left[2 * i]), hi = __float_as_uint(left[2 * i + 1]);
        if (ANY) lo -= left[2 * i] != 0.f, hi -= left[2 * i + 1] != 0.f;
        w[i] = __builtin_amdgcn_perm(hi, lo, 0x07060302u);  // the upper halves
        left[2 * i] -= __uint_as_float(lo & 0xffff0000u);
        left[2 * i + 1] -= __uint_as_float(hi & 0xffff0000u);
      } else {
        w[i] = pack_bf16x2(left[2 * i], left[2 * i + 1]);
      }
    }
    t[n] = __builtin_bit_cast(bf16x8, w);
  }
}

__device__ __forceinline__ void md_load8(const u16* p, float (&f)[8]) {
  u16 x[8];
  __builtin_memcpy(x, p, 16);
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = bf16_to_f32(x[e]);
}
__device__ __forceinline__ void md_load8(const float* p, float (&f)[8]) { __builtin_memcpy(f, p, 32); }
__device__ __forceinline__ void md_put(u16* p, float v) { *p = f32_to_bf16(v); }
__device__ __forceinline__ void md_put(float* p, float v) { *p = v; }

// o and lse of a row from its sums (den = 0: no key, or only scores of -inf).
template <typename T>
__device__ __forceinline__ float md_quotient(float num, float den) {
  return den == 0.f ? 0.f : num / den;
}
__device__ __forceinline__ float md_lse(float m, float den) {
  return den == 0.f ? -INFINITY : (m + __log2f(den)) * kLn2;
}

// Merges the splits of a row: 256 threads, D / 4 to a partial and 1024 / D
// partials side by side, which meet in LDS.
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_decode_merge_kernel(const float* __restrict__ part_o,
                                                                const float2* __restrict__ part_ml,
                                                                T* __restrict__ o, float* __restrict__ lse,
                                                                int nsplit) {
  constexpr int TPR = D / 4, G = 256 / TPR;
  __shared__ __align__(16) float s_acc[G][D];
  __shared__ float s_w[G];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, c = tid % TPR, g = tid / TPR;
  const float2* pl = part_ml + row * nsplit;
  const float* po = part_o + row * nsplit * D + 4 * c;
  float mx = -INFINITY;  // every wave forms the maximum by itself
  for (int s = tid & 63; s < nsplit; s += 64) mx = vmax(mx, pl[s].x);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) mx = vmax(mx, __shfl_xor(mx, off, 64));
  const float mb = mx == -INFINITY ? 0.f : mx;
  float sw = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = g; s < nsplit; s += G) {
    const float2 ml = pl[s];
    const float wgt = fast_exp2(ml.x - mb);
    sw += wgt * ml.y;
    acc += wgt * *reinterpret_cast<const f32x4*>(po + (int64_t)s * D);
  }
  *reinterpret_cast<f32x4*>(&s_acc[g][4 * c]) = acc;
  if (c == 0) s_w[g] = sw;
  __syncthreads();
  if (tid >= D) return;
  float num = 0.f, den = 0.f;
#pragma unroll
  for (int i = 0; i < G; ++i) {
    num += s_acc[i][tid];
    den += s_w[i];
  }
  md_put(o + row * D + tid, md_quotient<T>(num, den));
  if (tid == 0 && lse) lse[row] = md_lse(mx, den);
}

}  // namespace
}  // namespace tt
