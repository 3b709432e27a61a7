// A K / V cache in pages, and its 8-bit values.
//
// Pools [pages][Hkv][page][D] for K and for V; key j of sequence b is row j % page
// of page table[b][j / page].  A page that the pool does not have (a negative
// number, or one past its end) holds no keys: nothing is stored there, and its
// keys are not seen.
//
// An 8-bit pool holds e4m3 codes (sign, four exponent bits, three fraction bits: up
// to 448, steps of 2^-9 at least, 0x7f and 0xff NaN) under one scale byte, 2^(byte
// - 127), for each page and head: the smallest power of two that takes the largest
// value to at most 448, of 2^-124 (so that every value held is a bf16 number) to
// 2^119.  Being a power of two it changes no digit, so a page that gains larger
// values is scaled again without loss but in its smallest values.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "attn_common.h"
#include "tt_internal.h"

namespace tt {

// A cache's geometry, as the kernels take it.
struct Pages {
  const int* table;    // [B][width]
  const int* lengths;  // [B]
  int64_t pages;       // in the pool
  int64_t width;       // places of a sequence in the table
  uint32_t hkv;
  int lp;  // log2(page)
};

// The length of sequence b as far as its table reaches.
__device__ __forceinline__ int64_t paged_end(const Pages& pg, int64_t length) {
  return min(max(length, (int64_t)0), pg.width << pg.lp);
}

constexpr uint32_t kE4MinByte = 3, kE4MaxByte = 246;
// The scale byte for values whose largest magnitude has these bits (finite).
__device__ __forceinline__ uint32_t e4_scale_byte(uint32_t top) {
  const int byte = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)min(max(byte, (int)kE4MinByte), (int)kE4MaxByte);
}
__device__ __forceinline__ float e4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }
__device__ __forceinline__ float e4_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
// x as it goes into a code: infinities become NaN, values past 448 become 448.
__device__ __forceinline__ float e4_clamp(float x) {
  const float y = __builtin_amdgcn_fmed3f(x, -448.f, 448.f);
  return __builtin_isfpclass(x, 0x207) ? __uint_as_float(0x7fc00000u) : y;  // an infinity or NaN, of one v_cmp_class
}
// Four codes of values times `inverse`, nearest, halves to even.  CLAMP false: none is past
// 448 but infinities, which the conversion makes NaN.
template <bool CLAMP = true>
__device__ __forceinline__ uint32_t e4_codes(const float* x, float inverse) {
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = CLAMP ? e4_clamp(x[i] * inverse) : x[i] * inverse;
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], c, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], c, true);
}
// The values of four codes, not scaled.
__device__ __forceinline__ void e4_values(uint32_t c, float* x) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(c, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}

// What append, gather and attention have in common: the geometry and the types.
inline int check_paged(const char* fn, int dtype, int cache, int64_t B, int64_t Hkv, int64_t T, int64_t d,
                       int64_t npages, int64_t page, int64_t width, int* lp) {
  const std::string f(fn);
  if (dtype != TT_F32 && dtype != TT_BF16) return fail(TT_ERR_ARG, f + ": dtype must be TT_F32 or TT_BF16");
  if (cache != dtype && cache != TT_E4M3)
    return fail(TT_ERR_ARG, f + ": the cache must hold values of dtype, or TT_E4M3");
  if (B < 0 || Hkv < 0 || T < 0 || npages < 0 || width < 0) return fail(TT_ERR_ARG, f + ": negative dimension");
  if (d != 32 && d != 64 && d != 128)
    return fail(TT_ERR_UNSUPPORTED, f + ": head dim must be 32, 64 or 128 (got " + std::to_string(d) + ")");
  *lp = page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : page == 128 ? 7 : 0;
  if (*lp == 0)
    return fail(TT_ERR_UNSUPPORTED, f + ": pages hold 16, 32, 64 or 128 tokens (got " + std::to_string(page) + ")");
  if (T > (int64_t(1) << 30) || width > (int64_t(1) << 30) / page) return fail(TT_ERR_ARG, f + ": sequence too long");
  if (B > (int64_t(1) << 24) || Hkv > (int64_t(1) << 24) || B * Hkv > (int64_t(1) << 24))
    return fail(TT_ERR_ARG, f + ": too many heads");
  if (npages > 0x7fffffff || (Hkv > 0 && npages > (int64_t(1) << 52) / (Hkv * page * d)))
    return fail(TT_ERR_ARG, f + ": too many pages");
  return TT_OK;
}

// The pools, table and lengths of a call that reads or writes them.
inline int check_pools(const char* fn, int cache, const void* k_pages, const void* v_pages, const uint8_t* k_scales,
                       const uint8_t* v_scales, const int* table, const int* lengths) {
  const std::string f(fn);
  if (!k_pages || !v_pages || !table || !lengths) return fail(TT_ERR_ARG, f + ": null pointer");
  if (((uintptr_t)k_pages | (uintptr_t)v_pages) & 15) return fail(TT_ERR_ARG, f + ": pages must be 16-byte aligned");
  if (cache == TT_E4M3 && (!k_scales || !v_scales))
    return fail(TT_ERR_ARG, f + ": an 8-bit cache needs its scales");
  return TT_OK;
}

inline size_t cache_item(int cache) { return cache == TT_E4M3 ? 1 : cache == TT_BF16 ? 2 : 4; }

}  // namespace tt
