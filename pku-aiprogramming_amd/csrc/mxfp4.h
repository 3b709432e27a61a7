// Device-side building blocks of the microscaled 4-bit kernels.
//
// The format.  A row of n values is ceil(n / 32) blocks of 32, the last one
// padded with zeros.  A block is 16 bytes of codes (element 2 i in the low
// half of byte i; sign, two exponent bits, one fraction bit: 0, 0.5, 1, 1.5,
// 2, 3, 4, 6) and one scale byte: 2^(byte - 127), 255 for a block that holds
// an infinity or a NaN, all of whose values then read as NaN.  The scale is
// 2^(floor(log2 max|x|) - 2), so that the largest element lands in [4, 8),
// where 6 is the last code (the public OCP microscaling rule).  With a power
// of two as scale, x / scale is exact, so the only rounding is the one to the
// element grid (nearest, halves to even) and any two implementations agree
// bit for bit.
//
// gfx950 deals with it natively (checked on the MI355X): v_cvt_scalef32_pk_*
// divide by or multiply with the power of two in a float's exponent field (0
// is 2^-127, 255 gives NaN), and v_mfma_scale_f32_*_f8f6f4 take the codes as
// they are stored, 32 consecutive k of one row per lane, beside that block's
// scale byte.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "attn_common.h"
#include "tt_internal.h"

namespace tt {

constexpr int kMxBlock = 32;       // values under one scale
constexpr int kMxBlockBytes = 16;  // their codes
inline int64_t mx_blocks(int64_t n) { return n / kMxBlock + (n % kMxBlock != 0); }

// The shape of a call on a K / V cache held in the format.
inline int check_cache_mxfp4(const char* fn, int dtype, int64_t B, int64_t Hkv, int64_t T, int64_t cap, int64_t d) {
  const std::string f(fn);
  if (dtype != TT_F32 && dtype != TT_BF16) return fail(TT_ERR_ARG, f + ": dtype must be TT_F32 or TT_BF16");
  if (B < 0 || Hkv < 0 || T < 0 || cap < 0) return fail(TT_ERR_ARG, f + ": negative dimension");
  if (d != 32 && d != 64 && d != 128)
    return fail(TT_ERR_UNSUPPORTED, f + ": head dim must be 32, 64 or 128 (got " + std::to_string(d) + ")");
  if (T > (int64_t(1) << 30) || cap > (int64_t(1) << 30)) return fail(TT_ERR_ARG, f + ": sequence too long");
  if (B > (int64_t(1) << 24) || Hkv > (int64_t(1) << 24) || B * Hkv > (int64_t(1) << 24))
    return fail(TT_ERR_ARG, f + ": too many heads");
  return TT_OK;
}

// The float whose exponent field is the scale byte, as the conversions take it.
__device__ __forceinline__ float mx_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// The scale byte of a block from the largest exponent field among its values.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t e) { return e == 255u ? 255u : (e > 2u ? e - 2u : 0u); }

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// 16 bytes at any element alignment, non-temporally or not.
typedef uint32_t mx_word __attribute__((ext_vector_type(4), aligned(2)));
template <bool NT, typename T>
__device__ __forceinline__ void mx_load16(void* to, const T* p) {
  const mx_word* q = reinterpret_cast<const mx_word*>(p);
  const mx_word x = NT ? __builtin_nontemporal_load(q) : *q;
  __builtin_memcpy(to, &x, 16);
}
template <bool NT, typename T>
__device__ __forceinline__ void mx_store16(T* p, const void* from) {
  mx_word x;
  __builtin_memcpy(&x, from, 16);
  if constexpr (NT)
    __builtin_nontemporal_store(x, reinterpret_cast<mx_word*>(p));
  else
    *reinterpret_cast<mx_word*>(p) = x;
}

// Eight consecutive values in registers.
template <typename T> struct MxEight;
template <> struct MxEight<u16> {
  uint32_t w[4];
  template <bool NT = false>
  __device__ __forceinline__ void load(const u16* p) { mx_load16<NT>(w, p); }
  __device__ __forceinline__ void load_part(const u16* p, int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = 2 * i < n ? p[2 * i] : 0u, hi = 2 * i + 1 < n ? p[2 * i + 1] : 0u;
      w[i] = lo | (hi << 16);
    }
  }
  // the first n of them and zeros
  __device__ __forceinline__ void keep(int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = 2 * i + 1 < n ? w[i] : (2 * i < n ? w[i] & 0xffffu : 0u);
  }
  // the largest exponent field
  __device__ __forceinline__ uint32_t top() const {
    u16x2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7f807f80u));
    return (uint32_t)(m.x > m.y ? m.x : m.y) >> 7;
  }
  __device__ __forceinline__ uint32_t codes(float scale) const {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, w[0]), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, w[1]), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, w[2]), scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, w[3]), scale, 3);
    return c;
  }
  // the values that eight codes stand for
  __device__ __forceinline__ void from(uint32_t c, float scale) {
    w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0));
    w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1));
    w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2));
    w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3));
  }
  template <bool NT = false>
  __device__ __forceinline__ void store(u16* p) const { mx_store16<NT>(p, w); }
  __device__ __forceinline__ void store_part(u16* p, int n) const {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (u16)(w[i / 2] >> (16 * (i & 1)));
  }
};
template <> struct MxEight<float> {
  float v[8];
  template <bool NT = false>
  __device__ __forceinline__ void load(const float* p) {
    mx_load16<NT>(v, p);
    mx_load16<NT>(v + 4, p + 4);
  }
  __device__ __forceinline__ void load_part(const float* p, int n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.f;
  }
  __device__ __forceinline__ uint32_t top() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m >> 23;
  }
  __device__ __forceinline__ uint32_t codes(float scale) const {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], scale, 3);
    return c;
  }
};

// 16 bytes of values, as a lane of a kernel over whole rows holds them: eight
// bf16, or four fp32 (with 32 bytes a lane every access would leave out half of
// each line, which non-temporal stores pay for: 8192 x 4000 read back in 50 us).
template <typename T> struct MxWord;
template <> struct MxWord<u16> : MxEight<u16> {
  typedef uint32_t Codes;
  static constexpr int N = 8;
};
template <> struct MxWord<float> {
  typedef uint16_t Codes;
  static constexpr int N = 4;
  float v[4];
  template <bool NT = false>
  __device__ __forceinline__ void load(const float* p) { mx_load16<NT>(v, p); }
  __device__ __forceinline__ void load_part(const float* p, int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? p[i] : 0.f;
  }
  __device__ __forceinline__ void keep(int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? v[i] : 0.f;
  }
  __device__ __forceinline__ uint32_t top() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m >> 23;
  }
  __device__ __forceinline__ uint32_t codes(float scale) const {
    const uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], scale, 0);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], scale, 1);
  }
  __device__ __forceinline__ void from(uint32_t c, float scale) {
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 0);
    const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 1);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  }
  template <bool NT = false>
  __device__ __forceinline__ void store(float* p) const { mx_store16<NT>(p, v); }
  __device__ __forceinline__ void store_part(float* p, int n) const {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) p[i] = v[i];
  }
};

// The largest of x over the four lanes of a quad (all four must be active).
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xf, 0xf, true));  // lanes 1 0 3 2
  return max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xf, 0xf, true));  // lanes 2 3 0 1
}

// The block that neighbouring lanes hold a word each of (four or eight of them,
// all active): its scale byte, and the codes of this lane's word.
template <typename T>
__device__ __forceinline__ typename MxWord<T>::Codes mx_quantize_word(const MxWord<T>& x, uint32_t* scale_byte) {
  uint32_t e = quad_max(x.top());
  if constexpr (MxWord<T>::N == 4)  // the other quad of the eight lanes, by their mirror image
    e = max(e, (uint32_t)__builtin_amdgcn_mov_dpp((int)e, 0x141, 0xf, 0xf, true));
  const uint32_t s = mx_scale_byte(e);
  *scale_byte = s;
  return (typename MxWord<T>::Codes)(s == 255u ? 0u : x.codes(mx_scale(s)));
}

}  // namespace tt
