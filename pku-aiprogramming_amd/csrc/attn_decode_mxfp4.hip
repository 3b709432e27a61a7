// Attention of the newest tokens over a K / V cache held in the microscaled
// 4-bit format (mxfp4.h): o = softmax(s q K^T) V for T tokens of H query heads
// over Hkv cached heads.
//
// The bytes of the cache bound it (17/32 a value, K and V each read once), and
// with few bytes a value the arithmetic must stay small beside them, so both
// products run on the matrix unit for every group size: the R = H / Hkv * T
// query rows that share one K / V head are a tile of 16 columns (rows past R
// are zeros: the unit has the time, a memory access has not).  A wave owns 32
// keys at a time with a running maximum and sum of its own:
//   S^T [32 keys x 16 rows] = K Q^T: a lane's piece of a K row (D / 8 bytes of
//     codes, one scale) becomes the bf16 operand by v_cvt_scalef32_pk_bf16_fp4,
//     exactly, with no LDS: the k order of the contraction is free, and q is
//     laid out to match.  Result: a lane owns one query row and 8 keys.
//   O^T [D x 16 rows] += V^T P^T: P comes out of S^T in the operand's layout
//     (the order of the keys is free as well); V's rows are converted to bf16
//     into the wave's LDS tile and read back transposed (ds_read_b64_tr_b16).  P
//     is split into bf16 terms (two for bf16 tensors, 2^-17 off; three for fp32,
//     whose q is split into three exact terms too), so that no rounding of the
//     weights shows in the result.
// The codes of the next step are in flight meanwhile.  The waves of a workgroup
// meet in LDS at the end, and splits of the keys over workgroups in a second
// launch.  Measured: 64 x 32 heads x 8192 keys of 128, bf16, 356 us (6.4 TB/s),
// fp32 402; 16 x 8 heads x 16383 keys 51.5 us (5.5 TB/s); 1 x 32 heads x 4097 keys
// 11.0 us, of which the second launch 2 to 3.  A long prompt's tokens are right, but
// not what this is made for: every 16 rows convert all keys again, and 512 tokens
// of 32 / 8 heads over 8192 keys take 151 us.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <limits>
#include <optional>
#include <string>

#include "attn_tiles.h"
#include "mxfp4.h"
#include "tt_internal.h"

namespace tt {
namespace {

constexpr int kMdThreads = 256, kMdWaves = kMdThreads / 64;
constexpr int kMdRows = 16;  // query rows of a workgroup
constexpr int kMdKeys = 32;  // keys of a wave's step
// From this scale byte on a block may hold infinities (6 2^126 is 2^128 or more) or NaN.
constexpr uint32_t kMdNotFinite = 253;

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

// A lane's piece of a K or V row: W dwords of codes (8 values each) under one scale.
template <int W>
struct MdPiece {
  uint32_t c[W], s;
};
// codes and scales: the first row of a step, alike in all lanes; row: this lane's
// from there.  STREAM: codes that no other workgroup reads are loaded
// non-temporally (64 x 32 heads x 8192 keys 391 -> 359 us); those that a second
// tile of query rows reads too are better kept (2 x 8 x 16383 keys, 20 tokens: 18.5
// against 19.3).
template <bool STREAM, int W>
__device__ __forceinline__ void md_load(MdPiece<W>& p, const uint8_t* codes, const uint8_t* scales, uint32_t row,
                                        int g) {
  typedef uint32_t vec __attribute__((ext_vector_type(W)));
  const vec* from = reinterpret_cast<const vec*>(codes + (row * (16u * W) + (uint32_t)g * (4u * W)));
  const vec x = STREAM ? __builtin_nontemporal_load(from) : *from;
  __builtin_memcpy(p.c, &x, 4 * W);
  p.s = scales[W == 4 ? row * 4u + (uint32_t)g : (W == 2 ? row * 2u + (uint32_t)(g >> 1) : row)];
}
__device__ __forceinline__ bf16x8 md_bf16(uint32_t codes, float scale) {
  MxEight<u16> v;
  v.from(codes, scale);
  return __builtin_bit_cast(bf16x8, v.w);
}

// The wave's V tile: [32 keys][D] bf16 in 16-byte chunks, chunk c of row r at
// chunk c ^ exchange(r), where a row's chunks number D / 8 and 256 / 2 D rows make
// a line of all banks.  A row write puts one chunk of 16 consecutive rows, a
// transposed read takes two neighbouring chunks of eight; both spread over the
// banks.  The chunk enters an address by exclusive or alone, so that one register
// serves all of them.
template <int D>
__device__ __forceinline__ constexpr int md_exchange(int r) {
  return (r & 15) >> (D == 128 ? 0 : (D == 64 ? 1 : 2));
}

// x as a sum of N bf16 terms: each what the earlier ones leave, cut off, the last
// one rounded; three hold any fp32 value exactly.  Of two the first is rounded
// too: it leaves at most 2^-8 of the value, of which the second is 2^-17 off at
// most (cut off, it would leave 2^-7, and 2^-16 in the end).  ANY: x may be
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

__device__ __forceinline__ void lds_st(uint32_t a, const bf16x8& x) {
  *(__attribute__((address_space(3))) bf16x8*)(uintptr_t)a = x;
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

// The maximum is that of the products, the scale sl2 (of log2 e too, above zero:
// its sign goes into q, and zero is the smallest fp32, 2^-149, which still hides
// what is masked and takes no product to more than 2^-21) enters the exponent,
// 2^(sl2 s - sl2 m), one operation a score.
// Workgroup id = (head * tiles + tile) * nsplit + split, head = b Hkv + hkv,
// tile = 16 of the head's R query rows.  Each sequence's own length is cut into
// nsplit spans, so that sequences of any length keep every workgroup busy.
// Eight workgroups a CU of d = 32 bf16 keep its vector work busy: 64 x 32 heads x
// 8192 keys 143 us, with seven 147; the others' registers are let be.
template <typename T, int D, bool STREAM>
__global__ __launch_bounds__(kMdThreads, sizeof(T) == 2 && D == 32 ? 8 : 3) void attn_decode_mxfp4_kernel(
    const T* __restrict__ q, const uint8_t* __restrict__ kc, const uint8_t* __restrict__ ks,
    const uint8_t* __restrict__ vc, const uint8_t* __restrict__ vs, const int* __restrict__ lengths,
    float* __restrict__ part_o, float2* __restrict__ part_ml, T* __restrict__ o, float* __restrict__ lse,
    uint32_t Hkv, uint32_t R, uint32_t tokens, uint32_t tiles, int cap, uint32_t nsplit, float sl2, bool negative) {
  constexpr int W = D / 32;                                  // dwords of a lane's piece, and k steps of a key tile
  constexpr int NQ = sizeof(T) == 4 ? 3 : 1, NP = sizeof(T) == 4 ? 3 : 2;  // terms of q and of the weights
  constexpr int ND = D / 16;                                 // 16-row tiles of O^T
  __shared__ __align__(256) u16 s_v[kMdWaves][kMdKeys * D];
  __shared__ float s_m[kMdWaves][kMdRows], s_l[kMdWaves][kMdRows];
  static_assert(sizeof(s_v[0]) == kMdRows * D * sizeof(float), "the waves' sums reuse their tiles");

  const int l = threadIdx.x & 63, r = l & 15, g = l >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t unit = blockIdx.x / nsplit, split = blockIdx.x - unit * nsplit;
  const uint32_t head = unit / tiles, row0 = (unit - head * tiles) * kMdRows;
  const int64_t qrow = (int64_t)head * R + row0;  // the tile's first row of q and o
  const int nrows = (int)min((uint32_t)kMdRows, R - row0);

  float qx[W][8];
#pragma unroll
  for (int j = 0; j < W; ++j) {
#pragma unroll
    for (int e = 0; e < 8; ++e) qx[j][e] = 0.f;
    if (r < nrows) md_load8(q + (qrow + r) * D + g * (8 * W) + 8 * j, qx[j]);
  }

  // Keys that the newest token sees, and that this lane's row sees.
  const int full = lengths[head / Hkv];
  const int len = min(full, cap), before = (int)tokens - 1;
  const int t = r < nrows ? (int)((row0 + (uint32_t)r) % tokens) : 0;
  const int seen = r < nrows ? (int)min((int64_t)len, (int64_t)full - (before - t)) : 0;
  const int all_see = (int)min((int64_t)len, (int64_t)full - before);  // keys that every row sees
  int kbeg = 0, kend = 0;
  if (len > 0) {
    const uint32_t span = (((uint32_t)len + nsplit - 1) / nsplit + kMdKeys - 1) / kMdKeys * kMdKeys;
    kbeg = (int)min((uint64_t)split * span, (uint64_t)len);
    kend = (int)min((uint32_t)kbeg + span, (uint32_t)len);
  }

  f32x4 acc[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, lsum = 0.f;
  u16* tile = s_v[w];
  constexpr uint32_t kRow = 2 * D;  // bytes of a tile row
  // chunk g W of row r, and columns 4 (r % 4) of row 4 g + r / 4
  const uint32_t put = lds_addr(tile) + (uint32_t)r * kRow + 16u * (uint32_t)((g * W) ^ md_exchange<D>(r));
  const int krow = 4 * g + (r >> 2);
  const uint32_t get = lds_addr(tile) + (uint32_t)krow * kRow + 16u * (uint32_t)(((r & 3) >> 1) ^ md_exchange<D>(krow)) +
                       8u * (uint32_t)(r & 1);
  const int64_t base = (int64_t)head * cap;

  MdPiece<W> k[2], v[2];  // the next step's keys, as loaded
  auto fetch = [&](int j0) {
    const int64_t at = base + j0;  // the same for the wave: the address of a piece is this and a lane's offset
    const uint8_t *kp = kc + at * (16 * W), *vp = vc + at * (16 * W), *ksp = ks + at * W, *vsp = vs + at * W;
    const bool whole = j0 + kMdKeys <= len;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t row = 16u * u + (uint32_t)r;
      if (!whole) row = (uint32_t)min((int)row, len - 1 - j0);  // keys past the end: the last one, masked below
      md_load<STREAM>(k[u], kp, ksp, row, g);
      md_load<STREAM>(v[u], vp, vsp, row, g);
    }
  };
  int j0 = kbeg + w * kMdKeys;
  if (j0 < kend) fetch(j0);
  bf16x8 qf[W][NQ];
#pragma unroll
  for (int j = 0; j < W; ++j) {
    if (negative)
#pragma unroll
      for (int e = 0; e < 8; ++e) qx[j][e] = -qx[j][e];
    md_terms<NQ, true>(qx[j], qf[j]);
  }
  // s[u][i]: key 16 u + 4 g + i of the step, for this lane's row
  auto scores = [&](const MdPiece<W>(&kx)[2], f32x4(&s)[2]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      const float f = mx_scale(kx[u].s);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const bf16x8 a = md_bf16(kx[u].c[j], f);
#pragma unroll
        for (int n = NQ - 1; n >= 0; --n) s[u] = mfma_bf16_16x16x32(a, qf[j][n], s[u]);
      }
    }
  };
  auto mask = [&](f32x4(&s)[2], int j0) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[u][i] = j0 + 16 * u + 4 * g + i < min(seen, kend) ? s[u][i] : -INFINITY;
  };
  // A block of V that is taken out of the product: one that holds infinities, and
  // one of NaN where some row does not see it (the others' every weight makes NaN).
  auto apart = [](const MdPiece<W>& v, bool edge) { return v.s >= kMdNotFinite && (edge || v.s != 255u); };
  bool any_apart = false;
  for (; j0 < kend; j0 += kMdWaves * kMdKeys) {
    MdPiece<W> kx[2] = {k[0], k[1]}, vx[2] = {v[0], v[1]};
    if (j0 + kMdWaves * kMdKeys < kend) fetch(j0 + kMdWaves * kMdKeys);

    f32x4 s[2];
    scores(kx, s);
    // A weight of zero must not meet an infinity or a NaN, be it a masked key's or
    // a bf16 term of a weight: V rows that no row sees become zeros, and so do
    // blocks that may hold either, whose values are added after the loop.
    const bool edge = j0 + kMdKeys > min(kend, all_see);
    if (edge || wave_any(max(vx[0].s, vx[1].s) >= kMdNotFinite)) {
      mask(s, j0);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const bool out = j0 + 16 * u + r >= kend, odd = apart(vx[u], edge);
        any_apart |= wave_any(!out && odd);
        if (out || odd) {
          vx[u].s = 127u;
#pragma unroll
          for (int j = 0; j < W; ++j) vx[u].c[j] = 0u;
        }
      }
    }

    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = vmax(top, s[u][i]);
    top = max_rows(top);
    const float mn = vmax(m, top);
    const float mb = mn == -INFINITY ? 0.f : sl2 * mn;  // nothing seen yet: every weight 0
    if (wave_any(mn != m)) {
      // From the products as they were rounded (no fused multiply and add), so
      // exactly 1 for a row that keeps its maximum, whatever is beside it.
#pragma clang fp contract(off)
      const float a = m == -INFINITY ? 0.f : fast_exp2(sl2 * m - mb);
      lsum *= a;
#pragma unroll
      for (int i = 0; i < ND; ++i) acc[i] *= a;
      m = mn;
    }
    float p[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      p[e] = fast_exp2(__builtin_fmaf(sl2, s[e >> 2][e & 3], -mb));
      lsum += p[e];
    }
    bf16x8 pf[NP];
    md_terms<NP>(p, pf);

    // V rows to the wave's tile, 8 values a 16-byte chunk
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float f = mx_scale(vx[u].s);
#pragma unroll
      for (int j = 0; j < W; ++j)
        lds_st((put ^ (16u * j)) + u * 16 * kRow, md_bf16(vx[u].c[j], f));
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      const uint32_t at = get ^ (32u * i);
      const bf16x8 a = lds_tr16x2_at(at, at + 16 * kRow);
#pragma unroll
      for (int n = NP - 1; n >= 0; --n) acc[i] = mfma_bf16_16x16x32(a, pf[n], acc[i]);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }

  // Rare: the steps with such blocks once more, for the values of these alone,
  // under the weights that the final maximum gives.
  if (any_apart) {
    const float mb = m == -INFINITY ? 0.f : sl2 * m;
    for (j0 = kbeg + w * kMdKeys; j0 < kend; j0 += kMdWaves * kMdKeys) {
      fetch(j0);
      const bool edge = j0 + kMdKeys > min(kend, all_see);
      if (!wave_any(apart(v[0], edge) || apart(v[1], edge))) continue;
      f32x4 s[2];
      scores(k, s);
      mask(s, j0);
#pragma unroll
      for (int u = 0; u < 2; ++u)
        for (uint64_t left = __ballot(j0 + 16 * u + r < kend && apart(v[u], edge)); left; left &= left - 1) {
          const int at = __builtin_ctzll(left), in = at & 15, part = at >> 4, key = j0 + 16 * u + in;
          float wgt = (in & 2) ? ((in & 1) ? s[u][3] : s[u][2]) : ((in & 1) ? s[u][1] : s[u][0]);
          wgt = __shfl(wgt, 16 * (in >> 2) + r, 64);  // this row's score, from the lane that holds the key's
          wgt = fast_exp2(__builtin_fmaf(sl2, wgt, -mb));
          const uint8_t *codes = vc + (base + key) * (16 * W), *scales = vs + (base + key) * W;
#pragma unroll
          for (int i = 0; i < ND; ++i) {  // this lane's columns 16 i + 4 g and three more, if the piece has them
            if ((16 * i + 4 * g) / (8 * W) != part || key >= seen) continue;
            MxWord<float> x;
            x.from(*reinterpret_cast<const uint16_t*>(codes + 8 * i + 2 * g), mx_scale(scales[i / 2]));
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][e] += wgt * x.v[e];
          }
        }
    }
  }

  // The waves' sums meet in LDS: [row][D] fp32 over each wave's own tile, chunks
  // of four swizzled by the row.
  lsum = sum_rows(lsum);
  float* mine = reinterpret_cast<float*>(tile);
#pragma unroll
  for (int i = 0; i < ND; ++i)
    *reinterpret_cast<f32x4*>(&mine[r * D + 4 * ((4 * i + g) ^ (r & (D / 4 - 1)))]) = acc[i];
  if (g == 0) {
    s_m[w][r] = m == -INFINITY ? m : sl2 * m;
    s_l[w][r] = lsum;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < nrows * (D / 4); c += kMdThreads) {
    const int row = c / (D / 4), d4 = c - row * (D / 4);
    float top = s_m[0][row];
#pragma unroll
    for (int i = 1; i < kMdWaves; ++i) top = vmax(top, s_m[i][row]);
    const float mb = top == -INFINITY ? 0.f : top;
    float den = 0.f;
    f32x4 num = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kMdWaves; ++i) {
      const float wgt = fast_exp2(s_m[i][row] - mb);
      const float* theirs = reinterpret_cast<const float*>(s_v[i]);
      den += wgt * s_l[i][row];
      num += wgt * *reinterpret_cast<const f32x4*>(&theirs[row * D + 4 * (d4 ^ (row & (D / 4 - 1)))]);
    }
    if (nsplit > 1) {
      const int64_t at = (qrow + row) * nsplit + split;
      *reinterpret_cast<f32x4*>(part_o + at * D + 4 * d4) = num;
      if (d4 == 0) part_ml[at] = float2{top, den};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) md_put(o + (qrow + row) * D + 4 * d4 + e, md_quotient<T>(num[e], den));
      if (d4 == 0 && lse) lse[qrow + row] = md_lse(top, den);
    }
  }
}

// Merges the splits of a row: 256 threads, D / 4 to a partial and 1024 / D
// partials side by side, which meet in LDS.
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_decode_mxfp4_merge_kernel(const float* __restrict__ part_o,
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

constexpr size_t kMdWork = size_t(24) << 20;  // the partials' scratch, of one size so that graphs may keep its address

// Into how many splits to cut the keys.  A workgroup costs its keys and about
// kMdFixed more (its queries, the meeting of its waves), a CU's time goes by the
// workgroups that fall to it, up to per_cu of them at once, of which fewer keep
// less of memory's latency covered, and splits cost the second launch, about
// kMdMerge keys.  Measured (d = 128 bf16, 256 CUs, us): 16 x 8 heads x 16383 keys
// in 3 / 4 / 5 / 6 splits (1.5, 2, 2.5, 3 a CU) 58.5 / 51.1 / 57.4 / 52.3, 20 x 8 heads in
// 3 / 4 / 5 63.9 / 72.2 / 75.0, 64 x 32 heads x 8192 keys in 1 / 3 358 / 358.
constexpr int64_t kMdFixed = 150, kMdMerge = 300;
inline int64_t md_splits(int64_t units, int64_t keys, int64_t per_cu, int64_t cus, int64_t d, int64_t most) {
  constexpr int64_t step = kMdWaves * kMdKeys;
  most = std::min(most, (keys + step - 1) / step);
  most = std::min(most, std::max<int64_t>(4, 2 * per_cu * cus / units));
  int64_t best = 1;
  double least = std::numeric_limits<double>::max();
  for (int64_t n = 1; n <= most; n += 1 + n / 64) {  // the host's time counts too
    const int64_t here = (units * n + cus - 1) / cus;
    const int64_t last = here % per_cu, each = ((keys + n - 1) / n + step - 1) / step * step + kMdFixed;
    auto group = [&](int64_t w) { return w > 0 ? (double)w + 76.8 / (double)d : 0.0; };  // w at once
    const double cost = (double)each * ((double)(here / per_cu) * group(per_cu) + group(last)) +
                        (n > 1 ? (double)(kMdMerge + 4 * n) : 0.0);
    if (cost < least) {
      least = cost;
      best = n;
    }
  }
  return best;
}

template <typename T, int D>
int launch(const char* fn, const T* q, const uint8_t* kc, const uint8_t* ks, const uint8_t* vc, const uint8_t* vs,
           const int* lengths, T* o, float* lse, int64_t B, int64_t H, int64_t Hkv, int64_t tokens, int64_t cap,
           float scale, hipStream_t st) {
  const int64_t rows = B * H * tokens, R = H / Hkv * tokens;
  const int64_t tiles = (R + kMdRows - 1) / kMdRows, units = B * Hkv * tiles;
  static const int per_cu = [] {
    int n = 0;
    const hipError_t e = hipOccupancyMaxActiveBlocksPerMultiprocessor(
        &n, (const void*)attn_decode_mxfp4_kernel<T, D, true>, kMdThreads, 0);
    if (e != hipSuccess) (void)hipGetLastError();
    // The rule was measured with three at once at d = 128, where registers let a
    // fourth in; counted, it would take 16 x 8 heads x 16383 keys from 51.5 us to
    // 52.8 and 16 x 32 / 8 heads of ragged lengths from 46.2 to 47.5.
    return e != hipSuccess || n < 1 || (D == 128 && n > 3) ? 3 : n;
  }();
  int64_t nsplit = md_splits(units, std::max<int64_t>(cap, 1), per_cu, device_cu_count(), D,
                             (int64_t)(kMdWork / ((size_t)rows * (D + 2) * sizeof(float))));
  void* ws = nullptr;
  std::optional<WorkspaceLease> lease;  // held until both kernels are queued
  if (nsplit < 2 || !lease.emplace().get_fixed(st, kWsMxfp4Decode, kMdWork, &ws)) nsplit = 1;
  float* part_o = (float*)ws;
  float2* part_ml = (float2*)(part_o + rows * nsplit * D);
  float sl2 = std::fabs(scale * kLog2e);
  uint32_t bits;  // 1: the smallest fp32, formed as the host's arithmetic may flush it
  memcpy(&bits, &sl2, sizeof(bits));
  bits = std::max(bits, 1u);
  memcpy(&sl2, &bits, sizeof(bits));
#define TT_MD_LAUNCH(STREAM)                                                                                          \
  hipLaunchKernelGGL((attn_decode_mxfp4_kernel<T, D, STREAM>), dim3((unsigned)(units * nsplit)), dim3(kMdThreads), 0, \
                     st, q, kc, ks, vc, vs, lengths, part_o, part_ml, o, lse, (uint32_t)Hkv, (uint32_t)R,             \
                     (uint32_t)tokens, (uint32_t)tiles, (int)cap, (uint32_t)nsplit, sl2, scale < 0.f)
  if (tiles == 1)
    TT_MD_LAUNCH(true);
  else
    TT_MD_LAUNCH(false);
#undef TT_MD_LAUNCH
  TT_LAUNCHED(fn, st);
  if (nsplit > 1) {
    hipLaunchKernelGGL((attn_decode_mxfp4_merge_kernel<T, D>), dim3((unsigned)rows), dim3(256), 0, st, part_o, part_ml,
                       o, lse, (int)nsplit);
    TT_LAUNCHED(fn, st);
  }
  return ok();
}

template <typename T>
int launch_d(const char* fn, const void* q, const uint8_t* kc, const uint8_t* ks, const uint8_t* vc, const uint8_t* vs,
             const int* lengths, void* o, float* lse, int64_t B, int64_t H, int64_t Hkv, int64_t tokens, int64_t cap,
             int64_t d, float scale, hipStream_t st) {
#define TT_MD(D) \
  return launch<T, D>(fn, (const T*)q, kc, ks, vc, vs, lengths, (T*)o, lse, B, H, Hkv, tokens, cap, scale, st)
  switch (d) {
    case 32: TT_MD(32);
    case 64: TT_MD(64);
    default: TT_MD(128);
  }
#undef TT_MD
}

}  // namespace
}  // namespace tt

using namespace tt;

extern "C" int tt_attn_decode_mxfp4(int dtype, const void* q, const uint8_t* k_codes, const uint8_t* k_scales,
                                    const uint8_t* v_codes, const uint8_t* v_scales, const int* lengths, void* o,
                                    float* lse, int64_t B, int64_t H, int64_t Hkv, int64_t T, int64_t cap, int64_t d,
                                    float scale, void* stream) {
  const char* fn = "tt_attn_decode_mxfp4";
  int rc = check_cache_mxfp4(fn, dtype, B, Hkv, T, cap, d);
  if (rc) return rc;
  if (H < 0 || (Hkv == 0 ? H != 0 : H % Hkv != 0))
    return fail(TT_ERR_ARG, std::string(fn) + ": H must be a multiple of Hkv");
  if (B == 0 || H == 0 || T == 0) return ok();
  if (H > (int64_t(1) << 24) || B * H > (int64_t(1) << 24)) return fail(TT_ERR_ARG, std::string(fn) + ": too many heads");
  if (B * H * T > 0x7fffffff) return fail(TT_ERR_ARG, std::string(fn) + ": too many rows");
  // Splits, and the merge's workgroups of a row each, are few: the scratch holds all of their rows.
  if (!grid_fits(B * Hkv * ((H / Hkv * T + kMdRows - 1) / kMdRows), kMdThreads))
    return fail(TT_ERR_ARG, std::string(fn) + ": grid too large");
  if (!q || !o || !lengths || (cap > 0 && (!k_codes || !k_scales || !v_codes || !v_scales)))
    return fail(TT_ERR_ARG, std::string(fn) + ": null pointer");
  if (((uintptr_t)k_codes | (uintptr_t)v_codes) & 15)
    return fail(TT_ERR_ARG, std::string(fn) + ": codes must be 16-byte aligned");
  const size_t qb = (size_t)(B * H * T * d) * (dtype == TT_F32 ? 4 : 2);
  const size_t cb = (size_t)(B * Hkv * cap * d / 2), sb = (size_t)(B * Hkv * cap * d / kMxBlock);
  if ((rc = check_no_overlap(fn,
                             {{q, qb, "q"}, {k_codes, cb, "k_codes"}, {k_scales, sb, "k_scales"},
                              {v_codes, cb, "v_codes"}, {v_scales, sb, "v_scales"},
                              {lengths, (size_t)B * sizeof(int), "lengths"}},
                             {{o, qb, "o"}, {lse, (size_t)(B * H * T) * sizeof(float), "lse"}})))
    return rc;
  if ((rc = ensure_init())) return rc;
  hipStream_t st = stream_or_default(stream);
  return dtype == TT_F32 ? launch_d<float>(fn, q, k_codes, k_scales, v_codes, v_scales, lengths, o, lse, B, H, Hkv, T,
                                           cap, d, scale, st)
                         : launch_d<u16>(fn, q, k_codes, k_scales, v_codes, v_scales, lengths, o, lse, B, H, Hkv, T,
                                         cap, d, scale, st);
}
