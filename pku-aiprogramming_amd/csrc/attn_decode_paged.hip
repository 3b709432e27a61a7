// Attention of the newest tokens over a paged K / V cache (paged.h): o = softmax(s
// q K^T) V for T tokens of H query heads over Hkv cached heads, the cache in the
// call's own type or in 8 bits with a scale for each page and head.
//
// The bytes of the cache bound it, K and V each read once, so all R = H / Hkv * T
// query rows that share one K / V head go through the matrix unit as a tile of 16
// columns.  A wave owns a step of keys at a time (32; 16 of fp32) with a running
// maximum and sum of its own:
//   S^T [keys x 16 rows] = K Q^T: a lane's piece of a K row is the operand as it is
//     loaded (8-bit codes after v_cvt_scalef32_pk_bf16_fp8, exactly): the order of
//     the contraction is free, and q is laid out to match.  fp32 pools take the fp32
//     unit.  Result: a lane owns one query row and four keys of each 16.
//   O^T [D x 16 rows] += V^T P^T: P comes out of S^T in the operand's layout.  V
//     rows go through the wave's LDS tile and are read back transposed
//     (ds_read_b64_tr_b16); fp32 needs no transposition, since a lane holds one key
//     an operand there, and columns may be numbered as they were loaded.  P is
//     split into bf16 terms (two for bf16 calls, 2^-17 off; three for fp32 calls,
//     whose q is split into three exact terms too).
// A page is 16 keys or a multiple, so a step's 16 keys never straddle two.  The
// wave holds the next 128 places of its sequence's table in two registers, from
// which a page's number comes without memory's latency.  K of the next step is
// loaded once its registers are free, behind the scores, V behind the store to LDS.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <limits>
#include <optional>
#include <string>
#include <type_traits>

#include "attn_decode_tiles.h"
#include "attn_tiles.h"
#include "paged.h"
#include "tt_internal.h"

namespace tt {
namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x4 mfma_f32_16x16x4(float a, float b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// A lane's share of one row of 16, a quarter: DW dwords in pieces of up to 16 bytes
// that alternate between the four lanes of a row, so that a wave's load takes whole
// runs of a row.
template <typename C, int D>
struct PdRow {
  static constexpr int DW = D * sizeof(C) / 16, PW = DW < 4 ? DW : 4, NP = DW / PW;
  uint32_t w[DW];
  // STREAM: rows that no other workgroup reads are loaded past the caches.
  template <bool STREAM>
  __device__ __forceinline__ void load(const C* row, int g) {
    typedef uint32_t vec __attribute__((ext_vector_type(PW)));
    const vec* from = reinterpret_cast<const vec*>(row) + g;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const vec x = STREAM ? __builtin_nontemporal_load(from + 4 * i) : from[4 * i];
      __builtin_memcpy(w + PW * i, &x, 4 * PW);
    }
  }
};
// The first of the eight values that lane g brings to k step j.
template <typename C, int D>
__device__ __forceinline__ constexpr int pd_first(int j, int g) {
  if (sizeof(C) == 2) return 8 * (4 * j + g);
  return PdRow<C, D>::PW == 4 ? 16 * (4 * (j >> 1) + g) + 8 * (j & 1) : 8 * g;
}
template <int D>
__device__ __forceinline__ bf16x8 pd_operand(const PdRow<u16, D>& x, int j, float) {
  bf16x8 v;
  __builtin_memcpy(&v, x.w + 4 * j, 16);
  return v;
}
template <int D>
__device__ __forceinline__ bf16x8 pd_operand(const PdRow<uint8_t, D>& x, int j, float scale) {
  const uint32_t lo = x.w[2 * j], hi = x.w[2 * j + 1];
  const uint32_t w[4] = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false)),
                         __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true)),
                         __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false)),
                         __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true))};
  return __builtin_bit_cast(bf16x8, w);
}
// Whether a value may be infinite or NaN.
template <int D>
__device__ __forceinline__ bool pd_odd(const PdRow<u16, D>& x, uint32_t) {
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < PdRow<u16, D>::DW; ++i) any |= (x.w[i] & 0x7f807f80u) + 0x00800080u;
  return (any & 0x80008000u) != 0;
}
template <int D>
__device__ __forceinline__ bool pd_odd(const PdRow<uint8_t, D>& x, uint32_t byte) {
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < PdRow<uint8_t, D>::DW; ++i) any |= (x.w[i] & 0x7f7f7f7fu) + 0x01010101u;
  return (any & 0x80808080u) != 0 || byte > kE4MaxByte;
}
__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }
// The finite values, zeros for the others.
__device__ __forceinline__ bf16x8 pd_clean(const bf16x8& x) {
  uint32_t w[4];
  __builtin_memcpy(w, &x, 16);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t odd = ((w[i] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;  // the upper bit of such a half
    w[i] &= ~((odd >> 15) * 0xffffu);
  }
  return __builtin_bit_cast(bf16x8, w);
}
// Four values of a row from column `c` on, in fp32.
__device__ __forceinline__ void pd_four(const u16* row, int c, float, float (&x)[4]) {
  u16 v[4];
  __builtin_memcpy(v, row + c, 8);
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = bf16_to_f32(v[e]);
}
__device__ __forceinline__ void pd_four(const uint8_t* row, int c, float scale, float (&x)[4]) {
  uint32_t v;
  __builtin_memcpy(&v, row + c, 4);
  e4_values(v, x);
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] *= scale;
}
__device__ __forceinline__ void pd_four(const float* row, int c, float, float (&x)[4]) { __builtin_memcpy(x, row + c, 16); }

// The wave's place in its sequence's table: entries [base, base + 64) and the 64
// after them, one a lane.  Pages behind the sequence's last are none.
struct PdTable {
  const int* row;
  int count, base, now, next;
  __device__ __forceinline__ int load(int from) const {
    const int at = from + (int)(threadIdx.x & 63);
    return at < count ? row[at] : -1;
  }
  __device__ __forceinline__ void start(const int* r, int n, int from) {
    row = r, count = n, base = from;
    now = load(base);
    next = load(base + 64);
  }
  // Page `at`: asked for in order, each at most 64 behind the one before.
  __device__ __forceinline__ int page(int at) {
    if (at - base >= 64) {
      base += 64;
      now = next;
      next = load(base + 64);
    }
    return __builtin_amdgcn_readlane(now, at - base);
  }
};

// The maximum is that of the products, the scale sl2 (of log2 e too, above zero:
// its sign goes into q, and zero is the smallest fp32, 2^-149) enters the exponent,
// 2^(sl2 s - sl2 m), one operation a score.
// Workgroup id = (head * tiles + tile) * nsplit + split, head = b Hkv + hkv, tile =
// 16 of the head's R query rows.  Each sequence's own length is cut into nsplit
// spans, so that sequences of any length keep every workgroup busy.
template <typename T, typename C, int D, bool STREAM>
__global__ __launch_bounds__(kMdThreads, 3) void attn_decode_paged_kernel(
    const T* __restrict__ q, const C* __restrict__ kp, const C* __restrict__ vp, const uint8_t* __restrict__ ks,
    const uint8_t* __restrict__ vs, Pages pg, float* __restrict__ part_o, float2* __restrict__ part_ml,
    T* __restrict__ o, float* __restrict__ lse, uint32_t R, uint32_t tokens, uint32_t tiles, uint32_t nsplit,
    float sl2, bool negative) {
  constexpr bool F32 = sizeof(C) == 4, E4 = sizeof(C) == 1;  // fp32 pools; 8-bit ones
  constexpr int U = F32 ? 1 : 2, KEYS = 16 * U;              // 16s of keys, and keys, of a step
  constexpr int W = F32 ? D / 16 : D / 32;                   // k steps (fp32: pieces of four) of a key tile
  constexpr int NQ = sizeof(T) == 4 ? 3 : 1, NP = sizeof(T) == 4 ? 3 : 2;  // terms of q and of the weights
  constexpr int ND = D / 16;                                 // 16-row tiles of O^T
  constexpr int VW = F32 ? (D < 64 ? D / 16 : 4) : 4;        // fp32: neighbouring columns of a lane
  constexpr int VG = F32 ? ND / VW : 1;                      // and groups of them
  __shared__ __align__(256) u16 s_v[kMdWaves][kMdKeys * D];
  __shared__ float s_m[kMdWaves][kMdRows], s_l[kMdWaves][kMdRows];
  static_assert(sizeof(s_v[0]) == kMdRows * D * sizeof(float), "the waves' sums reuse their tiles");

  const int l = threadIdx.x & 63, r = l & 15, g = l >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t unit = blockIdx.x / nsplit, split = blockIdx.x - unit * nsplit;
  const uint32_t head = unit / tiles, row0 = (unit - head * tiles) * kMdRows;
  const int64_t qrow = (int64_t)head * R + row0;  // the tile's first row of q and o
  const int nrows = (int)min((uint32_t)kMdRows, R - row0);

  // Keys that the newest token sees, and that this lane's row sees.
  const uint32_t b = head / pg.hkv, hk = head - b * pg.hkv;
  const int full = pg.lengths[b];
  const int len = pg.pages > 0 ? (int)paged_end(pg, full) : 0, before = (int)tokens - 1;
  const int t = r < nrows ? (int)((row0 + (uint32_t)r) % tokens) : 0;
  const int seen = r < nrows ? (int)min((int64_t)len, (int64_t)full - (before - t)) : 0;
  const int all_see = (int)min((int64_t)len, (int64_t)full - before);  // keys that every row sees
  int kbeg = 0, kend = 0;
  if (len > 0) {
    const uint32_t span = (((uint32_t)len + nsplit - 1) / nsplit + kMdKeys - 1) / kMdKeys * kMdKeys;
    kbeg = (int)min((uint64_t)split * span, (uint64_t)len);
    kend = (int)min((uint32_t)kbeg + span, (uint32_t)len);
  }

  // q in the layout that K has: lane g's values of each k step
  typename std::conditional<F32, f32x4, bf16x8>::type qf[W][F32 ? 1 : NQ];
#pragma unroll
  for (int j = 0; j < W; ++j) {
    if constexpr (F32) {
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
      if (r < nrows) x = *reinterpret_cast<const f32x4*>(q + (qrow + r) * D + 4 * (4 * j + g));
      qf[j][0] = negative ? -x : x;
    } else {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = 0.f;
      if (r < nrows) md_load8(q + (qrow + r) * D + pd_first<C, D>(j, g), x);
      if (negative)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = -x[e];
      md_terms<NQ, true>(x, qf[j]);
    }
  }

  f32x4 acc[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, lsum = 0.f;
  u16* tile = s_v[w];
  constexpr uint32_t kRow = 2 * D;  // bytes of a tile row
  const uint32_t put = lds_addr(tile) + (uint32_t)r * kRow +
                       16u * (uint32_t)((E4 && PdRow<C, D>::PW == 4 ? 2 * g : g) ^ md_exchange<D>(r));
  const int krow = 4 * g + (r >> 2);
  const uint32_t get = lds_addr(tile) + (uint32_t)krow * kRow + 16u * (uint32_t)(((r & 3) >> 1) ^ md_exchange<D>(krow)) +
                       8u * (uint32_t)(r & 1);

  const int slots = (1 << pg.lp) - 1;
  const int64_t head_rows = (int64_t)hk << pg.lp, page_rows = (int64_t)pg.hkv << pg.lp;
  // A step's pages: its first row in the pool (the same for the wave), and what is known of it.
  struct Step {
    int64_t row[U];
    bool has[U];
    uint32_t kb[U], vb[U];
  };
  PdTable table;
  auto look = [&](Step& s, int j0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = j0 + 16 * u;
      int id = table.page(key >> pg.lp);
      s.has[u] = key < kend && id >= 0 && id < pg.pages;
      id = s.has[u] ? id : 0;
      s.row[u] = id * page_rows + head_rows + (key & slots);
      if constexpr (E4) {
        s.kb[u] = ks[(int64_t)id * pg.hkv + hk];
        s.vb[u] = vs[(int64_t)id * pg.hkv + hk];
      }
    }
  };
  // Rows of a 16 past the sequence's end are taken from its last: masked below.
  auto row_of = [&](int row, int key) { return key + 16 <= len ? row : min(row, max(len - 1 - key, 0)); };

  typedef typename std::conditional<F32, float, uint32_t>::type word;
  PdRow<C, D> kr[U];
  PdRow<C, D> vr[F32 ? 1 : U];
  float vf[F32 ? 4 : 1][VG][VW];
  auto fetch_k = [&](const Step& s, int j0) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      kr[u].template load<STREAM>(kp + (s.row[u] * D + row_of(r, j0 + 16 * u) * D), g);
  };
  auto fetch_v = [&](const Step& s, int j0) {
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const C* from = vp + (s.row[0] * D + row_of(4 * g + i, j0) * D + VW * r);
#pragma unroll
        for (int k = 0; k < VG; ++k) {
          typedef float vec __attribute__((ext_vector_type(VW)));
          const vec* p = reinterpret_cast<const vec*>(from + 16 * VW * k);
          const vec x = STREAM ? __builtin_nontemporal_load(p) : *p;
          __builtin_memcpy(vf[i][k], &x, 4 * VW);
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
        vr[u].template load<STREAM>(vp + (s.row[u] * D + row_of(r, j0 + 16 * u) * D), g);
    }
  };

  constexpr int kStep = kMdWaves * KEYS;
  int j0 = kbeg + w * KEYS;
  Step cur, nxt;
  if (j0 < kend) {
    const int64_t page = int64_t(1) << pg.lp;
    table.start(pg.table + (int64_t)b * pg.width, (int)((len + page - 1) >> pg.lp), j0 >> pg.lp);
    look(cur, j0);
    fetch_k(cur, j0);
    fetch_v(cur, j0);
  }
  for (; j0 < kend; j0 += kStep) {
    const bool more = j0 + kStep < kend;
    if (more) look(nxt, j0 + kStep);

    // s[u][i]: key 16 u + 4 g + i of the step, for this lane's row
    f32x4 s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < W; ++j) {
        if constexpr (F32) {
          f32x4 a;
          __builtin_memcpy(&a, kr[u].w + 4 * j, 16);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[u] = mfma_f32_16x16x4(a[e], qf[j][0][e], s[u]);
        } else {
          const bf16x8 a = pd_operand<D>(kr[u], j, e4_scale(E4 ? cur.kb[u] : 0));
#pragma unroll
          for (int n = NQ - 1; n >= 0; --n) s[u] = mfma_bf16_16x16x32(a, qf[j][n], s[u]);
        }
      }
    }
    if (more) fetch_k(nxt, j0 + kStep);

    bool edge = j0 + KEYS > min(kend, all_see);
#pragma unroll
    for (int u = 0; u < U; ++u) edge |= !cur.has[u];
    if (edge) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s[u][i] = cur.has[u] && j0 + 16 * u + 4 * g + i < min(seen, kend) ? s[u][i] : -INFINITY;
    }

    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u)
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
    for (int e = 0; e < 4 * U; ++e) {
      p[e] = fast_exp2(__builtin_fmaf(sl2, s[e >> 2][e & 3], -mb));
      lsum += p[e];
    }

    // A weight of zero must not meet an infinity or a NaN, be it a masked key's or a
    // bf16 term of a weight: such values of V are zeros in the product, and what
    // the rows that see them get is added apart.
    bool odd = false;
    if constexpr (F32) {
      if (edge)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int k = 0; k < VG; ++k)
#pragma unroll
            for (int c = 0; c < VW; ++c) {
              odd |= !finite(vf[i][k][c]);
              vf[i][k][c] = finite(vf[i][k][c]) ? vf[i][k][c] : 0.f;
            }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) odd |= pd_odd<D>(vr[u], E4 ? cur.vb[u] : 0);
    }
    odd = wave_any(odd);

    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < VG; ++k)
#pragma unroll
          for (int c = 0; c < VW; ++c) acc[k * VW + c] = mfma_f32_16x16x4(vf[i][k][c], p[i], acc[k * VW + c]);
      if (more) fetch_v(nxt, j0 + kStep);
    } else {
      bf16x8 pf[NP];
      md_terms<NP>(p, pf);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < W; ++j) {
          bf16x8 x = pd_operand<D>(vr[u], j, e4_scale(E4 ? cur.vb[u] : 0));
          if (odd) x = pd_clean(x);
          lds_st((put ^ (16u * (uint32_t)(pd_first<C, D>(j, 0) / 8))) + u * 16 * kRow, x);
        }
      if (more) fetch_v(nxt, j0 + kStep);
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
    if (odd) {  // rare
      for (int kk = 0; kk < KEYS; ++kk) {
        const int u = U > 1 ? kk >> 4 : 0, in = kk & 15, key = j0 + kk;
        if (key >= kend || !(u ? cur.has[U - 1] : cur.has[0])) continue;
        const float a = (in & 2) ? ((in & 1) ? p[3] : p[2]) : ((in & 1) ? p[1] : p[0]);
        const float z = (in & 2) ? ((in & 1) ? p[4 * U - 1] : p[4 * U - 2]) : ((in & 1) ? p[4 * U - 3] : p[4 * U - 4]);
        const float wgt = __shfl(u ? z : a, 16 * (in >> 2) + r, 64);  // this row's, from the lane that holds the key's
        const C* from = vp + ((u ? cur.row[U - 1] : cur.row[0]) + in) * D;
        const float scale = e4_scale(E4 ? (u ? cur.vb[U - 1] : cur.vb[0]) : 0);
        if (key >= seen) continue;
#pragma unroll
        for (int i = 0; i < ND; ++i)  // columns 16 i + 4 g and three more, in the order that acc has them
          if constexpr (!F32) {
            float x[4];
            pd_four(from, 16 * i + 4 * g, scale, x);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!finite(x[e])) acc[i][e] += wgt * x[e];
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = from[16 * VW * (i / VW) + VW * (4 * g + e) + i % VW];
              if (!finite(x) && edge) acc[i][e] += wgt * x;
            }
          }
      }
    }
    cur = nxt;
  }

  // The waves' sums meet in LDS: [row][D] fp32 over each wave's own tile, chunks
  // of four columns swizzled by the row.
  lsum = sum_rows(lsum);
  float* mine = reinterpret_cast<float*>(tile);
#pragma unroll
  for (int i = 0; i < ND; ++i) {
    f32x4 x = acc[i];
    int d4 = 4 * i + g;
    if constexpr (F32 && VW == 4) {  // columns 64 (i / 4) + 16 g + 4 (i % 4) and three more
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] = acc[i / 4 * 4 + c][i % 4];
      d4 = 16 * (i / 4) + 4 * g + i % 4;
    } else if constexpr (F32) {  // two neighbours a lane: columns 8 g + 4 i and three more
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] = acc[c & 1][2 * i + (c >> 1)];
      d4 = 2 * g + i;
    }
    *reinterpret_cast<f32x4*>(&mine[r * D + 4 * (d4 ^ (r & (D / 4 - 1)))]) = x;
  }
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

constexpr size_t kPdWork = size_t(24) << 20;  // the partials' scratch, of one size so that graphs may keep its address

// Into how many splits to cut the keys: a workgroup costs its keys and about kPdFixed
// more, a CU's time goes by the workgroups that fall to it, up to per_cu of them at
// once, and splits cost the second launch, about kPdMerge keys.
constexpr int64_t kPdFixed = 150, kPdMerge = 300;
inline int64_t pd_splits(int64_t units, int64_t keys, int64_t per_cu, int64_t cus, int64_t most) {
  constexpr int64_t step = kMdWaves * kMdKeys;
  most = std::min(most, (keys + step - 1) / step);
  most = std::min(most, std::max<int64_t>(4, 2 * per_cu * cus / units));
  int64_t best = 1;
  double least = std::numeric_limits<double>::max();
  for (int64_t n = 1; n <= most; n += 1 + n / 64) {  // the host's time counts too
    const int64_t here = (units * n + cus - 1) / cus;
    const int64_t last = here % per_cu, each = ((keys + n - 1) / n + step - 1) / step * step + kPdFixed;
    auto group = [&](int64_t w) { return w > 0 ? (double)w + 0.6 : 0.0; };  // w at once
    const double cost = (double)each * ((double)(here / per_cu) * group(per_cu) + group(last)) +
                        (n > 1 ? (double)(kPdMerge + 4 * n) : 0.0);
    if (cost < least) {
      least = cost;
      best = n;
    }
  }
  return best;
}

struct PdCall {
  const void* q;
  const void *kp, *vp;
  const uint8_t *ks, *vs;
  Pages pg;
  void* o;
  float* lse;
  int64_t B, H, Hkv, tokens;
  float scale;
};

template <typename T, typename C, int D>
int launch(const char* fn, const PdCall& a, hipStream_t st) {
  const int64_t rows = a.B * a.H * a.tokens, R = a.H / a.Hkv * a.tokens, cap = a.pg.width << a.pg.lp;
  const int64_t tiles = (R + kMdRows - 1) / kMdRows, units = a.B * a.Hkv * tiles;
  static const int per_cu = [] {
    int n = 0;
    const hipError_t e = hipOccupancyMaxActiveBlocksPerMultiprocessor(
        &n, (const void*)attn_decode_paged_kernel<T, C, D, true>, kMdThreads, 0);
    if (e != hipSuccess) (void)hipGetLastError();
    return e != hipSuccess || n < 1 ? 3 : n;
  }();
  int64_t nsplit = pd_splits(units, std::max<int64_t>(cap, 1), per_cu, device_cu_count(),
                             (int64_t)(kPdWork / ((size_t)rows * (D + 2) * sizeof(float))));
  void* ws = nullptr;
  std::optional<WorkspaceLease> lease;  // held until both kernels are queued
  if (nsplit < 2 || !lease.emplace().get_fixed(st, kWsPagedDecode, kPdWork, &ws)) nsplit = 1;
  float* part_o = (float*)ws;
  float2* part_ml = (float2*)(part_o + rows * nsplit * D);
  float sl2 = std::fabs(a.scale * kLog2e);
  uint32_t bits;  // 1: the smallest fp32, formed as the host's arithmetic may flush it
  memcpy(&bits, &sl2, sizeof(bits));
  bits = std::max(bits, 1u);
  memcpy(&sl2, &bits, sizeof(bits));
#define TT_PD_LAUNCH(STREAM)                                                                                         \
  hipLaunchKernelGGL((attn_decode_paged_kernel<T, C, D, STREAM>), dim3((unsigned)(units * nsplit)), dim3(kMdThreads), \
                     0, st, (const T*)a.q, (const C*)a.kp, (const C*)a.vp, a.ks, a.vs, a.pg, part_o, part_ml,        \
                     (T*)a.o, a.lse, (uint32_t)R, (uint32_t)a.tokens, (uint32_t)tiles, (uint32_t)nsplit, sl2,        \
                     a.scale < 0.f)
  if (tiles == 1)
    TT_PD_LAUNCH(true);
  else
    TT_PD_LAUNCH(false);
#undef TT_PD_LAUNCH
  TT_LAUNCHED(fn, st);
  if (nsplit > 1) {
    hipLaunchKernelGGL((attn_decode_merge_kernel<T, D>), dim3((unsigned)rows), dim3(256), 0, st, part_o, part_ml,
                       (T*)a.o, a.lse, (int)nsplit);
    TT_LAUNCHED(fn, st);
  }
  return ok();
}

template <typename T, typename C>
int launch_d(const char* fn, const PdCall& a, int64_t d, hipStream_t st) {
  switch (d) {
    case 32: return launch<T, C, 32>(fn, a, st);
    case 64: return launch<T, C, 64>(fn, a, st);
    default: return launch<T, C, 128>(fn, a, st);
  }
}

}  // namespace
}  // namespace tt

using namespace tt;

extern "C" int tt_attn_decode_paged(int dtype, int cache, const void* q, const void* k_pages, const void* v_pages,
                                    const uint8_t* k_scales, const uint8_t* v_scales, const int* table,
                                    const int* lengths, void* o, float* lse, int64_t B, int64_t H, int64_t Hkv,
                                    int64_t T, int64_t d, int64_t npages, int64_t page, int64_t width, float scale,
                                    void* stream) {
  const char* fn = "tt_attn_decode_paged";
  const std::string f(fn);
  int lp = 0, rc = check_paged(fn, dtype, cache, B, Hkv, T, d, npages, page, width, &lp);
  if (rc) return rc;
  if (H < 0 || (Hkv == 0 ? H != 0 : H % Hkv != 0)) return fail(TT_ERR_ARG, f + ": H must be a multiple of Hkv");
  if (B == 0 || H == 0 || T == 0) return ok();
  if (H > (int64_t(1) << 24) || B * H > (int64_t(1) << 24)) return fail(TT_ERR_ARG, f + ": too many heads");
  if (B * H * T > 0x7fffffff) return fail(TT_ERR_ARG, f + ": too many rows");
  // Splits, and the merge's workgroups of a row each, are few: the scratch holds all of their rows.
  if (!grid_fits(B * Hkv * ((H / Hkv * T + kMdRows - 1) / kMdRows), kMdThreads))
    return fail(TT_ERR_ARG, f + ": grid too large");
  if (!q || !o || !lengths) return fail(TT_ERR_ARG, f + ": null pointer");
  if (((uintptr_t)q | (uintptr_t)o) & 15) return fail(TT_ERR_ARG, f + ": q and o must be 16-byte aligned");
  const bool some = npages > 0 && width > 0;
  if (some && (rc = check_pools(fn, cache, k_pages, v_pages, k_scales, v_scales, table, lengths))) return rc;
  const size_t qb = (size_t)(B * H * T * d) * (dtype == TT_F32 ? 4 : 2);
  const size_t pool = (size_t)(npages * Hkv * page * d) * cache_item(cache);
  const size_t sb = cache == TT_E4M3 ? (size_t)(npages * Hkv) : 0;
  if ((rc = check_no_overlap(fn,
                             {{q, qb, "q"},
                              {k_pages, pool, "k_pages"},
                              {v_pages, pool, "v_pages"},
                              {k_scales, sb, "k_scales"},
                              {v_scales, sb, "v_scales"},
                              {table, (size_t)(B * width) * sizeof(int), "table"},
                              {lengths, (size_t)B * sizeof(int), "lengths"}},
                             {{o, qb, "o"}, {lse, (size_t)(B * H * T) * sizeof(float), "lse"}})))
    return rc;
  if ((rc = ensure_init())) return rc;
  hipStream_t st = stream_or_default(stream);
  const PdCall a{q, k_pages, v_pages, k_scales, v_scales, Pages{table, lengths, some ? npages : 0, width, (uint32_t)Hkv, lp},
                 o, lse, B, H, Hkv, T, scale};
  if (dtype == TT_F32)
    return cache == TT_E4M3 ? launch_d<float, uint8_t>(fn, a, d, st) : launch_d<float, float>(fn, a, d, st);
  return cache == TT_E4M3 ? launch_d<u16, uint8_t>(fn, a, d, st) : launch_d<u16, u16>(fn, a, d, st);
}
