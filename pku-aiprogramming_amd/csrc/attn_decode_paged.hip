// Attention of the newest tokens over a paged K / V cache (paged.h): o = softmax(s
// q K^T) V for T tokens of H query heads over Hkv cached heads, the cache in the
// call's own type or in 8 bits with a scale for each page and head.
//
// The bytes of the cache bound it, K and V each read once, so all R = H / Hkv * T
// query rows that share one K / V head go through the matrix unit as a tile of 16
// columns.  A wave owns a step of keys at a time (32; 16 of fp32) with a running
// maximum and sum of its own, and goes through them without meeting the others:
//   K and V rows come straight into the wave's own LDS tiles, a load the whole 128
//     byte lines of neighbouring rows, each tile loaded again as soon as it was read.
//     (Loaded to registers, in the operand's layout, every line took two requests:
//     490 us where this takes 284, of the first case below.)
//   S^T [keys x 16 rows] = K Q^T: a lane reads its piece of a K row; 8-bit codes
//     become bf16 by v_cvt_scalef32_pk_bf16_fp8, exactly.  The order of the
//     contraction is free, and q is laid out to match.  fp32 pools take the fp32
//     unit.  Result: a lane owns one query row and four keys of each 16.
//   O^T [D x 16 rows] += V^T P^T: P comes out of S^T in the operand's layout.  V is
//     read transposed (ds_read_b64_tr_b16, and _tr_b8 with the conversion behind
//     it); fp32 needs no transposition, since a lane holds one key an operand there,
//     and columns may be numbered as they were read.  P is split into three bf16 terms,
//     which hold it exactly, and so is the q of fp32 calls.  (Two would leave 2^-17 of P
//     and gain where the bytes do not bound: a chunk of 512 tokens of 32 / 8 heads x 8192
//     keys 161 us for 178, 8 x 8 heads x 2048 over 8 bits 12.4 for 13.0, but 64 x 32 x
//     8192 640 for 642.)
// A page is 16 keys or a multiple, so a step's 16 keys never straddle two.  The
// wave holds the next 128 places of its sequence's table in registers, from
// which a page's number comes without memory's latency.
// Measured (MI355X, d = 128): 64 sequences of up to 8192 keys, 32 / 8 heads of bf16, 255 us
// (6.3 TB/s); 32 / 32 heads over 8 bits, 647 us (6.6 TB/s); one of 4097 keys, 11.5 us, a
// chain of memory latencies; 3 tokens of 12 x 20 / 4 heads of fp32 over 8 bits, 34.5 us (4.2 TB/s:
// vector work of three terms of q and of the weights).
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

__device__ __forceinline__ f32x4 mfma_f32_16x16x4(float a, float b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// A wave's tile of rows as they lie in a pool, in 16-byte chunks: chunk c of row r
// at chunk c ^ exchange(r), so that chunk c of 16 rows, and four rows' neighbouring
// chunks, spread over the banks.
template <typename C, int D, int ROWS>
struct PdTile {
  static constexpr int ROWB = D * sizeof(C), CPR = ROWB / 16, BYTES = ROWS * ROWB;
  static constexpr int LOADS = BYTES / 1024, RPL = 64 / CPR;  // loads of a wave, rows of a load
  __device__ static __forceinline__ constexpr uint32_t exchange(uint32_t r) {
    return ROWB >= 256 ? r & 15u : (r / (256 / ROWB)) & (CPR - 1);  // the same for rows 16 apart
  }
  __device__ static __forceinline__ uint32_t at(uint32_t r, uint32_t chunk) {
    return r * ROWB + 16u * (chunk ^ exchange(r));
  }
};
// The chunk, and the first of the eight codes in it, that lane g brings to k step j.
template <typename C, int D>
__device__ __forceinline__ constexpr int pd_chunk(int j, int g) {
  return sizeof(C) != 1 ? 4 * j + g : D == 32 ? g >> 1 : 4 * (j >> 1) + g;
}
template <typename C, int D>
__device__ __forceinline__ constexpr int pd_half(int j, int g) {
  return sizeof(C) != 1 ? 0 : D == 32 ? 8 * (g & 1) : 8 * (j & 1);
}
// Four codes as two pairs of bf16.
__device__ __forceinline__ void pd_cvt(uint32_t codes, float scale, uint32_t* w) {
  w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false));
  w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true));
}
__device__ __forceinline__ bf16x8 pd_cvt8(const u32x2& codes, float lo, float hi) {
  uint32_t w[4];
  pd_cvt(codes.x, lo, w);
  pd_cvt(codes.y, hi, w + 2);
  return __builtin_bit_cast(bf16x8, w);
}
// ds_read_b64_tr_b8: within 16 lanes, lane t receives element t % 8 of the 8-byte
// chunks addressed by lanes 2 e + t / 8, e = 0 .. 7 (checked on the MI355X).
__device__ __forceinline__ u32x2 lds_tr8_at(uint32_t a) {
  typedef int i32x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2*)(uintptr_t)a));
}
// glds16 and glds16_at (attn_common.h), non-temporal where NT.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <bool NT>
__device__ __forceinline__ void pd_glds16(const void* sbase, uint32_t voff, uint32_t lds) {
  if constexpr (NT)
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt" ::"v"(voff), "s"(sbase), "s"(lds)
                 : "memory", "m0");
  else
    glds16(sbase, voff, lds);
}
template <bool NT>
__device__ __forceinline__ void pd_glds16_at(const void* p, uint32_t lds) {
  if constexpr (NT)
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt" ::"v"(p), "s"(lds)
                 : "memory", "m0");
  else
    glds16_at(p, lds);
}
#pragma clang diagnostic pop

// At most N of the wave's loads are outstanding (they retire in order), and none of
// its LDS reads: nothing that touches memory moves across either.
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

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

// Waves of a SIMD that the registers are held to: what their tiles let onto a CU, but
// for d = 128 over 8 bits, whose four would leave 128 registers: bf16 calls would keep
// four of their values in memory (64 x 32 heads x 8192 keys 662 us so and 640 with three;
// 16 x 16 x 1024 14.7 and 14.4, one user's 4097 keys 11.1 both).
template <typename C, int D>
constexpr int pd_waves() {
  return sizeof(C) > 1 ? 2 : D == 128 ? 3 : 4;
}

// The wave's place in its sequence's table: entries [base, base + 64) and the 64
// after them, one a lane, -1 where the pool has no such page or the sequence ends;
// of 8-bit pools with their scale bytes, which are loaded 64 pages ahead and their
// entries 128, so that no step waits for either.  (Loaded in the step, the scales
// cost it a latency, and all loads before them: 64 x 32 heads x 8192 keys 790 us for 725.)
template <bool E4>
struct PdTable {
  const int* row;
  const uint8_t *ks, *vs;  // of this head
  int count, pages, hkv, base, id[E4 ? 3 : 2];
  uint32_t kb[2], vb[2];
  __device__ __forceinline__ int load(int from) const {
    const int at = from + (int)(threadIdx.x & 63);
    const int x = at < count ? row[at] : -1;
    return x < pages ? x : -1;
  }
  __device__ __forceinline__ void scales(int i) {
    kb[i] = vb[i] = 127u;
    if (id[i] >= 0) {
      kb[i] = ks[(int64_t)id[i] * hkv];
      vb[i] = vs[(int64_t)id[i] * hkv];
    }
  }
  __device__ __forceinline__ void start(int from) {
    base = from;
#pragma unroll
    for (int i = 0; i < (E4 ? 3 : 2); ++i) id[i] = load(base + 64 * i);
    if constexpr (E4) scales(0), scales(1);
  }
  // The lane that holds place `at`: asked for in order, each at most 64 behind the one before.
  __device__ __forceinline__ int lane(int at) {
    if (at - base >= 64) {
      base += 64;
      id[0] = id[1];
      if constexpr (E4) {
        kb[0] = kb[1], vb[0] = vb[1], id[1] = id[2];
        scales(1);
      }
      id[E4 ? 2 : 1] = load(base + (E4 ? 128 : 64));
    }
    return at - base;
  }
};

// Two floats to and from where every compute unit sees them, past the caches that only some share.
__device__ __forceinline__ void pd_put_far(float* p, float a, float b) {
  const uint64_t x = __float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32);
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 pd_get_far(const float* p) {
  const uint64_t x = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return float2{__uint_as_float((uint32_t)x), __uint_as_float((uint32_t)(x >> 32))};
}

// The maximum is that of the products, the scale sl2 (of log2 e too, above zero:
// its sign goes into q, and zero is the smallest fp32, 2^-149) enters the exponent,
// 2^(sl2 s - sl2 m), one operation a score.
// A workgroup: tile, 16 of the R query rows of head = b Hkv + hkv, and a split of its keys.
// The tiles of a head's split are eight ids apart (the last, fewer than eight splits of all,
// as many): on one XCD, whose L2 hands the keys from one to the next.  (Side by side: 3
// tokens of 3 x 128 / 16 heads x up to 14211 keys 87 us for 65, 8 of 4 x 64 / 8 x 4096 22 for
// 19.  Two tiles of a wave, for which K and V come to LDS once: 58 in the first, but their
// registers leave half the waves; over 8 bits 22 for 19, fp32 at d = 64 91 for 76.)
// Each sequence's own length is cut into nsplit spans, so that sequences of any
// length keep every workgroup busy.
template <typename T, typename C, int D, bool STREAM>
__global__ __launch_bounds__(kMdThreads, (pd_waves<C, D>())) void attn_decode_paged_kernel(
    const T* __restrict__ q, const C* __restrict__ kp, const C* __restrict__ vp, const uint8_t* __restrict__ ks,
    const uint8_t* __restrict__ vs, Pages pg, float* __restrict__ part_o, float2* __restrict__ part_ml,
    T* __restrict__ o, float* __restrict__ lse, uint32_t R, uint32_t tokens, uint32_t tiles, uint32_t nsplit,
    float sl2, bool negative, uint32_t* __restrict__ count) {
  constexpr bool F32 = sizeof(C) == 4, E4 = sizeof(C) == 1;  // fp32 pools; 8-bit ones
  constexpr int U = F32 ? 1 : 2, KEYS = 16 * U;              // 16s of keys, and keys, of a step
  constexpr int W = F32 ? D / 16 : D / 32;                   // k steps (fp32: pieces of four) of a key tile
  constexpr int NQ = sizeof(T) == 4 ? 3 : 1, NP = 3;         // terms of q and of the weights
  constexpr int ND = D / 16;                                 // 16-row tiles of O^T
  constexpr int VW = F32 ? (D < 64 ? D / 16 : 4) : 4;        // fp32: neighbouring columns of a lane
  using Tile = PdTile<C, D, KEYS>;
  __shared__ __align__(1024) char s_tile[kMdWaves][2][Tile::BYTES];
  __shared__ float s_m[kMdWaves][kMdRows], s_l[kMdWaves][kMdRows];
  static_assert(sizeof(s_tile[0]) >= kMdRows * D * sizeof(float), "the waves' sums reuse their tiles");

  const int l = threadIdx.x & 63, r = l & 15, g = l >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t tile = 0, span = blockIdx.x;  // head * nsplit + split
  if constexpr (!STREAM) {
    const uint32_t spans = gridDim.x / tiles, eights = span / (8 * tiles), wide = min(spans - 8 * eights, 8u);
    span -= eights * 8 * tiles;
    tile = span / wide;
    span = 8 * eights + span - tile * wide;
  }
  const uint32_t head = span / nsplit, split = span - head * nsplit, unit = head * tiles + tile;
  const uint32_t row0 = tile * kMdRows;
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

  const int slots = (1 << pg.lp) - 1;
  const int64_t head_rows = (int64_t)hk << pg.lp, page_rows = (int64_t)pg.hkv << pg.lp;
  // A step's 16s: their first rows in the pool (the same for the wave), and what is known of them.
  struct Step {
    int64_t row[U];
    bool has[U];
    int lane[U];
    uint32_t kb[U], vb[U];
  };
  PdTable<E4> table{pg.table + (int64_t)b * pg.width, ks + hk, vs + hk, (len + slots) >> pg.lp,
                    (int)min(pg.pages, (int64_t)0x7fffffff), (int)pg.hkv};
  auto look = [&](Step& s, int j0) {
    // A wave's steps begin at even 16s from where its table does: a step's places are in one 64.
    const int at = table.lane(j0 >> pg.lp);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = j0 + 16 * u;
      s.lane[u] = at + (key >> pg.lp) - (j0 >> pg.lp);
      const int id = __builtin_amdgcn_readlane(table.id[0], s.lane[u]);
      s.has[u] = key < kend && id >= 0;
      s.row[u] = (s.has[u] ? id : 0) * page_rows + head_rows + (key & slots);
      if (u > 0 && key >= kend) s.row[u] = s.row[0];  // rows that have been written
    }
  };
  // The scales of what look() found last: apart, so that the rows' loads need not wait for them.
  auto scales = [&](Step& s) {
    if constexpr (E4)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s.kb[u] = (uint32_t)__builtin_amdgcn_readlane((int)table.kb[0], s.lane[u]);
        s.vb[u] = (uint32_t)__builtin_amdgcn_readlane((int)table.vb[0], s.lane[u]);
      }
  };

  // The step's rows of one pool into a tile.  Rows of a 16 past the sequence's end
  // are taken from its last: masked below.
  const uint32_t tile_k = lds_addr(s_tile[w][0]), tile_v = lds_addr(s_tile[w][1]);
  auto fetch = [&](const Step& s, const C* pool, uint32_t tile, int j0) {
    const bool whole = j0 + KEYS <= len;
#pragma unroll
    for (int n = 0; n < Tile::LOADS; ++n) {
      const uint32_t row = (uint32_t)(n * Tile::RPL) + (uint32_t)l / Tile::CPR;  // of the tile, and its chunk here
      const uint32_t chunk = ((uint32_t)l % Tile::CPR) ^ Tile::exchange(row);
      auto in_half = [&](uint32_t x, int u) { return whole ? x : (uint32_t)min((int)x, max(len - 1 - (j0 + 16 * u), 0)); };
      if constexpr (Tile::RPL <= 16) {
        const int u = n * Tile::RPL / 16;
        pd_glds16<STREAM>(pool + s.row[u] * D, in_half(row - 16u * u, u) * Tile::ROWB + 16u * chunk, tile + 1024u * n);
      } else {
        const int u = row >= 16u ? 1 : 0;
        const int64_t first = u ? s.row[U - 1] : s.row[0];
        pd_glds16_at<STREAM>(reinterpret_cast<const char*>(pool + first * D) + (in_half(row & 15u, u) * Tile::ROWB + 16u * chunk),
                  tile + 1024u * n);
      }
    }
  };

  constexpr int kStep = kMdWaves * KEYS;
  const int jbeg = kbeg + w * KEYS;
  int j0 = jbeg;
  Step cur, nxt;
  if (j0 < kend) {
    table.start(j0 >> pg.lp);
    look(cur, j0);
    fetch(cur, kp, tile_k, j0);
    fetch(cur, vp, tile_v, j0);
    scales(cur);
  }

  // q in the layout that K has: lane g's values of each k step
  typename std::conditional<F32, f32x4, bf16x8>::type qf[W][F32 ? 1 : NQ];
#pragma unroll
  for (int j = 0; j < W; ++j) {
    const int first = (16 * pd_chunk<C, D>(j, g) + pd_half<C, D>(j, g)) / (int)sizeof(C);
    if constexpr (F32) {
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
      if (r < nrows) x = *reinterpret_cast<const f32x4*>(q + (qrow + r) * D + first);
      qf[j][0] = negative ? -x : x;
    } else {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = 0.f;
      if (r < nrows) md_load8(q + (qrow + r) * D + first, x);
      if (negative)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = -x[e];
      md_terms<NQ, true>(x, qf[j]);
    }
  }

  f32x4 acc[ND];
  float m, lsum;
  const uint32_t kread = tile_k + (uint32_t)r * Tile::ROWB;
  const uint32_t kex = Tile::exchange((uint32_t)r);
  // rows 4 g + (0 .. 3) of each 16 of V, and a lane's place in its transposed read
  const int vrow = E4 ? 16 * ((r >> 3) & 1) + 4 * g + ((r >> 1) & 3) : 4 * g + (r >> 2);
  const uint32_t vread = tile_v + (uint32_t)vrow * Tile::ROWB + 8u * (uint32_t)(r & 1);
  const uint32_t vex = Tile::exchange((uint32_t)vrow);

  // s[u][i]: key 16 u + 4 g + i of the step, for this lane's row
  auto scores = [&](const Step& st, f32x4(&s)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      u32x4 x = {0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const uint32_t at = kread + u * 16 * Tile::ROWB + 16u * ((uint32_t)pd_chunk<C, D>(j, g) ^ kex);
        if constexpr (F32) {
          const f32x4 a = lds_ld<f32x4>(at);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[u] = mfma_f32_16x16x4(a[e], qf[j][0][e], s[u]);
        } else {
          bf16x8 a;
          if constexpr (!E4) {
            a = lds_ld<bf16x8>(at);
          } else {
            const float scale = e4_scale(st.kb[u]);
            if constexpr (D == 32)
              a = pd_cvt8(lds_ld<u32x2>(at + 8u * (uint32_t)(g & 1)), scale, scale);
            else {
              if (j % 2 == 0) x = lds_ld<u32x4>(at);
              a = pd_cvt8(j % 2 == 0 ? u32x2{x.x, x.y} : u32x2{x.z, x.w}, scale, scale);
            }
          }
#pragma unroll
          for (int n = NQ - 1; n >= 0; --n) s[u] = mfma_bf16_16x16x32(a, qf[j][n], s[u]);
        }
      }
    }
  };
  // whether some row does not see some key of the step
  auto at_edge = [&](const Step& st, int j0) {
    bool edge = j0 + KEYS > min(kend, all_see);
#pragma unroll
    for (int u = 0; u < U; ++u) edge |= !st.has[u];
    return edge;
  };
  auto mask = [&](const Step& st, f32x4(&s)[U], int j0) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        s[u][i] = st.has[u] && j0 + 16 * u + 4 * g + i < min(seen, kend) ? s[u][i] : -INFINITY;
  };

  // One step: the last one (MORE = false) loads nothing.  CAREFUL: without V's
  // infinite and NaN values.
  auto step = [&](auto more, auto careful) {
    constexpr bool MORE = decltype(more)::value, CAREFUL = decltype(careful)::value;
    if constexpr (MORE) {
      look(nxt, j0 + kStep);
      scales(nxt);
    }
    wait_loads<Tile::LOADS>();  // V's may go on
    f32x4 s[U];
    scores(cur, s);
    if constexpr (MORE) {
      wait_reads();
      fetch(nxt, kp, tile_k, j0 + kStep);
    }
    if (at_edge(cur, j0)) mask(cur, s, j0);

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

    wait_loads<MORE ? Tile::LOADS : 0>();  // V is there; the next K may go on
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t row = (uint32_t)(4 * g + i);
#pragma unroll
        for (int k = 0; k < ND / VW; ++k) {
          float v[VW];
          if constexpr (VW == 4) {
            const f32x4 x = lds_ld<f32x4>(tile_v + Tile::at(row, (uint32_t)(16 * k + r)));
            __builtin_memcpy(v, &x, 16);
          } else {
            typedef float f32x2 __attribute__((ext_vector_type(2)));
            const f32x2 x = lds_ld<f32x2>(tile_v + Tile::at(row, (uint32_t)(r >> 1)) + 8u * (uint32_t)(r & 1));
            v[0] = x[0], v[1] = x[1];
          }
#pragma unroll
          for (int c = 0; c < VW; ++c) {
            if (CAREFUL && !finite(v[c])) v[c] = 0.f;
            acc[k * VW + c] = mfma_f32_16x16x4(v[c], p[i], acc[k * VW + c]);
          }
        }
      }
    } else {
      bf16x8 pf[NP];
      md_terms<NP>(p, pf);
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        bf16x8 a;
        if constexpr (E4) {
          const uint32_t at = vread + 16u * ((uint32_t)i ^ vex);
          a = pd_cvt8(lds_tr8_at(at), e4_scale(cur.vb[0]), e4_scale(cur.vb[U - 1]));
        } else {
          const uint32_t at = vread + 16u * ((uint32_t)(2 * i + ((r & 3) >> 1)) ^ vex);
          a = lds_tr16x2_at(at, at + 16 * Tile::ROWB);
        }
        if constexpr (CAREFUL) a = pd_clean(a);
#pragma unroll
        for (int n = NP - 1; n >= 0; --n) acc[i] = mfma_bf16_16x16x32(a, pf[n], acc[i]);
      }
    }
    if constexpr (MORE) {
      wait_reads();
      fetch(nxt, vp, tile_v, j0 + kStep);
    }
  };
  auto steps = [&](auto careful) {
#pragma unroll
    for (int i = 0; i < ND; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY, lsum = 0.f;
    if (j0 >= kend) return;
    for (; j0 + kStep < kend; j0 += kStep) {
      step(std::true_type(), careful);
      cur = nxt;
    }
    step(std::false_type(), careful);
  };
  steps(std::false_type());

  // A weight of zero must not meet an infinity or a NaN of V, be it a masked key's
  // or a bf16 term of a weight.  Where one was met, some sum shows it (rare): then
  // the steps are gone through again without such values, and what the rows that
  // see their keys get of them is added under the weights of the final maximum.
  bool odd = false;
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) odd |= !finite(acc[i][e]);
  if (wave_any(odd && r < nrows)) {
    auto again = [&](auto&& body) {
      j0 = jbeg;
      wait_reads();
      table.start(j0 >> pg.lp);
      look(cur, j0);
      scales(cur);
      fetch(cur, kp, tile_k, j0);
      body();
    };
    again([&] {
      fetch(cur, vp, tile_v, j0);
      steps(std::true_type());
    });
    const float mb = m == -INFINITY ? 0.f : sl2 * m;
    again([&] {
      for (; j0 < kend; j0 += kStep) {
        if (j0 != jbeg) {
          wait_reads();
          look(cur, j0);
          scales(cur);
          fetch(cur, kp, tile_k, j0);
        }
        wait_loads<0>();
        f32x4 s[U];
        scores(cur, s);
        if (at_edge(cur, j0)) mask(cur, s, j0);
#pragma unroll
        for (int u = 0; u < U; ++u)
          for (int in = 0; in < 16 && cur.has[u]; ++in) {
            const int key = j0 + 16 * u + in;
            float wgt = (in & 2) ? ((in & 1) ? s[u][3] : s[u][2]) : ((in & 1) ? s[u][1] : s[u][0]);
            wgt = __shfl(wgt, 16 * (in >> 2) + r, 64);  // this row's score, from the lane that holds the key's
            wgt = fast_exp2(__builtin_fmaf(sl2, wgt, -mb));
            if (key >= min(seen, kend)) continue;
            const C* from = vp + (cur.row[u] + in) * D;
#pragma unroll
            for (int i = 0; i < ND; ++i) {  // the columns that acc[i] has here
              float x[4];
              if constexpr (F32) {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = from[16 * VW * (i / VW) + VW * (4 * g + e) + i % VW];
              } else {
                pd_four(from, 16 * i + 4 * g, e4_scale(E4 ? cur.vb[u] : 0), x);
              }
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (!finite(x[e])) acc[i][e] += wgt * x[e];
            }
          }
      }
    });
  }

  // The waves' sums meet in LDS: [row][D] fp32 over each wave's own tile, chunks
  // of four columns swizzled by the row.
  lsum = sum_rows(lsum);
  float* mine = reinterpret_cast<float*>(s_tile[w]);
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
      const float* theirs = reinterpret_cast<const float*>(s_tile[i]);
      den += wgt * s_l[i][row];
      num += wgt * *reinterpret_cast<const f32x4*>(&theirs[row * D + 4 * (d4 ^ (row & (D / 4 - 1)))]);
    }
    if (nsplit > 1) {
      const int64_t at = (qrow + row) * nsplit + split;
      if (count) {
        pd_put_far(part_o + at * D + 4 * d4, num[0], num[1]);
        pd_put_far(part_o + at * D + 4 * d4 + 2, num[2], num[3]);
        if (d4 == 0) pd_put_far(&part_ml[at].x, top, den);
      } else {
        *reinterpret_cast<f32x4*>(part_o + at * D + 4 * d4) = num;
        if (d4 == 0) part_ml[at] = float2{top, den};
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) md_put(o + (qrow + row) * D + 4 * d4 + e, md_quotient<T>(num[e], den));
      if (d4 == 0 && lse) lse[qrow + row] = md_lse(top, den);
    }
  }
  if (nsplit == 1 || !count) return;

  // The last workgroup of these rows to get here merges them: a workgroup's sums are
  // where all others see them once its stores have ended, before it counts itself.
  wait_loads<0>();
  __syncthreads();
  __shared__ uint32_t s_before;
  if (threadIdx.x == 0) s_before = atomicInc(count + unit, nsplit - 1);  // back at zero for the next call
  __syncthreads();
  if (s_before != nsplit - 1) return;
  // A wave a row: its splits' maxima and sums a lane each, D / 4 lanes to a partial.
  constexpr int TPR = D / 4, G = 64 / TPR;
  const int c = l % TPR, gr = l / TPR;
  for (int row = w; row < nrows; row += kMdWaves) {
    const int64_t first = (qrow + row) * nsplit;
    float2 ml = {-INFINITY, 0.f};
    if ((uint32_t)l < nsplit) ml = pd_get_far(&part_ml[first + l].x);
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    constexpr int UN = 8;
    float wgt = 0.f, mx = -INFINITY, den = 0.f;
    for (uint32_t i0 = 0; i0 < nsplit; i0 += G * UN) {
      float2 x[UN][2];
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const uint32_t i = min(i0 + u * G + gr, nsplit - 1);
        const float* po = part_o + (first + i) * D + 4 * c;
        x[u][0] = pd_get_far(po);
        x[u][1] = pd_get_far(po + 2);
      }
      if (i0 == 0) {  // behind the first partials' loads
        mx = ml.x;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) mx = vmax(mx, __shfl_xor(mx, off, 64));
        wgt = fast_exp2(ml.x - (mx == -INFINITY ? 0.f : mx));
        den = wgt * ml.y;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) den += __shfl_xor(den, off, 64);
      }
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const uint32_t i = i0 + u * G + gr;
        const float a = __shfl(wgt, (int)(i & 63u), 64);
        if (i < nsplit) sum += a * f32x4{x[u][0].x, x[u][0].y, x[u][1].x, x[u][1].y};
      }
    }
#pragma unroll
    for (int off = TPR; off < 64; off <<= 1)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += __shfl_xor(sum[e], off, 64);
    if (gr == 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) md_put(o + (qrow + row) * D + 4 * c + e, md_quotient<T>(sum[e], den));
      if (c == 0 && lse) lse[qrow + row] = md_lse(mx, den);
    }
  }
}

__global__ __launch_bounds__(256) void pd_zero_kernel(uint32_t* p, int n) {
  for (int i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) p[i] = 0u;
}

// Scratch, of one size so that graphs may keep its address: counts of the units'
// workgroups, zero between calls, and the partials.
constexpr int64_t kPdCounts = 16384;
constexpr size_t kPdPartials = size_t(24) << 20, kPdWork = kPdPartials + kPdCounts * sizeof(uint32_t);
// The last workgroup of a unit merges its splits where they are short, few, and a
// wave has one row of them; else a launch of its own does.  By it and by the launch (us):
// 8 x 8 heads x 300 keys 8.6 and 11.3, 1 x 32 x 4097 16.2 and 17.1, 1 x 32 / 8 x 4097 11.1
// and 11.6; but 16 x 32 / 8 x 16383 126 and 123, and with eight rows of a head, 4 x 64 /
// 8 x 4096, 31.7 and 27.6: partials past the caches cost more than those that stay there.
constexpr int64_t kPdMergeSpan = 512, kPdMergeSplits = 40;

// Into how many splits to cut the keys: a workgroup costs its keys and about kPdFixed
// more, a CU's time goes by the workgroups that fall to it, up to per_cu of them at
// once, and splits cost the second launch, about kPdMerge keys.  Of eighteen sizes, one
// sequence of 128 keys to 64 of 8192, within 4 % of the best number in each; 80 to 250 and
// 150 to 600 in place of the two choose the same but for 16 x 8 heads x 1024 and 8 x 8 x 300.
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
                             (int64_t)(kPdPartials / ((size_t)rows * (D + 2) * sizeof(float))));
  void* ws = nullptr;
  std::optional<WorkspaceLease> lease;  // held until both kernels are queued
  bool fresh = false;
  if (nsplit < 2 || !lease.emplace().get_fixed(st, kWsPagedDecode, kPdWork, &ws, &fresh)) nsplit = 1;
  if (fresh) {
    hipLaunchKernelGGL(pd_zero_kernel, dim3(16), dim3(256), 0, st, (uint32_t*)ws, (int)kPdCounts);
    if (const int rc = lease->cleared(fn, st, kWsPagedDecode)) return rc;
  }
  const bool fused = nsplit > 1 && nsplit <= kPdMergeSplits && cap <= nsplit * kPdMergeSpan && R <= kMdWaves &&
                     units <= kPdCounts;
  uint32_t* count = fused ? (uint32_t*)ws : nullptr;
  float* part_o = (float*)ws + kPdCounts;
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
                     a.scale < 0.f, count)
  // No second workgroup of a sequence reads the same keys: past the caches (64 x 32 / 8 heads
  // x 8192 keys 359 -> 316 us, over 8 bits with 32 heads 726 -> 660).  Else they are to be
  // found there.  Sequences that share pages, which the host does not see, lose by it where
  // they are many: of one prefix alone 82 -> 98 us and 242 -> 317, 8 of 8 bits 19 both.
  if (tiles == 1)
    TT_PD_LAUNCH(true);
  else
    TT_PD_LAUNCH(false);
#undef TT_PD_LAUNCH
  TT_LAUNCHED(fn, st);
  if (nsplit > 1 && !fused) {
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
