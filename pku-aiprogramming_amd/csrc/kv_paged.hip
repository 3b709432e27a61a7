// New keys and values into a paged cache, the keys normed and rotated on the way,
// and a cache read back to contiguous rows (paged.h, rope.h).
//
// Both move each value once with little arithmetic, so the bytes bound them.  Into
// 16 or 32 bits, a thread keeps one token's pairs, its angles and its page, and
// goes through the heads, as in the kernel that norms and rotates queries.  Into 8
// bits, a workgroup owns a page of some heads of K or V, whose scales it alone
// changes: of each head it forms the new rows once, in registers, for their largest
// value, and stores their codes; where the scale grows it rounds the page's older
// rows again.  K is normed and rotated in 64 bits there and cut to 32 with the last
// bit set where anything was cut off, so that each code is the nearest to the exact
// value and not to a neighbour of it.
// Measured (MI355X): 4 x 4001 tokens of 8 heads of 128 in fp32, 166 MB, 34 us (4.9 TB/s),
// 16 x 16 heads 288 us (5.4 TB/s); 8 x 4000 tokens of bf16 into 8 bits 46 us, in which a
// third of the wave cycles issue vector instructions, with two waves a SIMD (64-bit values in
// registers), and read back 23 us (5.9 TB/s).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "attn_tiles.h"
#include "paged.h"
#include "rope.h"
#include "tt_internal.h"

namespace tt {
namespace {

constexpr int kPgThreads = 256;
// Heads of a workgroup of the 8-bit append, under angles formed once in 64 bits (8 x 4000
// tokens of 8 heads of 128: 69 -> 57 us); fewer where there would be fewer than four
// workgroups a CU (eight: 8 x 40 tokens 25 -> 24 us with the cache read back, but 4 x 2000 of
// 16 heads of fp32 48 -> 51).
constexpr int64_t kPgHeads = 8;

template <typename T>
struct PgNew {  // new rows of K and V: token-major with ld values a token, or [B][Hkv][T][D] (0)
  const T *k, *v;
  int64_t ldk, ldv;
  const float* weight;  // of K's norm, or null
};

// A workgroup: 256 / LPR tokens, HC heads of K's chunks and then V's, loaded before
// the tokens' places are looked up.
template <typename T, int D, int HC>
__global__ __launch_bounds__(kPgThreads) void kv_append_kernel(PgNew<T> in, Rope rp, Pages pg, T* __restrict__ kp,
                                                               T* __restrict__ vp, uint32_t rows, uint32_t tokens,
                                                               uint32_t chunks) {
  constexpr int N = Chunk<T>::N, LPR = D / (2 * N), TPB = kPgThreads / LPR;
  const uint32_t tile = blockIdx.x / (2 * chunks), part = blockIdx.x - tile * 2 * chunks;
  const bool is_v = part >= chunks;
  const int heads = (int)pg.hkv, lo = (int)(is_v ? part - chunks : part) * HC, hi = min(lo + HC, heads);
  const uint32_t n = tile * TPB + threadIdx.x / LPR;
  if (n >= rows) return;  // whole rows of lanes
  const uint32_t b = n / tokens, t = n - b * tokens;
  const bool rotate = !is_v && rp.freq, norm = !is_v && in.weight;
  const Lay<N> lay(threadIdx.x % LPR, rotate ? rp.rot : 0, rp.inter != 0);
  const T* x = is_v ? in.v : in.k;
  const int64_t ld = is_v ? in.ldv : in.ldk, xs = ld ? D : (int64_t)tokens * D;
  x = ld ? x + (int64_t)n * ld : x + ((int64_t)b * heads * tokens + t) * D;
  uint4 r[HC][2];
#pragma unroll
  for (int u = 0; u < HC; ++u) {
    const int64_t at = min(lo + u, hi - 1) * xs;
    r[u][0] = ldg16(x + at + lay.a);
    r[u][1] = ldg16(x + at + lay.b);
  }
  const int64_t pos = (int64_t)pg.lengths[b] - tokens + t;
  if (pos < 0 || (pos >> pg.lp) >= pg.width) return;
  const int64_t page = pg.table[b * pg.width + (pos >> pg.lp)];
  if (page < 0 || page >= pg.pages) return;
  const int64_t row = ((page * heads) << pg.lp) + (pos & ((1 << pg.lp) - 1)), ys = (int64_t)D << pg.lp;  // of head 0
  T* y = (is_v ? vp : kp) + row * D;
  if (rotate || norm) {
    RopeTurn<N> turn;
    float c[N], s[N], w[2 * N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      c[e] = s[e] = 0.f;
      w[e] = norm ? in.weight[lay.a + e] : 1.f;
      w[N + e] = norm ? in.weight[lay.b + e] : 1.f;
    }
    if (lay.turns) rope_angles<N>(rp.freq + lay.pair, rp.positions ? rope_position(rp, b, t, tokens) : pos, c, s);
    turn.set(c, s, w, lay.turns, rp.inter != 0);
#pragma unroll
    for (int u = 0; u < HC; ++u) {
      float f[2 * N];
      Chunk<T>::get(r[u][0], f);
      Chunk<T>::get(r[u][1], f + N);
      turn(f, norm ? rope_rms<N, LPR>(f, rp.eps) : 1.f, lay.turns, rp.inter != 0);
      r[u][0] = Chunk<T>::put(f);
      r[u][1] = Chunk<T>::put(f + N);
    }
  }
#pragma unroll
  for (int u = 0; u < HC; ++u)
    if (lo + u < hi) {
      *reinterpret_cast<uint4*>(y + (lo + u) * ys + lay.a) = r[u][0];
      *reinterpret_cast<uint4*>(y + (lo + u) * ys + lay.b) = r[u][1];
    }
}

// x in fp32, cut off, the last bit set where anything was: on the same side as x
// of every number of fewer bits and of every middle between two of them.
__device__ __forceinline__ float cut_odd(double x) {
  const float f = (float)x;
  uint32_t bits = __float_as_uint(f);
  if ((bits & 0x7f800000u) != 0x7f800000u) {
    bits -= __builtin_fabs((double)f) > __builtin_fabs(x) ? 1u : 0u;
    bits |= (double)__uint_as_float(bits) != x ? 1u : 0u;
  } else if (__builtin_isfinite(x)) {
    bits -= 1u;  // past the largest fp32: that
  }
  return __uint_as_float(bits);
}
// M of them.  The digits come by shifts where all are of fp32's normal range: one test
// for the M, since zeros are rare among values.
template <int M>
__device__ __forceinline__ void cut_odd(const double (&x)[M], float (&f)[M]) {
  uint32_t odd = 0;
#pragma unroll
  for (int e = 0; e < M; ++e) {
    const uint64_t u = (uint64_t)__double_as_longlong(x[e]);
    const uint32_t hi = (uint32_t)(u >> 32), lo = (uint32_t)u;
    odd = max(odd, (hi << 1) - 2 * 0x38100000u);
    const uint32_t digits = __builtin_amdgcn_alignbit(hi, lo, 29) + 0x40000000u;  // of an exponent 896 less
    f[e] = __uint_as_float((hi & 0x80000000u) | (digits & 0x7fffffffu) | min(lo & 0x1fffffffu, 1u));
  }
  if (odd >= 2 * (0x47f00000u - 0x38100000u))
#pragma unroll
    for (int e = 0; e < M; ++e) f[e] = cut_odd(x[e]);
}

// A workgroup: the new tokens of one page, NEW at most, heads [first, first + heads) of
// K (blockIdx.y 0) or V (1), one after another, under the angles that it forms once.
// NEW goes by the call, not by the page: 16 tokens into pages of 64, 56 sequences of 32
// heads, 44 -> 29 us with the cache read back.
// Workgroup id = (b * count + i) * groups + group, i = 0 .. count - 1 the pages from
// the one that the first new token goes to.  All of K's come first: ids of K and V in
// turn, arithmetic beside memory, take longer (8 x 4000 tokens 70 -> 87 us).
template <typename T, int D, int NEW>
struct PgTile {
  static constexpr int N = Chunk<T>::N, LPR = D / (2 * N), LANES = NEW * LPR;
  // 16 values a side of the pairs a thread at most: 8 x 2000 tokens of 16 heads in pages of
  // 128 take 81 us by 512 threads and 102 by 256; of 64, 256 threads 73 and 512 89.
  static constexpr int MOST = LANES * N / 16 > kPgThreads ? LANES * N / 16 : kPgThreads;
  static constexpr int THREADS = LANES < 64 ? 64 : LANES > MOST ? MOST : LANES;
  static constexpr int ITER = (LANES + THREADS - 1) / THREADS, ROWS = THREADS / LPR;  // rows of an iteration
};
template <typename T, int D, int NEW>
__global__ __launch_bounds__((PgTile<T, D, NEW>::THREADS)) void kv_append_e4m3_kernel(
    PgNew<T> in, Rope rp, Pages pg, uint8_t* __restrict__ kp, uint8_t* __restrict__ vp, uint8_t* __restrict__ ks,
    uint8_t* __restrict__ vs, uint32_t tokens, uint32_t count, uint32_t groups, uint32_t heads) {
  using P = PgTile<T, D, NEW>;
  constexpr int N = P::N, LPR = P::LPR, ITER = P::ITER, WAVES = P::THREADS / 64;
  __shared__ uint32_t s_top[2][WAVES];
  const uint32_t group = blockIdx.x % groups, bi = blockIdx.x / groups, b = bi / count, i = bi - b * count;
  const uint32_t h0 = group * heads, h1 = min(h0 + heads, pg.hkv);
  const bool is_v = blockIdx.y != 0;
  const int64_t length = pg.lengths[b], end = paged_end(pg, length), first = max(length - (int64_t)tokens, (int64_t)0);
  const int64_t j = (first >> pg.lp) + i, base = j << pg.lp;
  if (base >= end) return;
  const int64_t page = pg.table[b * pg.width + j];
  if (page < 0 || page >= pg.pages) return;
  // rows [old, fill) are new
  const int old = (int)max(first - base, (int64_t)0), fill = (int)min(end - base, (int64_t)1 << pg.lp);
  if (old >= fill) return;
  const bool norm = !is_v && in.weight, turns = !is_v && rp.freq;
  const Lay<N> lay(threadIdx.x % LPR, turns ? rp.rot : 0, rp.inter != 0);
  const int row0 = old + (int)threadIdx.x / LPR;  // and every P::ROWS from there
  const T* x = is_v ? in.v : in.k;
  const int64_t ld = is_v ? in.ldv : in.ldk;
  bool mine[ITER];
  const T* from[ITER];  // this lane's rows of head h0
  const int64_t step = ld ? D : (int64_t)tokens * D;
#pragma unroll
  for (int it = 0; it < ITER; ++it) {
    const int row = row0 + it * P::ROWS;
    mine[it] = row < fill;
    const int64_t t = base + (mine[it] ? row : old) - (length - tokens);
    from[it] = (ld ? x + ((int64_t)b * tokens + t) * ld + h0 * D : x + (((int64_t)b * pg.hkv + h0) * tokens + t) * D);
  }
  uint4 raw[ITER][2];
  auto load = [&](uint32_t h) {
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
      raw[it][0] = ldg16(from[it] + (h - h0) * step + lay.a);
      raw[it][1] = ldg16(from[it] + (h - h0) * step + lay.b);
    }
  };
  load(h0);

  double c[ITER][N], s[ITER][N];
  float w[2 * N];
  if (lay.turns)
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
      const int64_t row = row0 + it * P::ROWS, t = base + row - (length - tokens);
      if (mine[it]) rope_angles<N>(rp.freq + lay.pair, rp.positions ? rope_position(rp, b, t, tokens) : base + row, c[it], s[it]);
    }
  if (norm)
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = in.weight[lay.a + e], w[N + e] = in.weight[lay.b + e];

  for (uint32_t h = h0; h < h1; ++h) {
    uint8_t* scale_at = (is_v ? vs : ks) + page * pg.hkv + h;
    const uint32_t before = old > 0 ? *scale_at : 0u;
    float f[ITER][2 * N];
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
      Chunk<T>::get(raw[it][0], f[it]);
      Chunk<T>::get(raw[it][1], f[it] + N);
    }
    if (h + 1 < h1) load(h + 1);
    uint32_t top = 0;
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
      if (!mine[it]) continue;
      if (norm || turns) {
        double g[2 * N];
#pragma unroll
        for (int e = 0; e < 2 * N; ++e) g[e] = f[it][e];
        if (norm) rope_scale<N>(g, rope_rms<N, LPR>(g, rp.eps), w);
        if (lay.turns) rope_turn<N>(g, c[it], s[it], rp.inter != 0);
        cut_odd(g, f[it]);
      }
      float most = 0.f;  // NaN is passed over, an infinity shows
#pragma unroll
      for (int e = 0; e < 2 * N; ++e) most = __builtin_fmaxf(most, __builtin_fabsf(f[it][e]));
      top = max(top, __float_as_uint(most));
      if (__float_as_uint(most) == 0x7f800000u) {  // rare: the largest of the finite ones
        top = 0;
#pragma unroll
        for (int i = 0; i <= it; ++i)
#pragma unroll
          for (int e = 0; e < 2 * N; ++e) {
            const uint32_t m = __float_as_uint(f[i][e]) & 0x7fffffffu;
            top = max(top, mine[i] && m < 0x7f800000u ? m : 0u);
          }
      }
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, 64));
    if constexpr (WAVES > 1) {  // two places, so that one barrier a head does
      uint32_t* place = s_top[(h - h0) & 1];
      if ((threadIdx.x & 63) == 0) place[threadIdx.x >> 6] = top;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < WAVES; ++i) top = max(top, place[i]);
    }
    uint32_t byte = e4_scale_byte(top);
    if (old > 0) byte = max(byte, before);
    const float inverse = byte > 253u ? 0.f : e4_inverse(byte);
    uint8_t* codes = (is_v ? vp : kp) + ((page * pg.hkv + h) << pg.lp) * D;
    auto store = [&](auto clamp) {
      constexpr bool CLAMP = decltype(clamp)::value;
#pragma unroll
      for (int it = 0; it < ITER; ++it) {
        if (!mine[it]) continue;
        uint8_t* to = codes + (row0 + it * P::ROWS) * D;
        if constexpr (N == 8) {
          *reinterpret_cast<uint2*>(to + lay.a) =
              uint2{e4_codes<CLAMP>(f[it], inverse), e4_codes<CLAMP>(f[it] + 4, inverse)};
          *reinterpret_cast<uint2*>(to + lay.b) =
              uint2{e4_codes<CLAMP>(f[it] + 8, inverse), e4_codes<CLAMP>(f[it] + 12, inverse)};
        } else {
          *reinterpret_cast<uint32_t*>(to + lay.a) = e4_codes<CLAMP>(f[it], inverse);
          *reinterpret_cast<uint32_t*>(to + lay.b) = e4_codes<CLAMP>(f[it] + 4, inverse);
        }
      }
    };
    if (byte < kE4MaxByte)
      store(std::false_type());
    else  // the largest scale, past which values are
      store(std::true_type());
    if (old > 0 && byte != before) {  // past 2^-126 nothing is left of them
      const int down = (int)byte - (int)before;
      const float by = down < 126 ? __uint_as_float((uint32_t)(127 - down) << 23) : 0.f;
      for (int u = threadIdx.x; u < old * (D / 4); u += P::THREADS) {
        uint32_t* at = reinterpret_cast<uint32_t*>(codes) + u;
        float v[4];
        e4_values(*at, v);
        *at = e4_codes(v, by);
      }
    }
    if (threadIdx.x == 0 && (old == 0 || byte != before)) *scale_at = (uint8_t)byte;
  }
}

// Rows that fill more than this go by the caches: 8 x 8 heads x 4096 keys of 128 in
// 8 bits, 134 MB as bf16, with their append 75 -> 68 us.  Smaller ones the next kernel may still find there.
constexpr int64_t kPgNtBytes = int64_t(64) << 20;
// Rows [B][Hkv][L][D] of T from a pool of C, 16 bytes of them a lane and kPgUnroll rows:
// workgroup id = head * tiles + tile of kPgUnroll 256 / W rows.  Of one, two, four and eight
// rows a lane 8 x 4000 tokens appended and read back take 69.5, 67.9, 69.8 and 73.0 us.
constexpr int kPgUnroll = 2;
template <typename T, typename C, int D, bool NT>
__global__ __launch_bounds__(kPgThreads) void kv_gather_kernel(const C* __restrict__ kp, const C* __restrict__ vp,
                                                               const uint8_t* __restrict__ ks,
                                                               const uint8_t* __restrict__ vs, Pages pg,
                                                               T* __restrict__ k, T* __restrict__ v, uint32_t L,
                                                               uint32_t tiles) {
  constexpr int N = Chunk<T>::N, W = D / N, ROWS = kPgThreads / W;  // values of a word, words of a row, rows at once
  const C* pool = blockIdx.y ? vp : kp;
  const uint8_t* scales = blockIdx.y ? vs : ks;
  T* out = blockIdx.y ? v : k;
  const uint32_t head = blockIdx.x / tiles, tile = blockIdx.x - head * tiles;
  const uint32_t b = head / pg.hkv, h = head - b * pg.hkv, c = threadIdx.x % W;
  const int64_t end = min(paged_end(pg, pg.lengths[b]), (int64_t)L);
  const int64_t j0 = (int64_t)tile * (ROWS * kPgUnroll) + threadIdx.x / W;
  typedef uint32_t vec __attribute__((ext_vector_type(N * sizeof(C) / 4)));
  vec x[kPgUnroll];
  uint32_t byte[kPgUnroll];
  bool has[kPgUnroll];
#pragma unroll
  for (int i = 0; i < kPgUnroll; ++i) {
    const int64_t j = j0 + i * ROWS;
    int64_t page = -1;
    if (j < end) page = pg.table[b * pg.width + (j >> pg.lp)];
    has[i] = page >= 0 && page < pg.pages;
    if (!has[i]) continue;
    x[i] = *reinterpret_cast<const vec*>(pool + (((page * pg.hkv + h) << pg.lp) + (j & ((1 << pg.lp) - 1))) * D + c * N);
    if constexpr (sizeof(C) == 1) byte[i] = scales[page * pg.hkv + h];
  }
#pragma unroll
  for (int i = 0; i < kPgUnroll; ++i) {
    if (!has[i]) continue;
    uint4 y;
    if constexpr (sizeof(C) == 1) {
      float f[N];
#pragma unroll
      for (int e = 0; e < N / 4; ++e) e4_values(x[i][e], f + 4 * e);
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] *= e4_scale(byte[i]);
      y = Chunk<T>::put(f);
    } else {
      __builtin_memcpy(&y, &x[i], 16);
    }
    u32x4* to = reinterpret_cast<u32x4*>(out + ((int64_t)head * L + j0 + i * ROWS) * D + c * N);
    const u32x4 z = {y.x, y.y, y.z, y.w};
    if constexpr (NT)
      __builtin_nontemporal_store(z, to);
    else
      *to = z;
  }
}

#define TT_PG_DIM(CALL)                               \
  switch (d) {                                        \
    case 32: { constexpr int D = 32; CALL; break; }   \
    case 64: { constexpr int D = 64; CALL; break; }   \
    default: { constexpr int D = 128; CALL; break; }  \
  }

template <typename T>
int append_launch(const char* fn, const PgNew<T>& in, const Rope& rp, const Pages& pg, void* kp, void* vp, int64_t B,
                  int64_t tokens, int64_t d, hipStream_t st) {
  // as the kernel that rotates queries: four heads a workgroup, or one where they would be few
  const int64_t tpb = kPgThreads / (d / (2 * Chunk<T>::N)), tiles = (B * tokens + tpb - 1) / tpb;
  const bool four = tiles * pg.hkv >= 4 * (int64_t)device_cu_count();
  const int64_t chunks = four ? (pg.hkv + 3) / 4 : pg.hkv;
  if (!grid_fits(tiles * chunks * 2, kPgThreads)) return fail(TT_ERR_ARG, std::string(fn) + ": too many rows");
#define TT_PG_APPEND_N(HC)                                                                                           \
  hipLaunchKernelGGL((kv_append_kernel<T, D, HC>), dim3((unsigned)(tiles * chunks * 2)), dim3(kPgThreads), 0, st, in, \
                     rp, pg, (T*)kp, (T*)vp, (uint32_t)(B * tokens), (uint32_t)tokens, (uint32_t)chunks)
#define TT_PG_APPEND     \
  if (four)              \
    TT_PG_APPEND_N(4);   \
  else                   \
    TT_PG_APPEND_N(1)
  TT_PG_DIM(TT_PG_APPEND)
#undef TT_PG_APPEND
#undef TT_PG_APPEND_N
  TT_LAUNCHED(fn, st);
  return ok();
}

template <typename T, int D, int NEW>
void append_e4m3_new(const PgNew<T>& in, const Rope& rp, const Pages& pg, uint8_t* kp, uint8_t* vp, uint8_t* ks,
                      uint8_t* vs, int64_t pages, int64_t tokens, int64_t count, int64_t heads, hipStream_t st) {
  const int64_t groups = (pg.hkv + heads - 1) / heads;
  hipLaunchKernelGGL((kv_append_e4m3_kernel<T, D, NEW>), dim3((unsigned)(pages * groups), 2),
                     dim3(PgTile<T, D, NEW>::THREADS), 0, st, in, rp, pg, kp, vp, ks, vs, (uint32_t)tokens,
                     (uint32_t)count, (uint32_t)groups, (uint32_t)heads);
}

template <typename T>
int append_e4m3_launch(const char* fn, const PgNew<T>& in, const Rope& rp, const Pages& pg, uint8_t* kp, uint8_t* vp,
                       uint8_t* ks, uint8_t* vs, int64_t B, int64_t tokens, int64_t d, hipStream_t st) {
  const int64_t page = int64_t(1) << pg.lp, count = (tokens + page - 2) / page + 1, pages = B * count;
  if (pages * pg.hkv > int64_t(0x7fffffff) || !grid_fits(pages * pg.hkv, 512))
    return fail(TT_ERR_ARG, std::string(fn) + ": too many pages of new tokens");
  int64_t heads = std::min<int64_t>(pg.hkv, kPgHeads);
  while (heads > 1 && 2 * pages * ((pg.hkv + heads - 1) / heads) < 4 * (int64_t)device_cu_count()) heads = (heads + 1) / 2;
  const int64_t most = std::min(page, tokens);  // new rows of a page
#define TT_PG_E4                                                                                          \
  if (most <= 16)                                                                                         \
    append_e4m3_new<T, D, 16>(in, rp, pg, kp, vp, ks, vs, pages, tokens, count, heads, st);               \
  else if (most <= 32)                                                                                    \
    append_e4m3_new<T, D, 32>(in, rp, pg, kp, vp, ks, vs, pages, tokens, count, heads, st);               \
  else if (most <= 64)                                                                                    \
    append_e4m3_new<T, D, 64>(in, rp, pg, kp, vp, ks, vs, pages, tokens, count, heads, st);               \
  else                                                                                                    \
    append_e4m3_new<T, D, 128>(in, rp, pg, kp, vp, ks, vs, pages, tokens, count, heads, st)
  TT_PG_DIM(TT_PG_E4)
#undef TT_PG_E4
  TT_LAUNCHED(fn, st);
  return ok();
}

template <typename T, typename C>
int gather_launch(const char* fn, const void* kp, const void* vp, const uint8_t* ks, const uint8_t* vs,
                  const Pages& pg, void* k, void* v, int64_t B, int64_t L, int64_t d, hipStream_t st) {
  const int64_t rows = kPgUnroll * kPgThreads / (d / Chunk<T>::N), tiles = (L + rows - 1) / rows;
  if (!grid_fits(B * pg.hkv * tiles, kPgThreads)) return fail(TT_ERR_ARG, std::string(fn) + ": too many rows");
#define TT_PG_GATHER_N(NT)                                                                                             \
  hipLaunchKernelGGL((kv_gather_kernel<T, C, D, NT>), dim3((unsigned)(B * pg.hkv * tiles), 2), dim3(kPgThreads), 0, st, \
                     (const C*)kp, (const C*)vp, ks, vs, pg, (T*)k, (T*)v, (uint32_t)L, (uint32_t)tiles)
#define TT_PG_GATHER                                                  \
  if (2 * B * pg.hkv * L * d * (int64_t)sizeof(T) > kPgNtBytes)       \
    TT_PG_GATHER_N(true);                                             \
  else                                                                \
    TT_PG_GATHER_N(false)
  TT_PG_DIM(TT_PG_GATHER)
#undef TT_PG_GATHER
#undef TT_PG_GATHER_N
  TT_LAUNCHED(fn, st);
  return ok();
}

}  // namespace
}  // namespace tt

using namespace tt;

extern "C" int tt_kv_append_paged(int dtype, int cache, const void* k, const void* v, int64_t ldk, int64_t ldv,
                                  const float* k_weight, float eps, const float* inv_freq, int64_t rot,
                                  int interleaved, const int* positions, void* k_pages, void* v_pages,
                                  uint8_t* k_scales, uint8_t* v_scales, const int* table, const int* lengths,
                                  int64_t B, int64_t Hkv, int64_t T, int64_t d, int64_t npages, int64_t page,
                                  int64_t width, void* stream) {
  const char* fn = "tt_kv_append_paged";
  const std::string f(fn);
  int lp = 0, rc = check_paged(fn, dtype, cache, B, Hkv, T, d, npages, page, width, &lp);
  if (rc) return rc;
  if (inv_freq && (rot < 0 || rot > d || rot % 16 != 0))
    return fail(TT_ERR_ARG, f + ": rot must be a multiple of 16 of at most d");
  if (interleaved != 0 && interleaved != 1) return fail(TT_ERR_ARG, f + ": interleaved must be 0 or 1");
  if (!(eps >= 0.f)) return fail(TT_ERR_ARG, f + ": eps must not be negative");
  if (B * T > 0x7fffffff - 256) return fail(TT_ERR_ARG, f + ": too many tokens");
  const int64_t e = dtype == TT_F32 ? 4 : 2;
  for (const int64_t ld : {ldk, ldv})
    if (ld != 0 && (ld < Hkv * d || ld > (int64_t(1) << 31) || ld * e % 16 != 0))
      return fail(TT_ERR_ARG, f + ": a leading dimension must hold the heads, in steps of 16 bytes");
  if (B == 0 || Hkv == 0 || T == 0 || width == 0 || npages == 0) return ok();
  if (!k || !v) return fail(TT_ERR_ARG, f + ": null pointer");
  if ((rc = check_pools(fn, cache, k_pages, v_pages, k_scales, v_scales, table, lengths))) return rc;
  if (((uintptr_t)k | (uintptr_t)v) & 15) return fail(TT_ERR_ARG, f + ": k and v must be 16-byte aligned");
  auto rows = [&](int64_t ld) { return (size_t)(ld ? (B * T - 1) * ld + Hkv * d : B * T * Hkv * d) * e; };
  const size_t pool = (size_t)(npages * Hkv * page * d) * cache_item(cache);
  const size_t sb = cache == TT_E4M3 ? (size_t)(npages * Hkv) : 0;
  if ((rc = check_no_overlap(fn,
                             {{k, rows(ldk), "k"},
                              {v, rows(ldv), "v"},
                              {k_weight, (size_t)d * sizeof(float), "k_weight"},
                              {inv_freq, (size_t)(inv_freq ? rot / 2 : 0) * sizeof(float), "inv_freq"},
                              {positions, (size_t)(B * T) * sizeof(int), "positions"},
                              {table, (size_t)(B * width) * sizeof(int), "table"},
                              {lengths, (size_t)B * sizeof(int), "lengths"}},
                             {{k_pages, pool, "k_pages"},
                              {v_pages, pool, "v_pages"},
                              {k_scales, sb, "k_scales"},
                              {v_scales, sb, "v_scales"}})))
    return rc;
  if ((rc = ensure_init())) return rc;
  hipStream_t st = stream_or_default(stream);
  const Pages pg{table, lengths, npages, width, (uint32_t)Hkv, lp};
  const Rope rp{inv_freq, positions, nullptr, (int)rot, interleaved, eps};
  if (dtype == TT_F32) {
    const PgNew<float> in{(const float*)k, (const float*)v, ldk, ldv, k_weight};
    return cache == TT_E4M3 ? append_e4m3_launch<float>(fn, in, rp, pg, (uint8_t*)k_pages, (uint8_t*)v_pages,
                                                        k_scales, v_scales, B, T, d, st)
                            : append_launch<float>(fn, in, rp, pg, k_pages, v_pages, B, T, d, st);
  }
  const PgNew<u16> in{(const u16*)k, (const u16*)v, ldk, ldv, k_weight};
  return cache == TT_E4M3 ? append_e4m3_launch<u16>(fn, in, rp, pg, (uint8_t*)k_pages, (uint8_t*)v_pages, k_scales,
                                                    v_scales, B, T, d, st)
                          : append_launch<u16>(fn, in, rp, pg, k_pages, v_pages, B, T, d, st);
}

extern "C" int tt_kv_gather_paged(int dtype, int cache, const void* k_pages, const void* v_pages,
                                  const uint8_t* k_scales, const uint8_t* v_scales, const int* table,
                                  const int* lengths, void* k, void* v, int64_t B, int64_t Hkv, int64_t L, int64_t d,
                                  int64_t npages, int64_t page, int64_t width, void* stream) {
  const char* fn = "tt_kv_gather_paged";
  const std::string f(fn);
  int lp = 0, rc = check_paged(fn, dtype, cache, B, Hkv, L, d, npages, page, width, &lp);
  if (rc) return rc;
  if (B == 0 || Hkv == 0 || L == 0 || width == 0 || npages == 0) return ok();
  if (!k || !v) return fail(TT_ERR_ARG, f + ": null pointer");
  if ((rc = check_pools(fn, cache, k_pages, v_pages, k_scales, v_scales, table, lengths))) return rc;
  if (((uintptr_t)k | (uintptr_t)v) & 15) return fail(TT_ERR_ARG, f + ": k and v must be 16-byte aligned");
  const size_t out = (size_t)(B * Hkv * L * d) * (dtype == TT_F32 ? 4 : 2);
  const size_t pool = (size_t)(npages * Hkv * page * d) * cache_item(cache);
  const size_t sb = cache == TT_E4M3 ? (size_t)(npages * Hkv) : 0;
  if ((rc = check_no_overlap(fn,
                             {{k_pages, pool, "k_pages"},
                              {v_pages, pool, "v_pages"},
                              {k_scales, sb, "k_scales"},
                              {v_scales, sb, "v_scales"},
                              {table, (size_t)(B * width) * sizeof(int), "table"},
                              {lengths, (size_t)B * sizeof(int), "lengths"}},
                             {{k, out, "k"}, {v, out, "v"}})))
    return rc;
  if ((rc = ensure_init())) return rc;
  hipStream_t st = stream_or_default(stream);
  const Pages pg{table, lengths, npages, width, (uint32_t)Hkv, lp};
  if (cache == TT_E4M3)
    return dtype == TT_F32
               ? gather_launch<float, uint8_t>(fn, k_pages, v_pages, k_scales, v_scales, pg, k, v, B, L, d, st)
               : gather_launch<u16, uint8_t>(fn, k_pages, v_pages, k_scales, v_scales, pg, k, v, B, L, d, st);
  return dtype == TT_F32
             ? gather_launch<float, float>(fn, k_pages, v_pages, k_scales, v_scales, pg, k, v, B, L, d, st)
             : gather_launch<u16, u16>(fn, k_pages, v_pages, k_scales, v_scales, pg, k, v, B, L, d, st);
}
