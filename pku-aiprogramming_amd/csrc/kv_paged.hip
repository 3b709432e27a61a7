// New keys and values into a paged cache, the keys normed and rotated on the way,
// and a cache read back to contiguous rows (paged.h, rope.h).
//
// Both move each value once with little arithmetic, so the bytes bound them.  Into
// 16 or 32 bits, a thread keeps one token's pairs, its angles and its page, and
// goes through the heads, as in the kernel that norms and rotates queries.  Into 8
// bits, a workgroup owns a page of one head of K or V, whose scale it alone
// changes: it forms the new rows once, in registers, for their largest value, and
// stores their codes; where the scale grows it rounds the page's older rows again.
// K is normed and rotated in 64 bits there and cut to 32 with the last bit set
// where anything was cut off, so that each code is the nearest to the exact value
// and not to a neighbour of it.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "attn_tiles.h"
#include "paged.h"
#include "rope.h"
#include "tt_internal.h"

namespace tt {
namespace {

constexpr int kPgThreads = 256;

template <typename T>
struct PgNew {  // new rows of K and V: token-major with ld values a token, or [B][Hkv][T][D] (0)
  const T *k, *v;
  int64_t ldk, ldv;
  const float* weight;  // of K's norm, or null
};

// A workgroup: 256 / LPR tokens, heads [first, first + count) of K's and then V's.
template <typename T, int D>
__global__ __launch_bounds__(kPgThreads) void kv_append_kernel(PgNew<T> in, Rope rp, Pages pg, T* __restrict__ kp,
                                                               T* __restrict__ vp, uint32_t rows, uint32_t tokens,
                                                               uint32_t chunks, int count) {
  constexpr int N = Chunk<T>::N, LPR = D / (2 * N), TPB = kPgThreads / LPR, UN = 2;
  const uint32_t tile = blockIdx.x / chunks;
  const int first = (int)(blockIdx.x - tile * chunks) * count, heads = (int)pg.hkv;
  const uint32_t n = tile * TPB + threadIdx.x / LPR;
  if (n >= rows) return;  // whole rows of lanes
  const uint32_t b = n / tokens, t = n - b * tokens;
  const int64_t pos = (int64_t)pg.lengths[b] - tokens + t;
  if (pos < 0 || (pos >> pg.lp) >= pg.width) return;
  const int64_t page = pg.table[b * pg.width + (pos >> pg.lp)];
  if (page < 0 || page >= pg.pages) return;
  const Lay<N> lay(threadIdx.x % LPR, rp.freq ? rp.rot : 0, rp.inter != 0);
  float c[N], s[N];
#pragma unroll
  for (int i = 0; i < N; ++i) c[i] = s[i] = 0.f;
  if (lay.turns && first < heads)
    rope_angles<N>(rp.freq + lay.pair, rp.positions ? rope_position(rp, b, t, tokens) : pos, c, s);
  RopeTurn<N> turn;
  if (first < heads) {
    float w[2 * N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      w[e] = in.weight ? in.weight[lay.a + e] : 1.f;
      w[N + e] = in.weight ? in.weight[lay.b + e] : 1.f;
    }
    turn.set(c, s, w, lay.turns, rp.inter != 0);
  }
  const int64_t row = ((page * heads) << pg.lp) + (pos & ((1 << pg.lp) - 1));  // of head 0
  for (int side = 0; side < 2; ++side) {
    const int lo = max(first - side * heads, 0), hi = min(first + count - side * heads, heads);
    if (lo >= hi) continue;
    const T* x = side ? in.v : in.k;
    const int64_t ld = side ? in.ldv : in.ldk, xs = ld ? D : (int64_t)tokens * D;
    x = ld ? x + (int64_t)n * ld : x + ((int64_t)b * heads * tokens + t) * D;
    T* y = (side ? vp : kp) + row * D;
    const int64_t ys = (int64_t)D << pg.lp;
    const bool change = !side && (in.weight || rp.freq);
    for (int h = lo; h < hi; h += UN) {
      uint4 r[UN][2];
#pragma unroll
      for (int u = 0; u < UN; ++u)
        if (h + u < hi) {
          r[u][0] = ldg16(x + (h + u) * xs + lay.a);
          r[u][1] = ldg16(x + (h + u) * xs + lay.b);
        }
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        if (h + u >= hi) break;
        T* to = y + (h + u) * ys;
        if (change) {
          float f[2 * N];
          Chunk<T>::get(r[u][0], f);
          Chunk<T>::get(r[u][1], f + N);
          turn(f, in.weight ? rope_rms<N, LPR>(f, rp.eps) : 1.f, lay.turns, rp.inter != 0);
          r[u][0] = Chunk<T>::put(f);
          r[u][1] = Chunk<T>::put(f + N);
        }
        *reinterpret_cast<uint4*>(to + lay.a) = r[u][0];
        *reinterpret_cast<uint4*>(to + lay.b) = r[u][1];
      }
    }
  }
}

// x in fp32, cut off, the last bit set where anything was: on the same side as x
// of every number of fewer bits and of every middle between two of them.
__device__ __forceinline__ float cut_odd(double x) {
  const float f = (float)x;
  uint32_t bits = __float_as_uint(f);
  if ((bits & 0x7f800000u) == 0x7f800000u) {  // NaN and infinities; past the largest fp32: that
    return (__double_as_longlong(x) & 0x7ff0000000000000ll) == 0x7ff0000000000000ll ? f : __uint_as_float(bits - 1);
  }
  bits -= __builtin_fabs((double)f) > __builtin_fabs(x) ? 1u : 0u;
  return __uint_as_float(bits | (((double)__uint_as_float(bits) != x) ? 1u : 0u));
}

// A workgroup: new tokens of one page of one head, of K (blockIdx.y 0) or V (1).
// Workgroup id = (b * count + i) * Hkv + h, i = 0 .. count - 1 the pages from the
// one that the first new token goes to.
template <typename T, int D, int PAGE>
struct PgTile {
  static constexpr int N = Chunk<T>::N, LPR = D / (2 * N), LANES = PAGE * LPR;
  static constexpr int THREADS = LANES < 64 ? 64 : LANES > kPgThreads ? kPgThreads : LANES;
  static constexpr int ITER = (LANES + THREADS - 1) / THREADS, ROWS = THREADS / LPR;  // rows of an iteration
};
template <typename T, int D, int PAGE>
__global__ __launch_bounds__((PgTile<T, D, PAGE>::THREADS)) void kv_append_e4m3_kernel(
    PgNew<T> in, Rope rp, Pages pg, uint8_t* __restrict__ kp, uint8_t* __restrict__ vp, uint8_t* __restrict__ ks,
    uint8_t* __restrict__ vs, uint32_t tokens, uint32_t count) {
  using P = PgTile<T, D, PAGE>;
  constexpr int N = P::N, LPR = P::LPR, ITER = P::ITER, WAVES = P::THREADS / 64;
  __shared__ uint32_t s_top[WAVES];
  const uint32_t h = blockIdx.x % pg.hkv, bi = blockIdx.x / pg.hkv, b = bi / count, i = bi - b * count;
  const bool is_v = blockIdx.y != 0;
  const int64_t length = pg.lengths[b], end = paged_end(pg, length), first = max(length - (int64_t)tokens, (int64_t)0);
  const int64_t j = first / PAGE + i, base = j * PAGE;
  if (base >= end) return;
  const int64_t page = pg.table[b * pg.width + j];
  if (page < 0 || page >= pg.pages) return;
  const int old = (int)max(first - base, (int64_t)0), fill = (int)min(end - base, (int64_t)PAGE);  // rows [old, fill) are new
  if (old >= fill) return;
  uint8_t* scale_at = (is_v ? vs : ks) + page * pg.hkv + h;
  const uint32_t before = old > 0 ? *scale_at : 0u;
  const Lay<N> lay(threadIdx.x % LPR, rp.freq && !is_v ? rp.rot : 0, rp.inter != 0);
  const int row0 = (int)threadIdx.x / LPR;
  const T* x = is_v ? in.v : in.k;
  const int64_t ld = is_v ? in.ldv : in.ldk;
  const bool norm = !is_v && in.weight;

  float f[ITER][2 * N];
  uint32_t top = 0;
#pragma unroll
  for (int it = 0; it < ITER; ++it) {
    const int row = row0 + it * P::ROWS;
    if (row < old || row >= fill) continue;
    const int64_t t = base + row - (length - tokens);
    const T* from = ld ? x + ((int64_t)b * tokens + t) * ld + h * D : x + (((int64_t)b * pg.hkv + h) * tokens + t) * D;
    Chunk<T>::get(ldg16(from + lay.a), f[it]);
    Chunk<T>::get(ldg16(from + lay.b), f[it] + N);
    if (norm || lay.turns) {
      double g[2 * N];
#pragma unroll
      for (int e = 0; e < 2 * N; ++e) g[e] = f[it][e];
      if (norm) {
        float w[2 * N];
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = in.weight[lay.a + e], w[N + e] = in.weight[lay.b + e];
        rope_scale<N>(g, rope_rms<N, LPR>(g, rp.eps), w);
      }
      if (lay.turns) {
        double c[N], s[N];
        rope_angles<N>(rp.freq + lay.pair, rp.positions ? rope_position(rp, b, t, tokens) : base + row, c, s);
        rope_turn<N>(g, c, s, rp.inter != 0);
      }
#pragma unroll
      for (int e = 0; e < 2 * N; ++e) f[it][e] = cut_odd(g[e]);
    }
#pragma unroll
    for (int e = 0; e < 2 * N; ++e) {
      const uint32_t m = __float_as_uint(f[it][e]) & 0x7fffffffu;
      top = max(top, m < 0x7f800000u ? m : 0u);
    }
  }
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, 64));
  if constexpr (WAVES > 1) {
    if ((threadIdx.x & 63) == 0) s_top[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = max(top, s_top[w]);
  }
  uint32_t byte = e4_scale_byte(top);
  if (old > 0) byte = max(byte, before);
  const float inverse = byte > 254u ? 0.f : e4_inverse(byte);
  uint8_t* codes = (is_v ? vp : kp) + (page * pg.hkv + h) * (int64_t)(PAGE * D);
#pragma unroll
  for (int it = 0; it < ITER; ++it) {
    const int row = row0 + it * P::ROWS;
    if (row < old || row >= fill) continue;
    uint8_t* to = codes + row * D;
    if constexpr (N == 8) {
      *reinterpret_cast<uint2*>(to + lay.a) = uint2{e4_codes(f[it], inverse), e4_codes(f[it] + 4, inverse)};
      *reinterpret_cast<uint2*>(to + lay.b) = uint2{e4_codes(f[it] + 8, inverse), e4_codes(f[it] + 12, inverse)};
    } else {
      *reinterpret_cast<uint32_t*>(to + lay.a) = e4_codes(f[it], inverse);
      *reinterpret_cast<uint32_t*>(to + lay.b) = e4_codes(f[it] + 4, inverse);
    }
  }
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

// 16 codes or 16 bytes of values a lane: rows [B][Hkv][L][D] of T from a pool of C.
template <typename T, typename C, int D>
__global__ __launch_bounds__(kPgThreads) void kv_gather_kernel(const C* __restrict__ kp, const C* __restrict__ vp,
                                                               const uint8_t* __restrict__ ks,
                                                               const uint8_t* __restrict__ vs, Pages pg,
                                                               T* __restrict__ k, T* __restrict__ v, uint32_t L,
                                                               uint64_t words) {
  constexpr int N = 16 / sizeof(C), W = D / N;  // values of a word, words of a row
  const C* pool = blockIdx.y ? vp : kp;
  const uint8_t* scales = blockIdx.y ? vs : ks;
  T* out = blockIdx.y ? v : k;
  const uint64_t step = (uint64_t)gridDim.x * kPgThreads;
  for (uint64_t u = (uint64_t)blockIdx.x * kPgThreads + threadIdx.x; u < words; u += step) {
    const uint64_t row = u / W;
    const uint32_t head = (uint32_t)(row / L), j = (uint32_t)(row - (uint64_t)head * L);
    const uint32_t b = head / pg.hkv, h = head - b * pg.hkv, c = (uint32_t)(u % W);
    if ((int64_t)j >= paged_end(pg, pg.lengths[b])) continue;
    const int64_t page = pg.table[b * pg.width + (j >> pg.lp)];
    if (page < 0 || page >= pg.pages) continue;
    const int64_t at = (((page * pg.hkv + h) << pg.lp) + (j & ((1u << pg.lp) - 1))) * D + c * N;
    const uint4 x = ldg16(pool + at);
    T* to = out + row * D + c * N;
    if constexpr (sizeof(C) == 1) {
      const float scale = e4_scale(scales[page * pg.hkv + h]);
      float f[16];
      e4_values(x.x, f);
      e4_values(x.y, f + 4);
      e4_values(x.z, f + 8);
      e4_values(x.w, f + 12);
#pragma unroll
      for (int e = 0; e < 16; ++e) f[e] *= scale;
#pragma unroll
      for (int e = 0; e < 16; e += Chunk<T>::N) *reinterpret_cast<uint4*>(to + e) = Chunk<T>::put(f + e);
    } else {
      *reinterpret_cast<uint4*>(to) = x;
    }
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
  const int64_t tpb = kPgThreads / (d / (2 * Chunk<T>::N)), tiles = (B * tokens + tpb - 1) / tpb, heads = 2 * pg.hkv;
  // as the kernel that rotates queries: some eight workgroups a CU, heads in a row in each
  const int64_t want = std::min(heads, std::max<int64_t>(1, (8 * (int64_t)device_cu_count() + tiles - 1) / tiles));
  const int64_t count = (heads + want - 1) / want, chunks = (heads + count - 1) / count;
  if (!grid_fits(tiles * chunks, kPgThreads)) return fail(TT_ERR_ARG, std::string(fn) + ": too many rows");
#define TT_PG_APPEND                                                                                               \
  hipLaunchKernelGGL((kv_append_kernel<T, D>), dim3((unsigned)(tiles * chunks)), dim3(kPgThreads), 0, st, in, rp,  \
                     pg, (T*)kp, (T*)vp, (uint32_t)(B * tokens), (uint32_t)tokens, (uint32_t)chunks, (int)count)
  TT_PG_DIM(TT_PG_APPEND)
#undef TT_PG_APPEND
  TT_LAUNCHED(fn, st);
  return ok();
}

template <typename T, int D, int PAGE>
void append_e4m3_page(const PgNew<T>& in, const Rope& rp, const Pages& pg, uint8_t* kp, uint8_t* vp, uint8_t* ks,
                      uint8_t* vs, int64_t groups, int64_t tokens, int64_t count, hipStream_t st) {
  hipLaunchKernelGGL((kv_append_e4m3_kernel<T, D, PAGE>), dim3((unsigned)groups, 2),
                     dim3(PgTile<T, D, PAGE>::THREADS), 0, st, in, rp, pg, kp, vp, ks, vs, (uint32_t)tokens,
                     (uint32_t)count);
}

template <typename T>
int append_e4m3_launch(const char* fn, const PgNew<T>& in, const Rope& rp, const Pages& pg, uint8_t* kp, uint8_t* vp,
                       uint8_t* ks, uint8_t* vs, int64_t B, int64_t tokens, int64_t d, hipStream_t st) {
  const int64_t page = int64_t(1) << pg.lp, count = (tokens + page - 2) / page + 1, groups = B * pg.hkv * count;
  if (groups > int64_t(0x7fffffff) || !grid_fits(groups, kPgThreads))
    return fail(TT_ERR_ARG, std::string(fn) + ": too many pages of new tokens");
#define TT_PG_E4                                                                                              \
  switch (pg.lp) {                                                                                            \
    case 4: append_e4m3_page<T, D, 16>(in, rp, pg, kp, vp, ks, vs, groups, tokens, count, st); break;         \
    case 5: append_e4m3_page<T, D, 32>(in, rp, pg, kp, vp, ks, vs, groups, tokens, count, st); break;         \
    case 6: append_e4m3_page<T, D, 64>(in, rp, pg, kp, vp, ks, vs, groups, tokens, count, st); break;         \
    default: append_e4m3_page<T, D, 128>(in, rp, pg, kp, vp, ks, vs, groups, tokens, count, st); break;       \
  }
  TT_PG_DIM(TT_PG_E4)
#undef TT_PG_E4
  TT_LAUNCHED(fn, st);
  return ok();
}

constexpr int64_t kPgMaxGrid = int64_t(1) << 20;

template <typename T, typename C>
int gather_launch(const char* fn, const void* kp, const void* vp, const uint8_t* ks, const uint8_t* vs,
                  const Pages& pg, void* k, void* v, int64_t B, int64_t L, int64_t d, hipStream_t st) {
  const uint64_t words = (uint64_t)(B * pg.hkv * L) * (uint64_t)(d * sizeof(C) / 16);
  const uint64_t want = (words + kPgThreads - 1) / kPgThreads;
  const dim3 grid((unsigned)std::min<uint64_t>(want, (uint64_t)kPgMaxGrid), 2);
#define TT_PG_GATHER                                                                                               \
  hipLaunchKernelGGL((kv_gather_kernel<T, C, D>), grid, dim3(kPgThreads), 0, st, (const C*)kp, (const C*)vp, ks, vs, \
                     pg, (T*)k, (T*)v, (uint32_t)L, words)
  TT_PG_DIM(TT_PG_GATHER)
#undef TT_PG_GATHER
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
