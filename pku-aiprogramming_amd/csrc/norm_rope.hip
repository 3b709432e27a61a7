// From a projection's output to the q, k and v that attention takes, and back:
// queries and keys normed over each head and rotated by their positions, in one
// pass that also moves token-major rows to [B][H][T][D] (rope.h has the formulas).
//
// Each value is read and written once with some ten operations, so the bytes bound
// it: 2 e a value forward, 3 e backward.  The angles are not stored: a thread keeps
// one token's N pairs and goes through a run of heads, so that its sines and cosines,
// formed from 64-bit angles, serve them all.
//
// Backward, of y = R (x r w) with r = 1 / sqrt(mean x^2 + eps), n = x r, g = R^T dy:
//   dw = sum over rows of g n,   dx = r (g w - n mean(g w n)).
// r is formed again from x, which is read anyway.  A thread sums its rows' g n in
// registers, a workgroup its threads' in LDS, a second launch the workgroups' in the
// order of their numbers (of a few, the last workgroup to end does), so the result does
// not depend on which ends first.
// Measured (MI355X): 4 x 4096 tokens of 32 / 32 heads of 128 in bf16, one fused projection:
// forward 155 us (805 MB, 5.2 TB/s), back 219 us (1074 MB, 4.9 TB/s); 8 tokens 4 us.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <optional>
#include <string>

#include "attn_tiles.h"
#include "rope.h"
#include "tt_internal.h"

namespace tt {
namespace {

constexpr int kNrThreads = 256;
constexpr int kNrHeads = 4;  // of a workgroup at most

// q, k or v: rows of `heads` heads, token-major with `ld` values a token, or
// head-major [B][heads][T][D] (ld = 0).
template <typename T>
struct NrPart {
  const T* x;
  T* y;
  const float* w;  // null: not normed
  int64_t ld;
  int heads;
};

template <bool NT>
__device__ __forceinline__ void nr_st(void* p, const uint4& x) {
  if constexpr (NT)
    __builtin_nontemporal_store(u32x4{x.x, x.y, x.z, x.w}, reinterpret_cast<u32x4*>(p));
  else
    *reinterpret_cast<uint4*>(p) = x;
}
// A lane's two chunks of a row.
template <typename T, int D, bool NT>
struct NrRow {
  static constexpr int N = Chunk<T>::N;
  uint4 a, b;
  __device__ __forceinline__ void load(const T* row, const Lay<N>& lay) {
    a = NT ? ldg16_stream(row + lay.a) : ldg16(row + lay.a);
    b = NT ? ldg16_stream(row + lay.b) : ldg16(row + lay.b);
  }
  __device__ __forceinline__ void get(float (&f)[2 * N]) const {
    Chunk<T>::get(a, f);
    Chunk<T>::get(b, f + N);
  }
  __device__ __forceinline__ void put(const float (&f)[2 * N]) {
    a = Chunk<T>::put(f);
    b = Chunk<T>::put(f + N);
  }
  __device__ __forceinline__ void store(T* row, const Lay<N>& lay) const {
    nr_st<NT>(row + lay.a, a);
    nr_st<NT>(row + lay.b, b);
  }
};
template <int N>
__device__ __forceinline__ void nr_weight(const float* w, const Lay<N>& lay, float (&f)[2 * N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) {
    f[e] = w ? w[lay.a + e] : 1.f;
    f[N + e] = w ? w[lay.b + e] : 1.f;
  }
}
// Heads [lo, hi), at most HC of them, R rows each: all loaded before the first is
// used, with `between` meanwhile.  A full chunk has a copy without branches, behind
// which the compiler would wait for stores too.
template <int HC, int R, typename Row, typename L, typename M, typename F>
__device__ __forceinline__ void nr_heads(int lo, int hi, L&& load, M&& between, F&& use) {
  Row r[HC][R];
  if (hi - lo == HC) {
#pragma unroll
    for (int u = 0; u < HC; ++u) load(r[u], lo + u);
    between();
#pragma unroll
    for (int u = 0; u < HC; ++u) use(r[u], lo + u);
  } else {
#pragma unroll
    for (int u = 0; u < HC; ++u) load(r[u], min(lo + u, hi - 1));
    between();
#pragma unroll
    for (int u = 0; u < HC; ++u)
      if (lo + u < hi) use(r[u], lo + u);
  }
}

// How a launch is cut: chunks of `count` heads of q's, k's and v's, one a workgroup.
struct NrCut {
  uint32_t chunks[3], all;
  int count;
};
// The part of chunk `c`, and c's place in it.
__device__ __forceinline__ int nr_part(const NrCut& cut, uint32_t* c) {
  int part = 0;
  if (*c >= cut.chunks[0]) {
    *c -= cut.chunks[0];
    part = 1;
    if (*c >= cut.chunks[1]) {
      *c -= cut.chunks[1];
      part = 2;
    }
  }
  return part;
}

// A workgroup: 256 / LPR tokens, a chunk of the heads of q, k or v.
template <typename T, int D, int HC>
__global__ __launch_bounds__(kNrThreads) void qkv_norm_rope_kernel(NrPart<T> q, NrPart<T> k, NrPart<T> v, Rope rp,
                                                                   uint32_t rows, uint32_t tokens, NrCut cut) {
  constexpr int N = Chunk<T>::N, LPR = D / (2 * N), TPB = kNrThreads / LPR;
  using Row = NrRow<T, D, false>;
  const uint32_t tile = blockIdx.x / cut.all;
  uint32_t chunk = blockIdx.x - tile * cut.all;
  const int part = nr_part(cut, &chunk);
  const NrPart<T> p = part == 0 ? q : part == 1 ? k : v;
  const uint32_t n = tile * TPB + threadIdx.x / LPR;
  if (n >= rows) return;  // whole rows of lanes
  const uint32_t b = n / tokens, t = n - b * tokens;
  const int lo = (int)chunk * cut.count, hi = min(lo + cut.count, p.heads);
  const T* x = p.ld ? p.x + (int64_t)n * p.ld : p.x + ((int64_t)b * p.heads * tokens + t) * D;
  T* y = p.y + ((int64_t)b * p.heads * tokens + t) * D;
  const int64_t xs = p.ld ? D : (int64_t)tokens * D, ys = (int64_t)tokens * D;
  const bool rotate = part < 2 && rp.freq;
  const Lay<N> lay(threadIdx.x % LPR, rotate ? rp.rot : 0, rp.inter != 0);
  auto load = [&](Row(&r)[1], int h) { r[0].load(x + h * xs, lay); };
  if (!rotate && !p.w) {  // moved alone
    nr_heads<HC, 1, Row>(lo, hi, load, [] {}, [&](const Row(&r)[1], int h) { r[0].store(y + h * ys, lay); });
    return;
  }
  RopeTurn<N> turn;
  nr_heads<HC, 1, Row>(
      lo, hi, load,
      [&] {
        float c[N], s[N], w[2 * N];
#pragma unroll
        for (int i = 0; i < N; ++i) c[i] = s[i] = 0.f;
        nr_weight<N>(p.w, lay, w);
        if (lay.turns) rope_angles<N>(rp.freq + lay.pair, rope_position(rp, b, t, tokens), c, s);
        turn.set(c, s, w, lay.turns, rp.inter != 0);
      },
      [&](Row(&r)[1], int h) {
        float f[2 * N];
        r[0].get(f);
        turn(f, p.w ? rope_rms<N, LPR>(f, rp.eps) : 1.f, lay.turns, rp.inter != 0);
        r[0].put(f);
        r[0].store(y + h * ys, lay);
      });
}

// A part on its way back: its gradient dy is head-major, dx lies as x does.
template <typename T>
struct NrBack {
  const T* x;
  const T* dy;
  T* dx;
  const float* w;
  int64_t ldx, ld;  // of x and of dx
  int heads;
};

// A workgroup: tiles slot, slot + slots, ... of 256 / LPR tokens, a chunk of the heads
// of q, k or v.  sums: [slots][chunks of q][D] and then [slots][chunks of k][D], or null
// where no weight's gradient is asked for.  count (of q, of k; zero between calls): the
// last workgroup of each adds them up to dwq or dwk.
template <typename T, int D, int HC, bool NT>
__global__ __launch_bounds__(kNrThreads) void qkv_norm_rope_bwd_kernel(NrBack<T> q, NrBack<T> k, NrBack<T> v, Rope rp,
                                                                       uint32_t rows, uint32_t tokens, uint32_t slots,
                                                                       NrCut cut, float* __restrict__ sums,
                                                                       uint32_t* __restrict__ count,
                                                                       float* __restrict__ dwq,
                                                                       float* __restrict__ dwk) {
  constexpr int N = Chunk<T>::N, LPR = D / (2 * N), TPB = kNrThreads / LPR;
  using Row = NrRow<T, D, NT>;
  const uint32_t slot = blockIdx.x / cut.all;
  uint32_t chunk = blockIdx.x - slot * cut.all;
  const int part = nr_part(cut, &chunk);
  const NrBack<T> p = part == 0 ? q : part == 1 ? k : v;
  const uint32_t tiles = (rows + TPB - 1) / TPB;
  const bool rotate = part < 2 && rp.freq;
  const Lay<N> lay(threadIdx.x % LPR, rotate ? rp.rot : 0, rp.inter != 0);
  const int lo = (int)chunk * cut.count, hi = min(lo + cut.count, p.heads);
  float acc[2 * N], w[2 * N];
#pragma unroll
  for (int e = 0; e < 2 * N; ++e) acc[e] = 0.f;
  nr_weight<N>(p.w, lay, w);

  for (uint32_t tile = slot; tile < tiles; tile += slots) {
    const uint32_t n = tile * TPB + threadIdx.x / LPR;
    if (n >= rows) break;  // whole rows of lanes, and the last tile
    const uint32_t b = n / tokens, t = n - b * tokens;
    const int64_t base = ((int64_t)b * p.heads * tokens + t) * D, ys = (int64_t)tokens * D;
    const T* x = p.ldx ? p.x + (int64_t)n * p.ldx : p.x + base;
    T* dx = p.ld ? p.dx + (int64_t)n * p.ld : p.dx + base;
    const T* dy = p.dy + base;
    const int64_t xs = p.ldx ? D : ys, ds = p.ld ? D : ys;
    auto load = [&](Row(&r)[1], int h) { r[0].load(dy + h * ys, lay); };
    if (!rotate && !p.w) {
      nr_heads<HC, 1, Row>(lo, hi, load, [] {}, [&](const Row(&r)[1], int h) { r[0].store(dx + h * ds, lay); });
      continue;
    }
    float c[N], s[N];
    auto angles = [&] {
      if (!lay.turns) return;
      rope_angles<N>(rp.freq + lay.pair, rope_position(rp, b, t, tokens), c, s);
#pragma unroll
      for (int i = 0; i < N; ++i) s[i] = -s[i];
    };
    if (!p.w) {
      nr_heads<HC, 1, Row>(lo, hi, load, angles, [&](Row(&r)[1], int h) {
        float f[2 * N];
        r[0].get(f);
        if (lay.turns) rope_turn<N>(f, c, s, rp.inter != 0);
        r[0].put(f);
        r[0].store(dx + h * ds, lay);
      });
      continue;
    }
    nr_heads<HC, 2, Row>(
        lo, hi,
        [&](Row(&r)[2], int h) {
          r[0].load(dy + h * ys, lay);
          r[1].load(x + h * xs, lay);
        },
        angles,
        [&](Row(&r)[2], int h) {
          float f[2 * N], z[2 * N], m = 0.f;
          r[0].get(f);
          if (lay.turns) rope_turn<N>(f, c, s, rp.inter != 0);
          r[1].get(z);
          const float scale = rope_rms<N, LPR>(z, rp.eps);
#pragma unroll
          for (int e = 0; e < 2 * N; ++e) {
            z[e] *= scale;
            acc[e] += f[e] * z[e];
            f[e] *= w[e];
            m += f[e] * z[e];
          }
          m = row_sum<LPR>(m) * (1.f / D);
#pragma unroll
          for (int e = 0; e < 2 * N; ++e) f[e] = scale * (f[e] - z[e] * m);
          r[0].put(f);
          r[0].store(dx + h * ds, lay);
        });
  }
  if (!sums || part == 2) return;
  __shared__ float s_sum[kNrThreads / 64 * D < kNrThreads ? kNrThreads / D : kNrThreads / 64][D];
#pragma unroll
  for (int e = 0; e < 2 * N; ++e) {
    float x = acc[e];
#pragma unroll
    for (int off = LPR; off < 64; off <<= 1) x += __shfl_xor(x, off, 64);
    if ((threadIdx.x & 63) < LPR) s_sum[threadIdx.x >> 6][(e < N ? lay.a : lay.b - N) + e] = x;
  }
  __syncthreads();
  const uint32_t nq = slots * cut.chunks[0], nk = slots * cut.chunks[1];
  const uint32_t at = part == 0 ? slot * cut.chunks[0] + chunk : nq + slot * cut.chunks[1] + chunk;
  if (threadIdx.x < D) {
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < kNrThreads / 64; ++i) x += s_sum[i][threadIdx.x];
    float* to = sums + (int64_t)at * D + threadIdx.x;
    if (count)  // past the caches that only some compute units share
      __hip_atomic_store(to, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    else
      *to = x;
  }
  if (!count) return;
  // Stores have ended, and all see them, before the workgroup counts itself.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  __shared__ uint32_t s_before;
  const uint32_t n = part == 0 ? nq : nk;
  if (threadIdx.x == 0) s_before = atomicInc(count + part, n - 1);
  __syncthreads();
  float* dw = part == 0 ? dwq : dwk;
  if (s_before != n - 1 || !dw) return;
  constexpr uint32_t G = kNrThreads / D;
  const uint32_t col = threadIdx.x % D, g = threadIdx.x / D;
  const float* from = sums + (part == 0 ? 0 : (int64_t)nq * D) + col;
  float x = 0.f;
  for (uint32_t i0 = g; i0 < n; i0 += 8 * G) {
    float y[8];
#pragma unroll
    for (uint32_t u = 0; u < 8; ++u)
      y[u] = __hip_atomic_load(from + (int64_t)min(i0 + u * G, n - 1) * D, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
    for (uint32_t u = 0; u < 8; ++u) x += i0 + u * G < n ? y[u] : 0.f;
  }
  float* all = &s_sum[0][0];  // [G][D]
  all[g * D + col] = x;
  __syncthreads();
  if (g > 0) return;
#pragma unroll
  for (uint32_t u = 1; u < G; ++u) x += all[u * D + col];
  dw[col] = x;
}

// Column i of sums [nq][D] to dwq, of the [nk][D] behind them to dwk, 16 columns a
// workgroup of 1024 threads.
constexpr int kNrSumThreads = 1024;
template <int D>
__global__ __launch_bounds__(kNrSumThreads) void norm_weight_sum_kernel(const float* __restrict__ sums,
                                                                        float* __restrict__ dwq,
                                                                        float* __restrict__ dwk, int nq, int nk) {
  constexpr int G = kNrSumThreads / 16;
  __shared__ float s_sum[G][17];
  const bool second = blockIdx.x >= D / 16;
  const int col = (blockIdx.x % (D / 16)) * 16 + (threadIdx.x & 15), g = threadIdx.x >> 4, n = second ? nk : nq;
  float* to = second ? dwk : dwq;
  if (!to) return;
  const float* from = sums + (second ? (int64_t)nq * D : 0) + col;
  float x = 0.f;
#pragma unroll 4
  for (int i = g; i < n; i += G) x += from[(int64_t)i * D];
  s_sum[g][threadIdx.x & 15] = x;
  __syncthreads();
  for (int half = G / 2; half > 0; half >>= 1) {
    if (g < half) s_sum[g][threadIdx.x & 15] += s_sum[g + half][threadIdx.x & 15];
    __syncthreads();
  }
  if (g == 0) to[col] = s_sum[0][threadIdx.x];
}

// Workgroups that leave sums behind, and their scratch: of one size, so that graphs may
// keep its address.  4 x 4096 tokens of 96 heads 229 us with 1024, 220 with 2048, 219 with
// 4096, 223 with 8192; 1843 tokens of 160 heads 59, 60, 63, 63.
constexpr int64_t kNrSums = 2048;
constexpr size_t kNrSumBytes = size_t(kNrSums) * 128 * sizeof(float), kNrWork = kNrSumBytes + 2 * sizeof(uint32_t);
// So many values of sums, of q and of k, the last workgroup adds up: 23 x 4 tokens of 8 / 1
// heads of 128 11.9 -> 8.9 us, 2 x 284 of 12 / 3 heads of 64 (6.9 k) 11.9 -> 9.5, in fp32 (13.8
// k) 11.9 -> 10.3.  More have a launch of their own: 2 x 480 of 4 / 4 heads of 128 (15 k) 11.8
// so and 12.2 without, 8 x 512 of 8 / 2 heads of 64 (33 k) 11.8 and 20.
constexpr int64_t kNrFewValues = 12288;
__global__ void nr_zero_kernel(uint32_t* p) { p[threadIdx.x] = 0u; }

// Four heads a workgroup, for the angles that it forms once and the loads that it has
// in flight; two, or one, where more would leave fewer than two workgroups a CU.
// Measured (bf16, 4 x 4096 tokens of 96 heads of 128, us): forward in ones 211, twos 161,
// fours 155, eights 160, and 145 to 193 by workgroups that go through 16 or 24 heads in a
// loop; back in twos 226, threes 225, fours 220.  3 x 1001 tokens of 20 heads of 64 in
// fp32, back: 15.5 in ones, 13.5 in twos, 17.9 in fours.
inline NrCut nr_cut(int64_t tiles, int64_t q, int64_t k, int64_t v) {
  int64_t count = kNrHeads;
  while (count > 1 && tiles * (q + k + v) < 2 * count * (int64_t)device_cu_count()) count /= 2;
  auto cut = [&](int64_t h) { return (uint32_t)((h + count - 1) / count); };
  NrCut c{{cut(q), cut(k), cut(v)}, 0, (int)count};
  c.all = c.chunks[0] + c.chunks[1] + c.chunks[2];
  return c;
}
// The backward passes values that fill more than this by the caches: 4 x 4096 tokens
// of 48 heads, 570 MB, 126 -> 116 us; the forward with its wider spread of writes loses
// by it (155 -> 183 us), as both do where less is moved.
constexpr int64_t kNrNtBytes = int64_t(256) << 20;

struct NrShape {
  int64_t B, H, Hkv, T, d;
};

template <typename T, int D>
int forward_launch(const char* fn, NrPart<T> q, NrPart<T> k, NrPart<T> v, const Rope& rp, const NrShape& n,
                   hipStream_t st) {
  constexpr int TPB = kNrThreads / (D / (2 * Chunk<T>::N));
  const int64_t tiles = (n.B * n.T + TPB - 1) / TPB;
  const NrCut cut = nr_cut(tiles, q.heads, k.heads, v.heads);
  if (!grid_fits(tiles * cut.all, kNrThreads)) return fail(TT_ERR_ARG, std::string(fn) + ": too many rows");
#define TT_NR_FWD(HC)                                                                                                  \
  hipLaunchKernelGGL((qkv_norm_rope_kernel<T, D, HC>), dim3((unsigned)(tiles * cut.all)), dim3(kNrThreads), 0, st, q, \
                     k, v, rp, (uint32_t)(n.B * n.T), (uint32_t)n.T, cut)
  if (cut.count == 1)
    TT_NR_FWD(1);
  else if (cut.count == 2)
    TT_NR_FWD(2);
  else
    TT_NR_FWD(kNrHeads);
#undef TT_NR_FWD
  TT_LAUNCHED(fn, st);
  return ok();
}

template <typename T, int D>
int backward_launch(const char* fn, NrBack<T> q, NrBack<T> k, NrBack<T> v, const Rope& rp, float* dwq, float* dwk,
                    const NrShape& n, hipStream_t st) {
  constexpr int TPB = kNrThreads / (D / (2 * Chunk<T>::N));
  const int64_t tiles = (n.B * n.T + TPB - 1) / TPB, heads = (int64_t)q.heads + k.heads + v.heads;
  float* sums = nullptr;
  uint32_t* count = nullptr;
  std::optional<WorkspaceLease> lease;  // held until both kernels are queued
  int64_t nq = 0, nk = 0;
  if (tiles > 0 && heads > 0) {
    NrCut cut = nr_cut(tiles, q.heads, k.heads, v.heads);
    int64_t slots = tiles;
    if (dwq || dwk) {
      const int64_t each = (int64_t)cut.chunks[0] + cut.chunks[1];
      void* ws = nullptr;
      bool fresh = false;
      if (!lease.emplace().get_fixed(st, kWsNormWeights, kNrWork, &ws, &fresh))
        return fail(TT_ERR_NOMEM, std::string(fn) + ": no scratch for the weights' gradients (under graph capture it "
                                                    "must be there from an earlier call on the stream)");
      sums = (float*)ws;
      count = (uint32_t*)((char*)ws + kNrSumBytes);
      if (fresh) {
        hipLaunchKernelGGL(nr_zero_kernel, dim3(1), dim3(2), 0, st, count);
        if (const int rc = lease->cleared(fn, st, kWsNormWeights)) return rc;
      }
      if (each > 0) slots = std::min(tiles, kNrSums / each);
      nq = slots * cut.chunks[0];
      nk = slots * cut.chunks[1];
      if (std::max(nq, nk) * D > kNrFewValues || (dwq && nq == 0) || (dwk && nk == 0)) count = nullptr;
    }
    if (!grid_fits(slots * cut.all, kNrThreads)) return fail(TT_ERR_ARG, std::string(fn) + ": too many rows");
#define TT_NR_BWD(HC, NT)                                                                                             \
  hipLaunchKernelGGL((qkv_norm_rope_bwd_kernel<T, D, HC, NT>), dim3((unsigned)(slots * cut.all)), dim3(kNrThreads), 0, \
                     st, q, k, v, rp, (uint32_t)(n.B * n.T), (uint32_t)n.T, (uint32_t)slots, cut, sums, count,           \
                     dwq, dwk)
    if (cut.count == 1)
      TT_NR_BWD(1, false);
    else if (cut.count == 2)
      TT_NR_BWD(2, false);
    else if (n.B * n.T * D * (3 * ((int64_t)q.heads + k.heads) + 2 * v.heads) * (int64_t)sizeof(T) > kNrNtBytes)
      TT_NR_BWD(kNrHeads, true);
    else
      TT_NR_BWD(kNrHeads, false);
#undef TT_NR_BWD
    TT_LAUNCHED(fn, st);
  }
  if ((dwq || dwk) && !count) {
    hipLaunchKernelGGL((norm_weight_sum_kernel<D>), dim3(2 * D / 16), dim3(kNrSumThreads), 0, st, sums, dwq, dwk,
                       (int)nq, (int)nk);
    TT_LAUNCHED(fn, st);
  }
  return ok();
}

// A strided or head-major tensor of a call, for the checks.
struct NrArg {
  const void* p;
  int64_t heads, ld;
  const char* name;
};

int check_shape(const std::string& f, int dtype, const NrShape& n, const float* freq, int64_t rot, int inter,
                float eps) {
  if (dtype != TT_F32 && dtype != TT_BF16) return fail(TT_ERR_ARG, f + ": dtype must be TT_F32 or TT_BF16");
  if (n.B < 0 || n.H < 0 || n.Hkv < 0 || n.T < 0) return fail(TT_ERR_ARG, f + ": negative dimension");
  if (n.d != 32 && n.d != 64 && n.d != 128)
    return fail(TT_ERR_UNSUPPORTED, f + ": head dim must be 32, 64 or 128 (got " + std::to_string(n.d) + ")");
  if (n.H > (int64_t(1) << 20) || n.Hkv > (int64_t(1) << 20)) return fail(TT_ERR_ARG, f + ": too many heads");
  if (n.B > 0x7fffffff || n.T > 0x7fffffff || n.B * n.T > 0x7fffffff - 256)
    return fail(TT_ERR_ARG, f + ": too many tokens");
  if (freq && (rot < 0 || rot > n.d || rot % 16 != 0))
    return fail(TT_ERR_ARG, f + ": rot must be a multiple of 16 of at most d");
  if (inter != 0 && inter != 1) return fail(TT_ERR_ARG, f + ": interleaved must be 0 or 1");
  if (!(eps >= 0.f)) return fail(TT_ERR_ARG, f + ": eps must not be negative");
  return TT_OK;
}

int check_arg(const std::string& f, const NrArg& a, const NrShape& n, size_t e) {
  if (!a.p) return TT_OK;
  if ((uintptr_t)a.p & 15) return fail(TT_ERR_ARG, f + ": " + a.name + " must be 16-byte aligned");
  if (a.ld == 0) return TT_OK;
  if (a.ld < a.heads * n.d || a.ld > (int64_t(1) << 31) || a.ld * (int64_t)e % 16 != 0)
    return fail(TT_ERR_ARG, f + ": the leading dimension of " + a.name +
                                " must hold its heads, in steps of 16 bytes");
  return TT_OK;
}

// From its first to behind its last byte.
ArgSpan span_of(const NrArg& a, const NrShape& n, size_t e) {
  const int64_t tokens = n.B * n.T;
  if (!a.p || tokens == 0 || a.heads == 0) return {nullptr, 0, a.name};
  return {a.p, (size_t)(a.ld ? (tokens - 1) * a.ld + a.heads * n.d : tokens * a.heads * n.d) * e, a.name};
}

// Strided tensors may lie between each other's rows: parts of one fused matrix.
bool apart(const NrArg& a, const NrArg& b, const NrShape& n, size_t e) {
  if (!spans_overlap(span_of(a, n, e), span_of(b, n, e))) return true;
  if (a.ld == 0 || a.ld != b.ld) return false;
  const int64_t ld = a.ld * (int64_t)e, wa = a.heads * n.d * (int64_t)e, wb = b.heads * n.d * (int64_t)e;
  int64_t off = (int64_t)((uintptr_t)b.p - (uintptr_t)a.p) % ld;
  if (off < 0) off += ld;
  return off >= wa && off + wb <= ld;
}

int check_apart(const std::string& f, std::initializer_list<NrArg> inputs, std::initializer_list<ArgSpan> others,
                std::initializer_list<NrArg> outputs, std::initializer_list<ArgSpan> sums, const NrShape& n, size_t e) {
  auto clash = [&](const char* a, const char* b) { return fail(TT_ERR_ARG, f + ": " + a + " overlaps " + b); };
  for (auto o = outputs.begin(); o != outputs.end(); ++o) {
    const ArgSpan so = span_of(*o, n, e);
    for (const NrArg& i : inputs)
      if (spans_overlap(so, span_of(i, n, e))) return clash(o->name, i.name);
    for (const ArgSpan& i : others)
      if (spans_overlap(so, i)) return clash(o->name, i.name);
    for (const ArgSpan& i : sums)
      if (spans_overlap(so, i)) return clash(o->name, i.name);
    for (auto p = outputs.begin(); p != o; ++p)
      if (!apart(*o, *p, n, e)) return clash(o->name, p->name);
  }
  for (auto o = sums.begin(); o != sums.end(); ++o) {
    for (const NrArg& i : inputs)
      if (spans_overlap(*o, span_of(i, n, e))) return clash(o->name, i.name);
    for (const ArgSpan& i : others)
      if (spans_overlap(*o, i)) return clash(o->name, i.name);
    for (auto p = sums.begin(); p != o; ++p)
      if (spans_overlap(*o, *p)) return clash(o->name, p->name);
  }
  return TT_OK;
}

#define TT_NR_DIM(T, CALL)                 \
  switch (n.d) {                           \
    case 32: { constexpr int D = 32; return CALL; }   \
    case 64: { constexpr int D = 64; return CALL; }   \
    default: { constexpr int D = 128; return CALL; }  \
  }

template <typename T>
int forward_d(const char* fn, const void* q, const void* k, const void* v, int64_t ldq, int64_t ldk, int64_t ldv,
              const float* wq, const float* wk, const Rope& rp, void* qo, void* ko, void* vo, const NrShape& n,
              hipStream_t st) {
  const int H = q ? (int)n.H : 0, Hk = k ? (int)n.Hkv : 0, Hv = v ? (int)n.Hkv : 0;
  const NrPart<T> pq{(const T*)q, (T*)qo, wq, ldq, H}, pk{(const T*)k, (T*)ko, wk, ldk, Hk},
      pv{(const T*)v, (T*)vo, nullptr, ldv, Hv};
  TT_NR_DIM(T, (forward_launch<T, D>(fn, pq, pk, pv, rp, n, st)))
}

template <typename T>
int backward_d(const char* fn, const void* q, const void* k, int64_t ldq, int64_t ldk, const float* wq,
               const float* wk, const Rope& rp, const void* dqo, const void* dko, const void* dvo, void* dq, void* dk,
               void* dv, int64_t lddq, int64_t lddk, int64_t lddv, float* dwq, float* dwk, const NrShape& n,
               hipStream_t st) {
  const int H = dq ? (int)n.H : 0, Hk = dk ? (int)n.Hkv : 0, Hv = dv ? (int)n.Hkv : 0;
  const NrBack<T> pq{(const T*)q, (const T*)dqo, (T*)dq, wq, ldq, lddq, H},
      pk{(const T*)k, (const T*)dko, (T*)dk, wk, ldk, lddk, Hk},
      pv{nullptr, (const T*)dvo, (T*)dv, nullptr, 0, lddv, Hv};
  TT_NR_DIM(T, (backward_launch<T, D>(fn, pq, pk, pv, rp, dwq, dwk, n, st)))
}

}  // namespace
}  // namespace tt

using namespace tt;

extern "C" int tt_qkv_norm_rope(int dtype, const void* q, const void* k, const void* v, int64_t ldq, int64_t ldk,
                                int64_t ldv, const float* q_weight, const float* k_weight, float eps,
                                const float* inv_freq, int64_t rot, int interleaved, const int* positions,
                                const int* lengths, void* q_out, void* k_out, void* v_out, int64_t B, int64_t H,
                                int64_t Hkv, int64_t T, int64_t d, void* stream) {
  const char* fn = "tt_qkv_norm_rope";
  const std::string f(fn);
  const NrShape n{B, H, Hkv, T, d};
  int rc = check_shape(f, dtype, n, inv_freq, rot, interleaved, eps);
  if (rc) return rc;
  const size_t e = dtype == TT_F32 ? 4 : 2, w = (size_t)d * sizeof(float);
  const NrArg in[3] = {{q, H, ldq, "q"}, {k, Hkv, ldk, "k"}, {v, Hkv, ldv, "v"}};
  const NrArg out[3] = {{q_out, H, 0, "q_out"}, {k_out, Hkv, 0, "k_out"}, {v_out, Hkv, 0, "v_out"}};
  if (B == 0 || T == 0) return ok();
  for (int i = 0; i < 3; ++i) {
    if ((in[i].p == nullptr) != (out[i].p == nullptr))
      return fail(TT_ERR_ARG, f + ": " + in[i].name + " and its output must both be given or both be null");
    if ((rc = check_arg(f, in[i], n, e)) || (rc = check_arg(f, out[i], n, e))) return rc;
  }
  if ((!q || H == 0) && ((!k && !v) || Hkv == 0)) return ok();
  if ((rc = check_apart(f, {in[0], in[1], in[2]},
                        {{q_weight, w, "q_weight"},
                         {k_weight, w, "k_weight"},
                         {inv_freq, (size_t)(inv_freq ? rot / 2 : 0) * sizeof(float), "inv_freq"},
                         {positions, (size_t)(B * T) * sizeof(int), "positions"},
                         {lengths, (size_t)B * sizeof(int), "lengths"}},
                        {out[0], out[1], out[2]}, {}, n, e)))
    return rc;
  if ((rc = ensure_init())) return rc;
  hipStream_t st = stream_or_default(stream);
  const Rope rp{inv_freq, positions, lengths, (int)rot, interleaved, eps};
  return dtype == TT_F32
             ? forward_d<float>(fn, q, k, v, ldq, ldk, ldv, q_weight, k_weight, rp, q_out, k_out, v_out, n, st)
             : forward_d<u16>(fn, q, k, v, ldq, ldk, ldv, q_weight, k_weight, rp, q_out, k_out, v_out, n, st);
}

extern "C" int tt_qkv_norm_rope_backward(int dtype, const void* q, const void* k, int64_t ldq, int64_t ldk,
                                         const float* q_weight, const float* k_weight, float eps,
                                         const float* inv_freq, int64_t rot, int interleaved, const int* positions,
                                         const int* lengths, const void* dq_out, const void* dk_out,
                                         const void* dv_out, void* dq, void* dk, void* dv, int64_t lddq, int64_t lddk,
                                         int64_t lddv, float* dq_weight, float* dk_weight, int64_t B, int64_t H,
                                         int64_t Hkv, int64_t T, int64_t d, void* stream) {
  const char* fn = "tt_qkv_norm_rope_backward";
  const std::string f(fn);
  const NrShape n{B, H, Hkv, T, d};
  int rc = check_shape(f, dtype, n, inv_freq, rot, interleaved, eps);
  if (rc) return rc;
  const size_t e = dtype == TT_F32 ? 4 : 2, w = (size_t)d * sizeof(float);
  const NrArg x[2] = {{q, H, ldq, "q"}, {k, Hkv, ldk, "k"}};
  const NrArg dy[3] = {{dq_out, H, 0, "dq_out"}, {dk_out, Hkv, 0, "dk_out"}, {dv_out, Hkv, 0, "dv_out"}};
  const NrArg dx[3] = {{dq, H, lddq, "dq"}, {dk, Hkv, lddk, "dk"}, {dv, Hkv, lddv, "dv"}};
  const float* weight[2] = {q_weight, k_weight};
  float* dw[2] = {dq_weight, dk_weight};
  const bool some = B > 0 && T > 0;
  for (int i = 0; i < 3; ++i) {
    if (some && (dy[i].p == nullptr) != (dx[i].p == nullptr))
      return fail(TT_ERR_ARG, f + ": " + dx[i].name + " and " + dy[i].name + " must both be given or both be null");
    if ((rc = check_arg(f, dy[i], n, e)) || (rc = check_arg(f, dx[i], n, e))) return rc;
    if (i == 2) continue;
    if (dw[i] && !weight[i])
      return fail(TT_ERR_ARG, f + ": the gradient of a weight that is not given");
    if (some && dw[i] && x[i].heads > 0 && !dx[i].p)
      return fail(TT_ERR_ARG, f + ": a weight's gradient comes with its input's, which is null");
    if (some && weight[i] && dx[i].p && x[i].heads > 0 && !x[i].p)
      return fail(TT_ERR_ARG, f + ": " + x[i].name + " is null, but normed");
    if ((rc = check_arg(f, x[i], n, e))) return rc;
  }
  const bool any = some && ((dq && H > 0) || ((dk || dv) && Hkv > 0));
  if (!any && !dq_weight && !dk_weight) return ok();
  if ((dq_weight || dk_weight) && (dq ? H : 0) + (dk ? Hkv : 0) > kNrSums)
    return fail(TT_ERR_ARG, f + ": too many heads for the weights' gradients");
  if ((rc = check_apart(f, {x[0], x[1], dy[0], dy[1], dy[2]},
                        {{q_weight, w, "q_weight"},
                         {k_weight, w, "k_weight"},
                         {inv_freq, (size_t)(inv_freq ? rot / 2 : 0) * sizeof(float), "inv_freq"},
                         {positions, (size_t)(B * T) * sizeof(int), "positions"},
                         {lengths, (size_t)B * sizeof(int), "lengths"}},
                        {dx[0], dx[1], dx[2]}, {{dq_weight, w, "dq_weight"}, {dk_weight, w, "dk_weight"}}, n, e)))
    return rc;
  if ((rc = ensure_init())) return rc;
  hipStream_t st = stream_or_default(stream);
  const Rope rp{inv_freq, positions, lengths, (int)rot, interleaved, eps};
  return dtype == TT_F32 ? backward_d<float>(fn, q, k, ldq, ldk, q_weight, k_weight, rp, dq_out, dk_out, dv_out, dq,
                                             dk, dv, lddq, lddk, lddv, dq_weight, dk_weight, n, st)
                         : backward_d<u16>(fn, q, k, ldq, ldk, q_weight, k_weight, rp, dq_out, dk_out, dv_out, dq, dk,
                                           dv, lddq, lddk, lddv, dq_weight, dk_weight, n, st);
}
