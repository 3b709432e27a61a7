// Products of matrices held in the microscaled 4-bit format (mxfp4.h), and the
// fully connected layer with such weights.
//
//   C[m][n] = alpha sum_k A[m][k] B[n][k] + beta C[m][n] + bias[n]
//
// A [M][K] and B [N][K] are both quantised along k, so a block of 32 k values
// of either has one scale and v_mfma_scale_f32_*_f8f6f4 multiplies them as they
// are stored: codes in a lane's four registers, the scale byte beside them,
// fp32 sums.  The products of two elements are multiples of 1/4 and the scales
// powers of two, so only the sums round.
#include <hip/hip_runtime.h>

#include <optional>
#include <string>

#include "attn_tiles.h"
#include "mxfp4.h"
#include "tt_internal.h"

namespace tt {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kFp4 = 4;  // the instruction's format code of e2m1
__device__ __forceinline__ i32x8 fp4_operand(const uint4& c) {
  return i32x8{(int)c.x, (int)c.y, (int)c.z, (int)c.w, 0, 0, 0, 0};
}
// 16 x 16 x 128: lane l holds row l % 16, k block l / 16 of both operands, and
// its scale in byte 0; result register i is C[4 (l / 16) + i][l % 16].
__device__ __forceinline__ f32x4 mfma_fp4_16(const uint4& a, const uint4& b, const f32x4& c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fp4_operand(a), fp4_operand(b), c, kFp4, kFp4, 0, (int)sa, 0,
                                                          (int)sb);
}

// alpha acc + bias + beta C and the store, for element (row, col) inside C.
template <typename O>
struct MxEpilogue {
  O* C;
  const O* bias;  // null: none
  int64_t bias_step;
  float alpha, beta;
  int64_t N;
  __device__ __forceinline__ static float get(const float* p) { return *p; }
  __device__ __forceinline__ static float get(const u16* p) { return bf16_to_f32(*p); }
  // four sums as they are stored
  __device__ __forceinline__ static void round4(float (&o)[4], const float (&v)[4]) { __builtin_memcpy(o, v, 16); }
  __device__ __forceinline__ static void round4(u16 (&o)[4], const float (&v)[4]) {
    const uint32_t x[2] = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    __builtin_memcpy(o, x, 8);
  }
  // bias of columns [col, col + 4), 0 past the last one
  __device__ __forceinline__ void load_bias(int64_t col, float (&b)[4]) const {
    O x[4] = {};
    if (bias && bias_step == 1 && col + 4 <= N) {
      __builtin_memcpy(x, bias + col, sizeof(x));
    } else if (bias) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < N) x[e] = bias[(col + e) * bias_step];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = get(&x[e]);
  }
  // C[row][col, col + 4), 0 past the last column
  __device__ __forceinline__ void load_four(int64_t row, int64_t col, float (&v)[4]) const {
    const O* c = C + row * N + col;
    O x[4] = {};
    if (col + 4 <= N) {
      __builtin_memcpy(x, c, sizeof(x));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < N) x[e] = c[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = get(&x[e]);
  }
  // 16 bytes of values to columns from col on of a row inside C.
  __device__ __forceinline__ void store16(int64_t row, int64_t col, const uint4& x) const {
    constexpr int E = 16 / (int)sizeof(O);
    O* c = C + row * N + col;
    if (col + E <= N) {
      __builtin_memcpy(c, &x, 16);
    } else {
      O o[E];
      __builtin_memcpy(o, &x, 16);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (col + e < N) c[e] = o[e];
    }
  }
  // The sums of columns [col, col + 4) of a row inside C, stored at once where all are.
  __device__ __forceinline__ void store_four(int64_t row, int64_t col, const f32x4& acc) const {
    O* c = C + row * N + col;
    float b[4], old[4] = {0.f, 0.f, 0.f, 0.f}, v[4];
    load_bias(col, b);
    if (beta != 0.f) load_four(row, col, old);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = alpha * acc[e] + b[e] + (beta != 0.f ? beta * old[e] : 0.f);
    O o[4];
    round4(o, v);
    if (col + 4 <= N) {
      __builtin_memcpy(c, o, sizeof(o));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < N) c[e] = o[e];
    }
  }
};

// Blocks: a workgroup makes 16 MT rows by 16 NT columns of C, its eight waves
// taking an eighth of the k steps of 128 each and meeting in LDS: for products
// of few tiles, whose time is the serial chain of one workgroup.  Operands go
// from global memory to the matrix unit's registers directly, four steps in
// flight a wave (their scales as one 16-byte load a row), with no barrier before
// the end.  QA: A is not quantised yet (X, rows of K values), and each wave
// quantises the 16 rows' k values that it multiplies: one launch for a layer of
// few or short rows.
constexpr int kBlockWaves = 8;
constexpr int kStepK = 128, kStepBytes = kStepK / 2;  // values of a k step, and bytes of their codes

// The scales of k steps [st, st + U) of a row, as this lane's half-filled words:
// block 4 u + g in byte g of w[u] at least, 0 past the row's nb blocks.
template <int U>
__device__ __forceinline__ void load_step_scales(uint32_t (&w)[U], const uint8_t* row, int st, int nb, int g) {
  if (4 * (st + U) <= nb) {
    __builtin_memcpy(w, row + 4 * st, 4 * U);
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = 4 * (st + u);
      w[u] = 0;
      if (at + 4 <= nb)
        __builtin_memcpy(&w[u], row + at, 4);
      else if (at + g < nb)
        w[u] = (uint32_t)row[at + g] << (8 * g);
    }
  }
}

template <typename O, int MT, int NT, bool QA>
__global__ __launch_bounds__(64 * kBlockWaves, QA ? 2 : 4) void k_mxfp4_block(
    const uint4* __restrict__ A, const uint8_t* __restrict__ As, const O* __restrict__ X, const uint4* __restrict__ B,
    const uint8_t* __restrict__ Bs, int64_t M, int64_t N, int64_t K, int nb, uint32_t ntiles, MxEpilogue<O> ep) {
  static_assert(!QA || MT == 1, "16 rows quantised in place");
  constexpr int TILES = MT * NT, HALF = kBlockWaves / 2, UN = QA ? MxWord<O>::N / 2 : 4;
  constexpr int QROW = UN * kStepBytes + 16, QSCALES = 20;  // a row's codes and scales of UN steps, spread over the banks
  __shared__ __align__(16) uint8_t s_q[QA ? kBlockWaves : 1][16][QA ? QROW : 16], s_qs[QA ? kBlockWaves : 1][16][QSCALES];
  __shared__ __align__(16) f32x4 red[HALF][TILES][64];
  const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = l & 15, g = l >> 4;
  const int64_t n0 = (int64_t)(blockIdx.x % ntiles) * (16 * NT), m0 = (int64_t)(blockIdx.x / ntiles) * (16 * MT);
  int64_t brow[NT], arow[MT];  // rows past the end repeat the last one and are not stored
#pragma unroll
  for (int i = 0; i < NT; ++i) brow[i] = min(n0 + 16 * i + r, N - 1) * nb;
#pragma unroll
  for (int j = 0; j < MT; ++j) arow[j] = min(m0 + 16 * j + r, M - 1) * nb;
  const int rows = (int)min((int64_t)16, M - m0);  // of this workgroup, where it quantises them
  f32x4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int steps = (nb + 3) / 4, share = (steps + kBlockWaves - 1) / kBlockWaves, end = min((w + 1) * share, steps);
  for (int st = w * share; st < end; st += UN) {
    uint4 b[UN][NT], a[UN][MT];
    uint32_t sb[NT][UN], sa[MT][UN];
#pragma unroll
    for (int i = 0; i < NT; ++i) load_step_scales<UN>(sb[i], Bs + brow[i], st, nb, g);
    if constexpr (!QA) {
#pragma unroll
      for (int j = 0; j < MT; ++j) load_step_scales<UN>(sa[j], As + arow[j], st, nb, g);
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      if (u > 0 && st + u >= end) break;
      // blocks past the row's end: its last one, made zero below
      const int at = min(4 * (st + u) + g, nb - 1);
#pragma unroll
      for (int i = 0; i < NT; ++i) b[u][i] = B[brow[i] + at];
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        if constexpr (!QA) a[u][j] = A[arow[j] + at];
      }
    }
    if constexpr (QA) {
      // A lane takes a word of each row, as they lie in memory (or of every second
      // or fourth, where the wave has half or a quarter of UN steps); the operands
      // come back from the wave's own LDS.  Rows past M hold anything: each stays
      // in its column of the tile, which is not stored.
      const int left = end - st, sh = left == 1 ? (UN == 4 ? 2 : 1) : (2 * left <= UN ? 1 : 0);
      const int word = l & (63 >> sh), first = l >> (6 - sh);
      MxWord<O> v[16] = {};
      const int64_t k0 = (int64_t)st * kStepK + word * MxWord<O>::N;
      const int n = (int)min((int64_t)MxWord<O>::N, min(K, (int64_t)end * kStepK) - k0);  // at most 0: no value
      const O* p = X + (m0 + first) * K + k0;
      const int own = rows - first, each = 1 << sh;  // the lane's rows: first + i each
      if (n == MxWord<O>::N) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (i * each < own) v[i].load(p + (i * each) * K);
      } else if (n > 0) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (i * each < own) v[i].load_part(p + (i * each) * K, n);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (i * each < own) {
          uint32_t sc;
          const typename MxWord<O>::Codes c = mx_quantize_word<O>(v[i], &sc);
          const int m = first + i * each;
          __builtin_memcpy(&s_q[w][m][word * sizeof(c)], &c, sizeof(c));
          if (word % (kMxBlock / MxWord<O>::N) == 0) s_qs[w][m][word / (kMxBlock / MxWord<O>::N)] = (uint8_t)sc;
        }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        __builtin_memcpy(&a[u][0], __builtin_assume_aligned(&s_q[w][r][(4 * u + g) * kMxBlockBytes], 16), 16);
        sa[0][u] = s_qs[w][r][4 * u + g];
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      if (u > 0 && st + u >= end) break;
      const bool in = 4 * (st + u) + g < nb;
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        if constexpr (!QA) sa[j][u] >>= 8 * g;
        if (!in) {
          a[u][j] = uint4{0, 0, 0, 0};
          sa[j][u] = 0u;
        }
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const uint32_t sbi = in ? sb[i][u] >> (8 * g) : 0u;
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = mfma_fp4_16(b[u][i], a[u][j], acc[i][j], sbi, sa[j][u]);
      }
    }
  }
  // The upper half of the waves hands its sums to the lower half, whose sums
  // then meet in a fixed order.
  if (w >= HALF) {
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) red[w - HALF][i * MT + j][l] = acc[i][j];
  }
  __syncthreads();
  if (w < HALF) {
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) red[w][i * MT + j][l] += acc[i][j];
  }
  __syncthreads();
  for (int t = w; t < TILES; t += kBlockWaves) {
    f32x4 s = red[0][t][l];
#pragma unroll
    for (int q = 1; q < HALF; ++q) s += red[q][t][l];
    const int64_t row = m0 + 16 * (t % MT) + r, col = n0 + 16 * (t / MT) + 4 * g;
    if (row < M) ep.store_four(row, col, s);
  }
}

template <typename O, int MT, int NT, bool QA>
int block_launch(const char* fn, const uint8_t* A, const uint8_t* As, const O* X, const uint8_t* B, const uint8_t* Bs,
                 int64_t M, int64_t N, int64_t K, const MxEpilogue<O>& ep, hipStream_t s) {
  const int64_t nt = (N + 16 * NT - 1) / (16 * NT), tiles = nt * ((M + 16 * MT - 1) / (16 * MT));
  if (!grid_fits(tiles, 64 * kBlockWaves)) return fail(TT_ERR_ARG, std::string(fn) + ": m and n too large");
  hipLaunchKernelGGL((k_mxfp4_block<O, MT, NT, QA>), dim3((unsigned)tiles), dim3(64 * kBlockWaves), 0, s,
                     (const uint4*)A, As, X, (const uint4*)B, Bs, M, N, K, (int)mx_blocks(K), (uint32_t)nt, ep);
  TT_LAUNCHED(fn, s);
  return ok();
}

// p, which every lane holds alike, in scalar registers.
__device__ __forceinline__ const uint8_t* uniform_ptr(const uint8_t* p) {
  const uint64_t x = (uint64_t)(uintptr_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x), hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
  return (const uint8_t*)(uintptr_t)(((uint64_t)hi << 32) | lo);
}

// Tiles: BM x BN of C a workgroup of WM x WN waves, k in stages of 128 (4
// blocks, 64 bytes of codes a row).  A stage's codes of both operands come
// straight into LDS (global_load_lds, 16 bytes a lane) three stages ahead
// through a ring of four; chunk c of row r lies at chunk c ^ (r / 4 % 4), so that
// the 32 rows of which an operand read takes one chunk spread over all banks.
// The scales of four stages (16 bytes a row) come the same way, at any
// alignment: as the two aligned 16-byte words that hold them (a load through
// registers would wait for every load of the ring, a third more time at 8192 x
// 8192 x 8224), which the wave that loaded them then lays out by stage.  A wave
// reads the operands of a k step of 64 while it multiplies the one before, also
// across the barrier of the next stage.  Rows past M or N repeat the last one and
// are not stored.  The matrix unit takes B's rows first, so a lane ends with runs
// of four consecutive columns of one row of C.
// Measured, bf16: 8192 x 8192 x 8192 287 to 300 us, 3.7 to 3.8 PFLOP/s, 4096 x 4096 x
// 4096 41 us, 3.4 PFLOP/s, 2048 x 4096 x 1000 (128 x 128 tiles) 10.5 us, 1.6 PFLOP/s.
// Of constant codes, which the board's power does not hold back, 8192 x 8192 x 8192
// takes 224 us where the bare matrix unit would take 117: of a stage's cycles that
// unit needs 1024, the LDS 768 for operand reads and 256 for its fills, and after
// each barrier all waves read, load and multiply in step, so these add up in part.
constexpr int kStageBlocks = 4, kStageBytes = kStageBlocks * kMxBlockBytes, kStages = 4;

template <typename O, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2) void k_mxfp4_tile(const uint8_t* __restrict__ A,
                                                                const uint8_t* __restrict__ As,
                                                                const uint8_t* __restrict__ B,
                                                                const uint8_t* __restrict__ Bs, int64_t M, int64_t N,
                                                                int nb, int mtiles, int ntiles, MxEpilogue<O> ep) {
  constexpr int NT = 64 * WM * WN, ROWS = BM + BN;
  constexpr int MT = BM / WM / 32, NTL = BN / WN / 32;  // 32-row operand tiles of a wave
  constexpr int LOADS = ROWS * kStageBlocks / NT;       // 16-byte loads a lane and stage
  static_assert(NT == ROWS && LOADS == kStageBlocks && BM % 64 == 0 && BN % 64 == 0, "one row's scales a thread");
  __shared__ __align__(16) uint8_t s_c[kStages][ROWS * kStageBytes];
  __shared__ __align__(16) uint4 s_w[2 * ROWS];        // a batch of scales as loaded
  __shared__ __align__(16) uint32_t s_s[2][4][ROWS];  // and as used: a stage's four bytes of each row

  // Workgroups go round the eight XCDs in turn: each gets one run of tiles, four
  // rows of them high, so that what its workgroups share lies in its own L2.
  const int tiles = mtiles * ntiles, per = (tiles + 7) / 8;
  const int tl = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
  if ((int)(blockIdx.x / 8) >= per || tl >= tiles) return;
  const int band = tl / (4 * ntiles), high = min(4, mtiles - 4 * band), in = tl - band * 4 * ntiles;
  const int64_t m0 = (int64_t)(4 * band + in % high) * BM, n0 = (int64_t)(in / high) * BN;

  const int tid = threadIdx.x, l = tid & 63, r32 = l & 31, g = l >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), wm = w / WN, wn = w % WN;
  const int64_t row_bytes = (int64_t)nb * kMxBlockBytes;
  const int amax = (int)min((int64_t)BM, M - m0) - 1, bmax = (int)min((int64_t)BN, N - n0) - 1;
  const int stages = (nb + kStageBlocks - 1) / kStageBlocks;

  // Load i of wave w fills chunk slots 64 (w LOADS + i) + l: 16 rows of one
  // operand (BM is a multiple of 64, a wave's 64 rows belong to one).  Chunks
  // past the row's end repeat its last one and are not used.
  const bool is_a = w * 64 < BM;
  const uint8_t* src = uniform_ptr(is_a ? A + m0 * row_bytes : B + n0 * row_bytes);
  const int wrow = is_a ? w * 64 : w * 64 - BM, rmax = is_a ? amax : bmax;
  const uint32_t lds0 = lds_addr(&s_c[0][0]) + (uint32_t)w * (64 * kStageBytes);
  uint32_t roff[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) roff[i] = (uint32_t)min(wrow + 16 * i + (l >> 2), rmax) * (uint32_t)row_bytes;
  const int chunk = (l & 3) ^ (l >> 4);
  auto issue = [&](int st, int i) {
    const uint32_t c = 16u * (uint32_t)min(chunk, nb - st * kStageBlocks - 1);
    glds16(src + (int64_t)st * kStageBytes, roff[i] + c,
           lds0 + (uint32_t)(st % kStages) * (ROWS * kStageBytes) + 1024u * (uint32_t)i);
  };
  // Scales: the 16 bytes of blocks [16 bt, 16 bt + 16) of row r lie in words 2 r
  // and 2 r + 1; bytes past the row's end are some other ones, of words that
  // hold a scale of the operand at least.
  const uint8_t* sall = is_a ? As : Bs;
  const uintptr_t send = ((uintptr_t)sall + (uint64_t)(is_a ? M : N) * nb - 1) & ~(uintptr_t)15;  // the last such word
  auto issue_scales = [&](int bt) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint8_t* row = sall + ((is_a ? m0 : n0) + min(wrow + 32 * i + (l >> 1), rmax)) * nb + 16 * bt;
      const uintptr_t at = ((uintptr_t)row & ~(uintptr_t)15) + 16u * (l & 1);
      glds16_at((const void*)(at < send ? at : send), lds_addr(s_w) + (uint32_t)(2 * w + i) * 1024u);
    }
  };
  const uint32_t first = (uint32_t)((uintptr_t)sall + (uint64_t)((is_a ? m0 : n0) + min(wrow + l, rmax)) * nb) & 15u;
  auto lay_out_scales = [&](int bt) {  // this thread's row
    const uint32_t* x = reinterpret_cast<const uint32_t*>(s_w + 2 * (w * 64 + l)) + (first >> 2);
    uint32_t d[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) d[i] = x[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) s_s[bt & 1][i][w * 64 + l] = __builtin_amdgcn_alignbyte(d[i + 1], d[i], first);
  };

  f32x16 acc[NTL][MT];
#pragma unroll
  for (int i = 0; i < NTL; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  // Operand reads: this lane's row of tile 0, chunk 2 s + g.
  const uint32_t coff[2] = {(uint32_t)r32 * kStageBytes + 16u * (uint32_t)(g ^ ((r32 >> 2) & 3)),
                            (uint32_t)r32 * kStageBytes + 16u * (uint32_t)((2 + g) ^ ((r32 >> 2) & 3))};
  const uint8_t* abase = &s_c[0][0] + wm * (MT * 32 * kStageBytes);
  const uint8_t* bbase = &s_c[0][0] + (BM + wn * (NTL * 32)) * kStageBytes;
  uint4 av[2][MT], bv[2][NTL];
  uint32_t sa[2][MT], sb[2][NTL];  // [0]: a stage's scales, this half's bytes at 0 and 2; [1]: the next stage's, as read
  auto read = [&](int st, int s) {
    const uint32_t at = (uint32_t)(st % kStages) * (ROWS * kStageBytes) + coff[s];
#pragma unroll
    for (int i = 0; i < NTL; ++i) bv[s][i] = *reinterpret_cast<const uint4*>(bbase + i * (32 * kStageBytes) + at);
#pragma unroll
    for (int j = 0; j < MT; ++j) av[s][j] = *reinterpret_cast<const uint4*>(abase + j * (32 * kStageBytes) + at);
  };
  auto read_scales = [&](int st) {
    const uint32_t* ss = s_s[(st >> 2) & 1][st & 3];
#pragma unroll
    for (int j = 0; j < MT; ++j) sa[1][j] = ss[(wm * MT + j) * 32 + r32];
#pragma unroll
    for (int i = 0; i < NTL; ++i) sb[1][i] = ss[BM + (wn * NTL + i) * 32 + r32];
  };
  auto multiply = [&](int s) {
#pragma unroll
    for (int i = 0; i < NTL; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const i32x8 x = fp4_operand(bv[s][i]), y = fp4_operand(av[s][j]);
        acc[i][j] = s == 0 ? __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, acc[i][j], kFp4, kFp4, 0,
                                                                             (int)sb[0][i], 0, (int)sa[0][j])
                           : __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, acc[i][j], kFp4, kFp4, 2,
                                                                             (int)sb[0][i], 2, (int)sa[0][j]);
      }
  };
  auto shift_scales = [&]() {
#pragma unroll
    for (int j = 0; j < MT; ++j) sa[0][j] = sa[1][j] >> (8 * g);
#pragma unroll
    for (int i = 0; i < NTL; ++i) sb[0][i] = sb[1][i] >> (8 * g);
  };
  // Stage st has landed for every wave, and nobody reads the stage before any more.
  auto meet = [&](int st) {
    wait_vmem_tiles<LOADS, 2>(min(2, stages - 1 - st));
    __syncthreads();
  };
  auto zero_odd = [&](int s, int left) {  // an odd last block: no partner, whatever lies in its place
    if (2 * s + 1 >= left && g == 1) {
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        av[s][j] = uint4{0, 0, 0, 0};
        sa[0][j] = 0;
      }
#pragma unroll
      for (int i = 0; i < NTL; ++i) sb[0][i] = 0;
    }
  };

  if (stages > 0) {
    issue_scales(0);
    for (int st = 0; st < min(stages, 3); ++st)
#pragma unroll
      for (int i = 0; i < LOADS; ++i) issue(st, i);
    meet(0);
    lay_out_scales(0);
    __syncthreads();
    read(0, 0);
    read_scales(0);
    // Stages that another one follows are whole.
    for (int st = 0; st + 1 < stages; ++st) {
      shift_scales();
      read(st, 1);
      if ((st & 3) == 0 && st + 4 < stages) issue_scales((st + 4) >> 2);  // landed with stage st + 3
      if ((st & 3) == 3) lay_out_scales((st + 1) >> 2);
      if (st + 3 < stages)
#pragma unroll
        for (int i = 0; i < LOADS; ++i) issue(st + 3, i);
      multiply(0);
      meet(st + 1);
      read(st + 1, 0);
      read_scales(st + 1);
      multiply(1);
    }
    const int left = nb - (stages - 1) * kStageBlocks;
    shift_scales();
    zero_odd(0, left);
    multiply(0);
    if (left > 2) {
      read(stages - 1, 1);
      zero_odd(1, left);
      multiply(1);
    }
  }

  const int64_t row0 = m0 + wm * (MT * 32), col0 = n0 + wn * (NTL * 32);
  float alpha = ep.alpha;
  if (ep.beta != 0.f || ep.bias) {
#pragma unroll
    for (int i = 0; i < NTL; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t col = col0 + 32 * i + 8 * q + 4 * g;
        float bias[4], old[4];
        ep.load_bias(col, bias);
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          const int64_t row = row0 + 32 * j + r32;
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] = alpha * acc[i][j][4 * q + e] + bias[e];
          if (ep.beta != 0.f && row < M) {
            ep.load_four(row, col, old);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] += ep.beta * old[e];
          }
        }
      }
    alpha = 1.f;
  }
  // C leaves through LDS, so that a store takes whole runs of the wave's columns
  // (stored as the lanes hold them, 16 bytes a row and half, 8192 x 8192 values took
  // 56 us, now 13).  A lane's four columns lie in one of a row's 16-byte chunks,
  // which the row swizzles over the banks.
  constexpr int ROW = NTL * 32 * (int)sizeof(O), CHUNKS = ROW / 16, UPC = 16 / (4 * (int)sizeof(O));
  constexpr int MINE = (int)sizeof(s_c) / (WM * WN), JP = MINE / (32 * ROW) < MT ? MINE / (32 * ROW) : MT;
  constexpr int RPS = 64 / CHUNKS;  // rows of a store
  static_assert(JP > 0 && MT % JP == 0, "whole tiles a pass");
  auto chunk_at = [](int row, int c) { return row * ROW + 16 * (c ^ (row / UPC % CHUNKS)); };
  uint8_t* mine = &s_c[0][0] + w * MINE;
  const bool whole = m0 + BM <= M && n0 + BN <= N;
  const int c = l % CHUNKS;
  __syncthreads();  // nobody reads the ring any more
#pragma unroll
  for (int j0 = 0; j0 < MT; j0 += JP) {
#pragma unroll
    for (int j = j0; j < j0 + JP; ++j)
#pragma unroll
      for (int i = 0; i < NTL; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = alpha * acc[i][j][4 * q + e];
          O o[4];
          ep.round4(o, v);
          const int unit = 8 * i + 2 * q + g;
          __builtin_memcpy(mine + chunk_at(32 * (j - j0) + r32, unit / UPC) + (unit % UPC) * (int)sizeof(o), o,
                           sizeof(o));
        }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const int64_t first_row = row0 + 32 * j0 + l / CHUNKS, col = col0 + c * (16 / (int)sizeof(O));
    if (whole) {
      O* to = ep.C + first_row * N + col;
#pragma unroll
      for (int t = 0; t < JP * 32 / RPS; ++t) {
        __builtin_memcpy(to, mine + chunk_at(t * RPS + l / CHUNKS, c), 16);
        to += RPS * N;
      }
    } else {
      for (int t = 0; t < JP * 32 / RPS; ++t) {
        uint4 x;
        __builtin_memcpy(&x, mine + chunk_at(t * RPS + l / CHUNKS, c), 16);
        if (first_row + t * RPS < M) ep.store16(first_row + t * RPS, col, x);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

template <typename O, int BM, int BN, int WM, int WN>
int tile_launch(const char* fn, const uint8_t* A, const uint8_t* As, const uint8_t* B, const uint8_t* Bs, int64_t M,
                int64_t N, int64_t K, const MxEpilogue<O>& ep, hipStream_t s) {
  const int64_t mt = (M + BM - 1) / BM, nt = (N + BN - 1) / BN, grid = (mt * nt + 7) / 8 * 8;
  if (!grid_fits(grid, 64 * WM * WN)) return fail(TT_ERR_ARG, std::string(fn) + ": m and n too large");
  hipLaunchKernelGGL((k_mxfp4_tile<O, BM, BN, WM, WN>), dim3((unsigned)grid), dim3(64 * WM * WN), 0, s, A, As, B, Bs, M,
                     N, (int)mx_blocks(K), (int)mt, (int)nt, ep);
  TT_LAUNCHED(fn, s);
  return ok();
}

template <typename O>
int product(const char* fn, const uint8_t* A, const uint8_t* As, const uint8_t* B, const uint8_t* Bs, int64_t M,
            int64_t N, int64_t K, const MxEpilogue<O>& ep, hipStream_t s) {
  auto tiles = [&](int64_t t) { return ((M + t - 1) / t) * ((N + t - 1) / t); };
  // Few tiles: the smallest blocks that are not more than two a CU.  Measured
  // (16 x 16 / 32 x 32 / 128 x 128, us): 1 x 4096 x 4096 3.6 / 5.4 / 14.8 (256
  // blocks), 100 x 1000 x 500 3.5 / 3.6 / 5.5 (441), 64 x 4096 x 4096 11.0 (1024) /
  // 7.2 / 15.5, 128 x 4096 x 4096 19.9 / 11.4 (512) / 15.0, 600 x 1101 x 1000 12.5 /
  // 10.3 (665) / 7.4, 500 x 2000 x 3000 24 / 17.1 (1008) / 12.6.  Up to 16 rows stay
  // with them for their long rows: 1 x 16384 x 16384 24.7 / 36.5 / 50.4, 1 x 128000 x
  // 4096 46.5 / 47.7 / 50.5; from some 50000 columns on the tiles are the faster
  // for several rows, 16 x 128000 x 4096 73 / 64 / 53, 10 x 70000 x 784 16.6 / 19.7 /
  // 11.1.
  if (tiles(16) <= 512 || (M <= 16 && grid_fits(tiles(16), 64 * kBlockWaves)))
    return block_launch<O, 1, 1, false>(fn, A, As, nullptr, B, Bs, M, N, K, ep, s);
  // the tiles keep the offsets of their rows in 32 bits
  const bool wide = mx_blocks(K) * kMxBlockBytes * 256 > 0xffffffffll;
  if (wide || tiles(32) <= 512) return block_launch<O, 2, 2, false>(fn, A, As, nullptr, B, Bs, M, N, K, ep, s);
  // 128 x 128 tiles, two a CU, where one round takes them all, and where a larger
  // one could not be filled on one side.  Measured (128 / 256, us): 1531 x 4099 x
  // 4096 25.3 / 32.6 (396 small tiles), 2048 x 4096 x 1000 10.3 / 13.1 (512), 2600 x
  // 3328 x 2048 20.9 / 19.0 (546), 3500 x 3500 x 2000 29.6 / 25.1 (784), 8192 x 8192 x
  // 8192 394 / 279; 70000 x 10 x 784 13.9 / 25.0, 70000 x 128 x 1024 16.0 / 28.9, 17 x
  // 70000 x 784 11.7 / 18.3, 128 x 131072 x 1024 22.6 / 35.3.
  if (tiles(128) <= 512 || M <= 128 || N <= 128)
    return tile_launch<O, 128, 128, 2, 2>(fn, A, As, B, Bs, M, N, K, ep, s);
  return tile_launch<O, 256, 256, 2, 4>(fn, A, As, B, Bs, M, N, K, ep, s);
}

// Rows of x quantised at a time; the scratch is of one size, so that graphs may keep its address.
constexpr size_t kMxRowsWork = size_t(32) << 20;

template <typename O>
int fc(const char* fn, const O* x, const uint8_t* W, const uint8_t* Ws, const O* bias, int64_t bias_step, int64_t M,
       int64_t N, int64_t K, O* out, hipStream_t s) {
  const MxEpilogue<O> all{out, bias, bias_step, 1.f, 0.f, N};
  const int64_t nb = mx_blocks(K), row_bytes = nb * (kMxBlockBytes + 1);
  const int64_t fit = row_bytes > 0 ? (int64_t)(kMxRowsWork / row_bytes) / 16 * 16 : 0;
  // One launch, in which every workgroup quantises its 16 rows over again, where
  // these are short or few, or two launches.  Measured (one / two, us): 256 x 100 x
  // 784 bf16 4.5 / 6.7, 32 x 4096 x 512 fp32 4.7 / 6.2, 256 x 512 x 2048 bf16 (rows
  // of 4 KiB) 6.6 / 7.6, fp32 8.0 / 7.4, 16 x 16384 x 1024 (1024 blocks) 9.1 / 8.3;
  // 1 x 4096 x 4096 bf16 4.4 / 6.1, fp32 5.4 / 6.1, 4 x 4096 x 4096 bf16 (32 KiB) 4.8 /
  // 6.3, fp32 6.1 / 6.1, 1 x 4096 x 16384 bf16 9.5 / 10.5, fp32 15.0 / 10.3.
  const int64_t row = K * (int64_t)sizeof(O), blocks = ((M + 15) / 16) * ((N + 15) / 16);
  const bool once = blocks <= 512 && (row <= 4096 || M * row <= 32768);
  void* ws = nullptr;
  std::optional<WorkspaceLease> lease;  // held until the last kernel that reads the buffer is queued
  if (once || fit < 16 || !lease.emplace().get_fixed(s, kWsMxfp4Rows, kMxRowsWork, &ws)) {
    // as many rows a launch as its grid takes
    const int64_t most = 0xffffffffu / (64 * kBlockWaves) / ((N + 15) / 16) * 16, step = most > 0 ? most : M;
    for (int64_t r0 = 0; r0 < M; r0 += step) {
      MxEpilogue<O> ep = all;
      ep.C = out + r0 * N;
      const int64_t rows = M - r0 < step ? M - r0 : step;
      const int rc = block_launch<O, 1, 1, true>(fn, nullptr, nullptr, x + r0 * K, W, Ws, rows, N, K, ep, s);
      if (rc) return rc;
    }
    return ok();
  }
  for (int64_t r0 = 0; r0 < M; r0 += fit) {
    const int64_t rows = M - r0 < fit ? M - r0 : fit;
    uint8_t* codes = (uint8_t*)ws;
    uint8_t* scales = codes + (size_t)(rows * nb) * kMxBlockBytes;
    int rc = tt_mxfp4_quantize(sizeof(O) == 4 ? TT_F32 : TT_BF16, 0, x + r0 * K, codes, scales, rows, K, s);
    if (rc) return rc;
    MxEpilogue<O> ep = all;
    ep.C = out + r0 * N;
    if ((rc = product<O>(fn, codes, scales, W, Ws, rows, N, K, ep, s))) return rc;
  }
  return ok();
}

int check_product(const char* fn, int dtype, int64_t m, int64_t n, int64_t k) {
  const std::string f(fn);
  if (dtype != TT_F32 && dtype != TT_BF16) return fail(TT_ERR_ARG, f + ": dtype must be TT_F32 or TT_BF16");
  if (m < 0 || n < 0 || k < 0) return fail(TT_ERR_ARG, f + ": negative size");
  if (m > 0x7fffffff || n > 0x7fffffff || k > 0x7fffffff)
    return fail(TT_ERR_ARG, f + ": dimension above 2^31 - 1");
  return TT_OK;
}

}  // namespace
}  // namespace tt

using namespace tt;

extern "C" int tt_gemm_mxfp4(int dtype, int64_t m, int64_t n, int64_t k, float alpha, const uint8_t* a_codes,
                             const uint8_t* a_scales, const uint8_t* b_codes, const uint8_t* b_scales, float beta,
                             void* C, void* stream) {
  const char* fn = "tt_gemm_mxfp4";
  int rc = check_product(fn, dtype, m, n, k);
  if (rc) return rc;
  if (m == 0 || n == 0) return ok();
  if (!C || (k > 0 && (!a_codes || !a_scales || !b_codes || !b_scales)))
    return fail(TT_ERR_ARG, std::string(fn) + ": null pointer");
  if (k > 0 && (((uintptr_t)a_codes | (uintptr_t)b_codes) & 15))
    return fail(TT_ERR_ARG, std::string(fn) + ": codes must be 16-byte aligned");
  const size_t na = (size_t)(m * mx_blocks(k)), nb = (size_t)(n * mx_blocks(k));
  if ((rc = check_no_overlap(fn, {{a_codes, na * kMxBlockBytes, "a_codes"}, {a_scales, na, "a_scales"},
                                  {b_codes, nb * kMxBlockBytes, "b_codes"}, {b_scales, nb, "b_scales"}},
                             {{C, (size_t)(m * n) * (dtype == TT_F32 ? 4 : 2), "C"}})))
    return rc;
  if ((rc = ensure_init())) return rc;
  hipStream_t s = stream_or_default(stream);
  if (dtype == TT_F32)
    return product<float>(fn, a_codes, a_scales, b_codes, b_scales, m, n, k,
                          MxEpilogue<float>{(float*)C, nullptr, 0, alpha, beta, n}, s);
  return product<u16>(fn, a_codes, a_scales, b_codes, b_scales, m, n, k,
                      MxEpilogue<u16>{(u16*)C, nullptr, 0, alpha, beta, n}, s);
}

extern "C" int tt_fc_forward_mxfp4(int dtype, int64_t batch, int64_t fin, int64_t fout, const void* in,
                                   const uint8_t* w_codes, const uint8_t* w_scales, const void* bias, int bias_scalar,
                                   void* out, void* stream) {
  const char* fn = "tt_fc_forward_mxfp4";
  int rc = check_product(fn, dtype, batch, fout, fin);
  if (rc) return rc;
  if (batch == 0 || fout == 0) return ok();
  if (!bias || !out || (fin > 0 && (!in || !w_codes || !w_scales)))
    return fail(TT_ERR_ARG, std::string(fn) + ": null pointer");
  if (fin > 0 && ((uintptr_t)w_codes & 15)) return fail(TT_ERR_ARG, std::string(fn) + ": codes must be 16-byte aligned");
  const size_t e = dtype == TT_F32 ? 4 : 2, nw = (size_t)(fout * mx_blocks(fin));
  if ((rc = check_no_overlap(fn, {{in, (size_t)(batch * fin) * e, "in"}, {w_codes, nw * kMxBlockBytes, "w_codes"},
                                  {w_scales, nw, "w_scales"}, {bias, (size_t)(bias_scalar ? 1 : fout) * e, "bias"}},
                             {{out, (size_t)(batch * fout) * e, "out"}})))
    return rc;
  if ((rc = ensure_init())) return rc;
  hipStream_t s = stream_or_default(stream);
  const int64_t step = bias_scalar ? 0 : 1;
  if (dtype == TT_F32)
    return fc<float>(fn, (const float*)in, w_codes, w_scales, (const float*)bias, step, batch, fout, fin, (float*)out, s);
  return fc<u16>(fn, (const u16*)in, w_codes, w_scales, (const u16*)bias, step, batch, fout, fin, (u16*)out, s);
}
