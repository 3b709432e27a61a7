// Rows to the microscaled 4-bit format and back, and new K / V rows into a
// cache held in it (mxfp4.h describes the format).
//
// Each is one pass over the data with next to no arithmetic, so the bytes
// bound it: 2 (bf16) or 4 (fp32) read or written a value, 17/32 for the codes
// and scales.  A lane holds 16 bytes of values and their codes, four or eight
// neighbouring lanes a block, whose largest exponent takes two or three lane
// permutes: every access of a wave is one contiguous run.
#include <hip/hip_runtime.h>

#include <string>

#include "attn_tiles.h"
#include "mxfp4.h"
#include "tt_internal.h"

namespace tt {
namespace {

constexpr int kMxThreads = 256;
constexpr int kMxUnroll = 2;  // words a thread, loaded before the first is used
// Values that fill more than this go by non-temporally: 8192 x 8192 bf16 quantised
// in 28.1 us instead of 33.8 (6.0 TB/s), read back in 24.3 instead of 33.2 (7.0
// TB/s).  Smaller ones the next kernel may still find in a cache; 33 MB take 8.3 us
// either way.
constexpr int64_t kMxNtBytes = int64_t(64) << 20;

// u / n and u % n, in 32 bits where u fits them.
__device__ __forceinline__ void mx_divmod(uint64_t u, uint32_t n, uint64_t* q, uint32_t* r) {
  if ((u >> 32) == 0) {
    *q = (uint32_t)u / n;
    *r = (uint32_t)u - (uint32_t)*q * n;
  } else {
    *q = u / n;
    *r = (uint32_t)(u - *q * n);
  }
}

// Quantises (QUANT) x into codes and scales, or reads them back into x.
// FLAT: cols is a multiple of 32, so rows follow one another without padding
// and a word's number is its place; otherwise rows have nb blocks of their own
// and end inside the last one.
template <typename T, bool QUANT, bool FLAT, bool NT>
__global__ __launch_bounds__(kMxThreads) void k_mxfp4_rows(T* x, typename MxWord<T>::Codes* codes, uint8_t* scales,
                                                           uint64_t words, int64_t rows, int64_t cols, uint32_t nb) {
  constexpr int N = MxWord<T>::N, WPB = kMxBlock / N;  // values of a word, words of a block
  const T* end = x + rows * cols;
  const uint64_t step = (uint64_t)gridDim.x * (kMxThreads * kMxUnroll);
  for (uint64_t base = (uint64_t)blockIdx.x * (kMxThreads * kMxUnroll); base < words; base += step) {
    MxWord<T> v[kMxUnroll];
    T* at[kMxUnroll];
    int n[kMxUnroll];  // values of this word inside its row
    uint32_t c[kMxUnroll], s[kMxUnroll];
#pragma unroll
    for (int i = 0; i < kMxUnroll; ++i) {
      const uint64_t u = base + i * kMxThreads + threadIdx.x;
      n[i] = 0;
      if (u >= words) continue;  // whole blocks: words is a multiple of WPB
      if constexpr (FLAT) {
        at[i] = x + N * u;
        n[i] = N;
      } else {
        uint64_t row;
        uint32_t blk;
        mx_divmod(u / WPB, nb, &row, &blk);
        const int64_t c0 = (int64_t)blk * kMxBlock + N * (int64_t)(u % WPB);
        at[i] = x + (int64_t)row * cols + c0;
        n[i] = (int)max((int64_t)0, min((int64_t)N, cols - c0));
      }
      if constexpr (QUANT) {
        // a word past its row's end is loaded whole where the next row's values
        // follow, which keep() takes out
        if (FLAT || at[i] + N <= end)
          v[i].template load<NT>(at[i]);
        else
          v[i].load_part(at[i], n[i]);
      } else {
        c[i] = codes[u];
        s[i] = scales[u / WPB];
      }
    }
#pragma unroll
    for (int i = 0; i < kMxUnroll; ++i) {
      const uint64_t u = base + i * kMxThreads + threadIdx.x;
      if (u >= words) continue;
      if constexpr (QUANT) {
        if (!FLAT && n[i] < N) v[i].keep(n[i]);
        uint32_t sb;
        codes[u] = mx_quantize_word<T>(v[i], &sb);
        if (u % WPB == 0) scales[u / WPB] = (uint8_t)sb;
      } else {
        v[i].from(c[i], mx_scale(s[i]));
        if (FLAT || n[i] == N)
          v[i].template store<NT>(at[i]);
        else
          v[i].store_part(at[i], n[i]);
      }
    }
  }
}

// The rows of a matrix stored column by column (x [cols][rows], row r of the
// result takes its column r): a layer's weight [fin, fout], laid out once for
// the product.  A lane takes one block of one row, 32 loads that are
// contiguous over the wave; the four waves of a workgroup take neighbouring
// blocks, so that their 16-byte stores fill whole 64-byte runs.  Each load of a
// wave takes 128 bytes of bf16 or 256 of fp32, which bounds it: 8192 x 8192 in 59 us
// (2.9 TB/s) or 83 us (3.7), 4096 x 11008 in 37 or 53, once a weight.
template <typename T>
__global__ __launch_bounds__(kMxThreads) void k_mxfp4_columns(const T* __restrict__ x, uint4* __restrict__ codes,
                                                              uint8_t* __restrict__ scales, int64_t rows, int64_t cols,
                                                              int64_t nb, int64_t row_tiles) {
  const int64_t r = (int64_t)(blockIdx.x % row_tiles) * 64 + (threadIdx.x & 63);
  const int64_t blk = (int64_t)(blockIdx.x / row_tiles) * 4 + (threadIdx.x >> 6);
  if (r >= rows || blk >= nb) return;
  const T* p = x + blk * kMxBlock * rows + r;
  const int n = (int)min((int64_t)kMxBlock, cols - blk * kMxBlock);
  T raw[kMxBlock];
#pragma unroll
  for (int i = 0; i < kMxBlock; ++i) raw[i] = i < n ? p[i * rows] : T(0);
  MxEight<T> v[4];
  uint32_t e = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[j].load(raw + 8 * j);
    e = max(e, v[j].top());
  }
  const uint32_t s = mx_scale_byte(e);
  const float f = mx_scale(s);
  uint4 c{0, 0, 0, 0};
  if (s != 255u) c = uint4{v[0].codes(f), v[1].codes(f), v[2].codes(f), v[3].codes(f)};
  codes[r * nb + blk] = c;
  scales[r * nb + blk] = (uint8_t)s;
}

// New K (blockIdx.y 0) and V (1) rows [B, Hkv, T, D] into the caches [B, Hkv,
// cap, D]: token t of sequence b goes to row lengths[b] - T + t where that
// lies in [0, cap), and nowhere otherwise.  The new values are loaded beside the
// lengths, not behind them: 16 x 8 heads x 4096 tokens of 128 bf16 in 57 us
// instead of 71 (6.0 TB/s).
template <typename T, int D>
__global__ __launch_bounds__(kMxThreads) void k_mxfp4_append(
    const T* __restrict__ k, const T* __restrict__ v, typename MxWord<T>::Codes* __restrict__ kc,
    uint8_t* __restrict__ ks, typename MxWord<T>::Codes* __restrict__ vc, uint8_t* __restrict__ vs,
    const int* __restrict__ lengths, uint64_t words, uint32_t Hkv, uint32_t tokens, int64_t cap) {
  constexpr int N = MxWord<T>::N, WPB = kMxBlock / N, W = D / N;  // words of a block and of a row
  const T* x = blockIdx.y ? v : k;
  typename MxWord<T>::Codes* codes = blockIdx.y ? vc : kc;
  uint8_t* scales = blockIdx.y ? vs : ks;
  constexpr int UN = kMxUnroll;
  const uint64_t step = (uint64_t)gridDim.x * (kMxThreads * UN);
  for (uint64_t base = (uint64_t)blockIdx.x * (kMxThreads * UN); base < words; base += step) {
    MxWord<T> w[UN];
    int64_t pos[UN], to[UN];
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const uint64_t u = base + i * kMxThreads + threadIdx.x;
      pos[i] = -1;
      if (u >= words) continue;
      w[i].load(x + N * u);
      uint64_t head;  // b Hkv + h
      uint32_t t;
      mx_divmod(u / W, tokens, &head, &t);
      pos[i] = (int64_t)lengths[(uint32_t)head / Hkv] - tokens + t;
      to[i] = ((int64_t)head * cap + pos[i]) * W + (int64_t)(u % W);
    }
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      if (pos[i] < 0 || pos[i] >= cap) continue;  // the same for the whole row, so for whole blocks
      uint32_t s;
      codes[to[i]] = mx_quantize_word<T>(w[i], &s);
      if (to[i] % WPB == 0) scales[to[i] / WPB] = (uint8_t)s;
    }
  }
}

constexpr int64_t kMxMaxGrid = int64_t(1) << 20;

template <typename T, bool QUANT>
int rows_launch(const char* fn, T* x, uint8_t* codes, uint8_t* scales, int64_t rows, int64_t cols, hipStream_t s) {
  const int64_t nb = mx_blocks(cols);
  using Codes = typename MxWord<T>::Codes;
  const uint64_t words = (uint64_t)(rows * nb) * (kMxBlock / MxWord<T>::N);
  const uint64_t per = kMxThreads * kMxUnroll;
  const uint64_t want = (words + per - 1) / per;
  const dim3 grid((unsigned)(want < (uint64_t)kMxMaxGrid ? want : (uint64_t)kMxMaxGrid)), block(kMxThreads);
#define TT_MX_ROWS(FLAT, NT)                                                                                      \
  hipLaunchKernelGGL((k_mxfp4_rows<T, QUANT, FLAT, NT>), grid, block, 0, s, x, (Codes*)codes, scales, words, rows, \
                     cols, (uint32_t)nb)
  const bool nt = rows * cols * (int64_t)sizeof(T) > kMxNtBytes;
  if (cols % kMxBlock == 0) {
    if (nt)
      TT_MX_ROWS(true, true);
    else
      TT_MX_ROWS(true, false);
  } else if (nt) {
    TT_MX_ROWS(false, true);
  } else {
    TT_MX_ROWS(false, false);
  }
#undef TT_MX_ROWS
  TT_LAUNCHED(fn, s);
  return ok();
}

template <typename T>
int columns_launch(const char* fn, const T* x, uint8_t* codes, uint8_t* scales, int64_t rows, int64_t cols,
                   hipStream_t s) {
  const int64_t nb = mx_blocks(cols), row_tiles = (rows + 63) / 64;
  hipLaunchKernelGGL(k_mxfp4_columns<T>, dim3((unsigned)(row_tiles * ((nb + 3) / 4))), dim3(kMxThreads), 0, s, x,
                     (uint4*)codes, scales, rows, cols, nb, row_tiles);
  TT_LAUNCHED(fn, s);
  return ok();
}

template <typename T>
int append_launch(const char* fn, const T* k, const T* v, uint8_t* kc, uint8_t* ks, uint8_t* vc, uint8_t* vs,
                  const int* lengths, int64_t B, int64_t Hkv, int64_t tokens, int64_t cap, int64_t d, hipStream_t s) {
  using Codes = typename MxWord<T>::Codes;
  const uint64_t words = (uint64_t)(B * Hkv * tokens) * (d / MxWord<T>::N);
  const uint64_t per = kMxThreads * kMxUnroll;
  const uint64_t want = (words + per - 1) / per;
  const dim3 grid((unsigned)(want < (uint64_t)kMxMaxGrid ? want : (uint64_t)kMxMaxGrid), 2), block(kMxThreads);
#define TT_MX_APPEND(D)                                                                                         \
  hipLaunchKernelGGL((k_mxfp4_append<T, D>), grid, block, 0, s, k, v, (Codes*)kc, ks, (Codes*)vc, vs, lengths, words, \
                     (uint32_t)Hkv, (uint32_t)tokens, cap)
  switch (d) {
    case 32: TT_MX_APPEND(32); break;
    case 64: TT_MX_APPEND(64); break;
    default: TT_MX_APPEND(128); break;
  }
#undef TT_MX_APPEND
  TT_LAUNCHED(fn, s);
  return ok();
}

int check_rows(const char* fn, int dtype, const void* x, const uint8_t* codes, const uint8_t* scales, int64_t rows,
               int64_t cols) {
  const std::string f(fn);
  if (dtype != TT_F32 && dtype != TT_BF16) return fail(TT_ERR_ARG, f + ": dtype must be TT_F32 or TT_BF16");
  if (rows < 0 || cols < 0) return fail(TT_ERR_ARG, f + ": negative size");
  if (rows > 0x7fffffff || cols > 0x7fffffff) return fail(TT_ERR_ARG, f + ": dimension above 2^31 - 1");
  if (rows == 0 || cols == 0) return TT_OK;
  if (!x || !codes || !scales) return fail(TT_ERR_ARG, f + ": null pointer");
  if ((uintptr_t)codes & 15) return fail(TT_ERR_ARG, f + ": codes must be 16-byte aligned");
  return TT_OK;
}

}  // namespace
}  // namespace tt

using namespace tt;

extern "C" int tt_mxfp4_quantize(int dtype, int trans, const void* x, uint8_t* codes, uint8_t* scales, int64_t rows,
                                 int64_t cols, void* stream) {
  const char* fn = "tt_mxfp4_quantize";
  int rc = check_rows(fn, dtype, x, codes, scales, rows, cols);
  if (rc) return rc;
  if (trans != 0 && trans != 1) return fail(TT_ERR_ARG, std::string(fn) + ": trans must be 0 or 1");
  if (rows == 0 || cols == 0) return ok();
  if (trans && !grid_fits((rows + 63) / 64 * ((mx_blocks(cols) + 3) / 4), kMxThreads))
    return fail(TT_ERR_ARG, std::string(fn) + ": too large");
  const size_t nb = (size_t)(rows * mx_blocks(cols)), e = dtype == TT_F32 ? 4 : 2;
  if ((rc = check_no_overlap(fn, {{x, (size_t)rows * cols * e, "x"}},
                             {{codes, nb * kMxBlockBytes, "codes"}, {scales, nb, "scales"}})))
    return rc;
  if ((rc = ensure_init())) return rc;
  hipStream_t s = stream_or_default(stream);
  if (trans)
    return dtype == TT_F32 ? columns_launch<float>(fn, (const float*)x, codes, scales, rows, cols, s)
                           : columns_launch<u16>(fn, (const u16*)x, codes, scales, rows, cols, s);
  return dtype == TT_F32 ? rows_launch<float, true>(fn, (float*)x, codes, scales, rows, cols, s)
                         : rows_launch<u16, true>(fn, (u16*)x, codes, scales, rows, cols, s);
}

extern "C" int tt_mxfp4_dequantize(int dtype, const uint8_t* codes, const uint8_t* scales, void* y, int64_t rows,
                                   int64_t cols, void* stream) {
  const char* fn = "tt_mxfp4_dequantize";
  int rc = check_rows(fn, dtype, y, codes, scales, rows, cols);
  if (rc) return rc;
  if (rows == 0 || cols == 0) return ok();
  const size_t nb = (size_t)(rows * mx_blocks(cols)), e = dtype == TT_F32 ? 4 : 2;
  if ((rc = check_no_overlap(fn, {{codes, nb * kMxBlockBytes, "codes"}, {scales, nb, "scales"}},
                             {{y, (size_t)rows * cols * e, "y"}})))
    return rc;
  if ((rc = ensure_init())) return rc;
  hipStream_t s = stream_or_default(stream);
  return dtype == TT_F32
             ? rows_launch<float, false>(fn, (float*)y, (uint8_t*)codes, (uint8_t*)scales, rows, cols, s)
             : rows_launch<u16, false>(fn, (u16*)y, (uint8_t*)codes, (uint8_t*)scales, rows, cols, s);
}

extern "C" int tt_kv_append_mxfp4(int dtype, const void* k, const void* v, uint8_t* k_codes, uint8_t* k_scales,
                                  uint8_t* v_codes, uint8_t* v_scales, const int* lengths, int64_t B, int64_t Hkv,
                                  int64_t T, int64_t cap, int64_t d, void* stream) {
  const char* fn = "tt_kv_append_mxfp4";
  int rc = check_cache_mxfp4(fn, dtype, B, Hkv, T, cap, d);
  if (rc) return rc;
  if (B == 0 || Hkv == 0 || T == 0 || cap == 0) return ok();
  if (!k || !v || !k_codes || !k_scales || !v_codes || !v_scales || !lengths)
    return fail(TT_ERR_ARG, std::string(fn) + ": null pointer");
  if (((uintptr_t)k_codes | (uintptr_t)v_codes) & 15)
    return fail(TT_ERR_ARG, std::string(fn) + ": codes must be 16-byte aligned");
  const size_t xb = (size_t)(B * Hkv * T * d) * (dtype == TT_F32 ? 4 : 2);
  const size_t cb = (size_t)(B * Hkv * cap * d / 2), sb = (size_t)(B * Hkv * cap * d / kMxBlock);
  if ((rc = check_no_overlap(fn, {{k, xb, "k"}, {v, xb, "v"}, {lengths, (size_t)B * sizeof(int), "lengths"}},
                             {{k_codes, cb, "k_codes"},
                              {k_scales, sb, "k_scales"},
                              {v_codes, cb, "v_codes"},
                              {v_scales, sb, "v_scales"}})))
    return rc;
  if ((rc = ensure_init())) return rc;
  hipStream_t s = stream_or_default(stream);
  return dtype == TT_F32 ? append_launch<float>(fn, (const float*)k, (const float*)v, k_codes, k_scales, v_codes,
                                                v_scales, lengths, B, Hkv, T, cap, d, s)
                         : append_launch<u16>(fn, (const u16*)k, (const u16*)v, k_codes, k_scales, v_codes, v_scales,
                                              lengths, B, Hkv, T, cap, d, s);
}
