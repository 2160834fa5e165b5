// Layer norm over the columns of rows of bf16, fp16 or fp32, and its backward pass, for gfx950: the norm in front of a
// routed layer (moe.py, layer_norm=True).
//
//   m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), z = (x - m) r, y = z w + b
//   g = dy w, dx = r (g - mean(g) - z mean(g z)), dw = sum over rows of dy z, db = sum over rows of dy
//
// Bound by memory: x and y pass once, and in the backward pass x, dy and dx.  A row stays in the registers of the threads
// that share it, so the squares are taken around the mean that is already known (no cancellation where a row lies far off
// zero) and nothing is read twice.  The statistics are kept in fp32 for the backward pass, m and r of every row; every
// sum is taken in fp32, and a result is rounded once.
#include <algorithm>
#include <type_traits>

#include "elements.h"

namespace fp8gmm {
namespace {

constexpr int kNormMaxBlocks = 512;   // workgroups of a backward pass, each with one partial sum of the parameters' gradients
constexpr int kNormLongThreads = 1024;
constexpr int kNormSlab = 1 << 21;   // rows of a launch with a workgroup to a row: a grid has fewer than 2^32 threads

// The sum over the THREADS threads of a row, the same in all of them.  `slot`: THREADS / 64 floats of LDS per row that nobody
// uses before the next barrier but one.
template <int THREADS>
__device__ __forceinline__ float row_sum(float v, float* slot) {
  if constexpr (THREADS <= 64) {
    return lanes_sum<THREADS>(v);
  } else {
    v = lanes_sum<64>(v);
    if (threadIdx.x % 64 == 0) slot[threadIdx.x % THREADS / 64] = v;
    __syncthreads();
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) sum += slot[i];
    return sum;
  }
}

// THREADS threads share a row, C pieces each; a workgroup of 256 at least.
template <int TYPE, int PTYPE, int THREADS, int C>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void layer_norm_kernel(
    const void* __restrict__ x_, int64_t ldx, const void* __restrict__ w, const void* __restrict__ b, void* __restrict__ y_,
    float* __restrict__ mean_out, float* __restrict__ rstd_out, int rows, int cols, float eps) {
  typedef Elements<TYPE> E;
  typedef typename E::bits bits;
  constexpr int V = E::kVec, ROWS = THREADS < 256 ? 256 / THREADS : 1;
  __shared__ float slots[2][THREADS > 64 ? THREADS / 64 : 1];
  const int t = threadIdx.x % THREADS;
  int64_t row = (int64_t)blockIdx.x * ROWS;
  if constexpr (THREADS == 64) row += __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  else if constexpr (THREADS < 64) row += threadIdx.x / THREADS;
  if (row >= rows) return;   // never with more than a wavefront to a row
  const bits* const x = static_cast<const bits*>(x_) + row * ldx;
  u32x4 raw[C];
  Parameters<TYPE, PTYPE> pw[C], pb[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int at = (c * THREADS + t) * V;
    raw[c] = E::load(x + at, cols - at);
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int at = (c * THREADS + t) * V;
    pw[c].load(w, at, cols - at);
    if (b != nullptr) pb[c].load(b, at, cols - at);
  }
  const float count = (float)cols;
  float sum = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    float f[V];
    E::unpack(raw[c], f);
#pragma unroll
    for (int i = 0; i < V; ++i) sum += f[i];
  }
  const float mean = row_sum<THREADS>(sum, slots[0]) / count;
  float squares = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int n = cols - (c * THREADS + t) * V;
    float f[V];
    E::unpack(raw[c], f);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float d = i < n ? f[i] - mean : 0.f;
      squares = __builtin_fmaf(d, d, squares);
    }
  }
  const float rstd = 1.0f / sqrtf(row_sum<THREADS>(squares, slots[1]) / count + eps);
  if (mean_out != nullptr && t == 0) {
    mean_out[row] = mean;
    rstd_out[row] = rstd;
  }
  bits* const y = static_cast<bits*>(y_) + row * cols;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int at = (c * THREADS + t) * V;
    float f[V], fw[V], fb[V];
    E::unpack(raw[c], f);
    pw[c].get(fw);
    if (b != nullptr) pb[c].get(fb);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = __builtin_fmaf((f[i] - mean) * rstd, fw[i], b != nullptr ? fb[i] : 0.f);
    E::store(y + at, cols - at, E::pack(f));
  }
}

// Rows that no workgroup's registers hold are read three times, from the cache the second and third time.
template <int TYPE, int PTYPE>
__global__ __launch_bounds__(kNormLongThreads) void layer_norm_long_kernel(
    const void* __restrict__ x_, int64_t ldx, const void* __restrict__ w, const void* __restrict__ b, void* __restrict__ y_,
    float* __restrict__ mean_out, float* __restrict__ rstd_out, int cols, float eps) {
  typedef Elements<TYPE> E;
  typedef typename E::bits bits;
  constexpr int V = E::kVec, STEP = kNormLongThreads * V;
  __shared__ float slots[2][kNormLongThreads / 64];
  const int64_t row = blockIdx.x;
  const int t = threadIdx.x;
  const bits* const x = static_cast<const bits*>(x_) + row * ldx;
  const float count = (float)cols;
  float sum = 0.f;
  for (int64_t at = t * V; at < cols; at += STEP) {
    float f[V];
    E::unpack(E::load(x + at, (int)(cols - at)), f);
#pragma unroll
    for (int i = 0; i < V; ++i) sum += f[i];
  }
  const float mean = row_sum<kNormLongThreads>(sum, slots[0]) / count;
  float squares = 0.f;
  for (int64_t at = t * V; at < cols; at += STEP) {
    const int n = (int)(cols - at);
    float f[V];
    E::unpack(E::load(x + at, n), f);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float d = i < n ? f[i] - mean : 0.f;
      squares = __builtin_fmaf(d, d, squares);
    }
  }
  const float rstd = 1.0f / sqrtf(row_sum<kNormLongThreads>(squares, slots[1]) / count + eps);
  if (mean_out != nullptr && t == 0) {
    mean_out[row] = mean;
    rstd_out[row] = rstd;
  }
  bits* const y = static_cast<bits*>(y_) + row * cols;
  for (int64_t at = t * V; at < cols; at += STEP) {
    const int n = (int)(cols - at);
    Parameters<TYPE, PTYPE> pw, pb;
    pw.load(w, (int)at, n);
    if (b != nullptr) pb.load(b, (int)at, n);
    float f[V], fw[V], fb[V];
    E::unpack(E::load(x + at, n), f);
    pw.get(fw);
    if (b != nullptr) pb.get(fb);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = __builtin_fmaf((f[i] - mean) * rstd, fw[i], b != nullptr ? fb[i] : 0.f);
    E::store(y + at, n, E::pack(f));
  }
}

// Threads of a workgroup of the backward pass whose threads hold C pieces of a row each: as many rows at a time as their
// registers allow, since every workgroup leaves one partial sum of the parameters' gradients in memory.
constexpr int backward_threads(int c) { return c >= 4 ? 512 : 1024; }

// A workgroup takes ROWS rows at a time, THREADS threads and C pieces each, and keeps the sums of dy z and dy for its
// columns; the rows' next ones are loaded before the sums of the present ones are shared.  `part`: [workgroup][2][cols], the
// second without a bias left out; NULL where the parameters take no gradients.  dx may be NULL.
template <int TYPE, int PTYPE, int THREADS, int C>
__global__ __launch_bounds__(THREADS > backward_threads(C) ? THREADS : backward_threads(C)) void layer_norm_backward_kernel(
    const void* __restrict__ dy_, int64_t ldy, const void* __restrict__ x_, int64_t ldx, const void* __restrict__ w,
    const float* __restrict__ mean_in, const float* __restrict__ rstd_in, void* __restrict__ dx_, float* __restrict__ part,
    int bias, int rows, int cols) {
  typedef Elements<TYPE> E;
  typedef typename E::bits bits;
  constexpr int BLOCK = THREADS > backward_threads(C) ? THREADS : backward_threads(C);
  constexpr int V = E::kVec, ROWS = BLOCK / THREADS, WAVES = THREADS > 64 ? THREADS / 64 : 1;
  __shared__ float slots[2][2][ROWS][WAVES];
  __shared__ float sums[BLOCK * V];
  const int t = threadIdx.x % THREADS;
  int group = threadIdx.x / THREADS;
  if constexpr (THREADS >= 64) group = __builtin_amdgcn_readfirstlane(group);
  Parameters<TYPE, PTYPE> pw[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int at = (c * THREADS + t) * V;
    pw[c].load(w, at, cols - at);
  }
  float dw[C][V] = {}, db[C][V] = {};
  u32x4 nx[C], ny[C];
  float nm = 0.f, nr = 0.f;
  const auto load = [&](int64_t row) {
    const bool live = row < rows;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int at = (c * THREADS + t) * V;
      nx[c] = E::load(static_cast<const bits*>(x_) + row * ldx + at, live ? cols - at : 0);
      ny[c] = E::load(static_cast<const bits*>(dy_) + row * ldy + at, live ? cols - at : 0);
    }
    nm = live ? mean_in[row] : 0.f;
    nr = live ? rstd_in[row] : 0.f;
  };
  const int64_t stride = (int64_t)gridDim.x * ROWS;
  int64_t row = (int64_t)blockIdx.x * ROWS + group;
  load(row);
  int turn = 0;
  for (int64_t first = (int64_t)blockIdx.x * ROWS; first < rows; first += stride, row += stride, turn ^= 1) {
    u32x4 x[C], y[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      x[c] = nx[c];
      y[c] = ny[c];
    }
    const float mean = nm, rstd = nr;
    load(row + stride);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float fx[V], fy[V], fw[V];
      E::unpack(x[c], fx);
      E::unpack(y[c], fy);
      pw[c].get(fw);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float z = (fx[i] - mean) * rstd, g = fy[i] * fw[i];
        s1 += g;
        s2 = __builtin_fmaf(g, z, s2);
        dw[c][i] = __builtin_fmaf(fy[i], z, dw[c][i]);
        db[c][i] += fy[i];
      }
    }
    if (dx_ == nullptr) continue;
    if constexpr (THREADS <= 64) {
      s1 = lanes_sum<THREADS>(s1);
      s2 = lanes_sum<THREADS>(s2);
    } else {   // both with one barrier; the other turn's slots are read before the next one
      s1 = lanes_sum<64>(s1);
      s2 = lanes_sum<64>(s2);
      if (threadIdx.x % 64 == 0) {
        slots[turn][0][group][t / 64] = s1;
        slots[turn][1][group][t / 64] = s2;
      }
      __syncthreads();
      s1 = s2 = 0.f;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) {
        s1 += slots[turn][0][group][i];
        s2 += slots[turn][1][group][i];
      }
    }
    if (row >= rows) continue;
    const float m1 = s1 / (float)cols, m2 = s2 / (float)cols;
    bits* const dx = static_cast<bits*>(dx_) + row * cols;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int at = (c * THREADS + t) * V;
      float fx[V], fy[V], fw[V];
      E::unpack(x[c], fx);
      E::unpack(y[c], fy);
      pw[c].get(fw);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float z = (fx[i] - mean) * rstd;
        fx[i] = rstd * (__builtin_fmaf(fy[i], fw[i], -m1) - z * m2);
      }
      E::store(dx + at, cols - at, E::pack(fx));
    }
  }
  if (part == nullptr) return;
  // the workgroup's rows together, in their order: THREADS * V columns at a time
  float* const out = part + (int64_t)blockIdx.x * 2 * cols;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      if (which == 1 && !bias) continue;
      if constexpr (ROWS > 1) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) sums[(group * THREADS + t) * V + i] = which == 0 ? dw[c][i] : db[c][i];
        __syncthreads();
        for (int col = threadIdx.x; col < THREADS * V; col += BLOCK) {
          float sum = 0.f;
#pragma unroll
          for (int r = 0; r < ROWS; ++r) sum += sums[r * THREADS * V + col];
          const int64_t at = (int64_t)c * THREADS * V + col;
          if (at < cols) out[(int64_t)which * cols + at] = sum;
        }
      } else {
        const int at = (c * THREADS + t) * V;
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (at + i < cols) out[(int64_t)which * cols + at + i] = which == 0 ? dw[c][i] : db[c][i];
      }
    }
}

// dx of a row that no workgroup's registers hold
template <int TYPE, int PTYPE>
__global__ __launch_bounds__(kNormLongThreads) void layer_norm_long_dx_kernel(
    const void* __restrict__ dy_, int64_t ldy, const void* __restrict__ x_, int64_t ldx, const void* __restrict__ w,
    const float* __restrict__ mean_in, const float* __restrict__ rstd_in, void* __restrict__ dx_, int cols) {
  typedef Elements<TYPE> E;
  typedef typename E::bits bits;
  constexpr int V = E::kVec, STEP = kNormLongThreads * V;
  __shared__ float slots[2][kNormLongThreads / 64];
  const int64_t row = blockIdx.x;
  const int t = threadIdx.x;
  const bits* const x = static_cast<const bits*>(x_) + row * ldx;
  const bits* const dy = static_cast<const bits*>(dy_) + row * ldy;
  bits* const dx = static_cast<bits*>(dx_) + row * cols;
  const float mean = mean_in[row], rstd = rstd_in[row];
  float s1 = 0.f, s2 = 0.f, m1 = 0.f, m2 = 0.f;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    for (int64_t at = t * V; at < cols; at += STEP) {
      const int n = (int)(cols - at);
      Parameters<TYPE, PTYPE> pw;
      pw.load(w, (int)at, n);
      float fx[V], fy[V], fw[V];
      E::unpack(E::load(x + at, n), fx);
      E::unpack(E::load(dy + at, n), fy);
      pw.get(fw);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float z = (fx[i] - mean) * rstd, g = fy[i] * fw[i];
        s1 += g;
        s2 = __builtin_fmaf(g, z, s2);
        fx[i] = rstd * (g - m1 - z * m2);
      }
      if (pass == 1) E::store(dx + at, n, E::pack(fx));
    }
    if (pass == 0) {
      m1 = row_sum<kNormLongThreads>(s1, slots[0]) / (float)cols;
      m2 = row_sum<kNormLongThreads>(s2, slots[1]) / (float)cols;
    }
  }
}

// The parameters' gradients of such rows: a thread keeps one piece of the columns for a slice of the rows.
template <int TYPE>
__global__ __launch_bounds__(256) void layer_norm_long_params_kernel(
    const void* __restrict__ dy_, int64_t ldy, const void* __restrict__ x_, int64_t ldx, const float* __restrict__ mean_in,
    const float* __restrict__ rstd_in, float* __restrict__ part, int bias, int rows, int cols) {
  typedef Elements<TYPE> E;
  typedef typename E::bits bits;
  constexpr int V = E::kVec;
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
  if (at >= cols) return;
  const int n = (int)(cols - at);
  float dw[V] = {}, db[V] = {};
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const float mean = mean_in[row], rstd = rstd_in[row];
    float fx[V], fy[V];
    E::unpack(E::load(static_cast<const bits*>(x_) + row * ldx + at, n), fx);
    E::unpack(E::load(static_cast<const bits*>(dy_) + row * ldy + at, n), fy);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      dw[i] = __builtin_fmaf(fy[i], (fx[i] - mean) * rstd, dw[i]);
      db[i] += fy[i];
    }
  }
  float* const out = part + (int64_t)blockIdx.y * 2 * cols + at;
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < n) {
      out[i] = dw[i];
      if (bias) out[cols + i] = db[i];
    }
}

// The workgroups' partial sums, in their order: 64 columns a workgroup, a sixteenth of the sums a wavefront.  Without any
// (no rows) the gradients are zeros.
template <int PTYPE>
__global__ __launch_bounds__(1024) void layer_norm_params_kernel(const float* __restrict__ part, int blocks, int cols,
                                                                 void* __restrict__ dweight, void* __restrict__ dbias) {
  typedef Elements<PTYPE> P;
  __shared__ float sums[16][64];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, which = blockIdx.y;
  const int64_t col = (int64_t)blockIdx.x * 64 + lane;
  void* const out = which == 0 ? dweight : dbias;
  float sum = 0.f;
  if (col < cols) {
    const int per = (blocks + 15) / 16, last = min(blocks, (wave + 1) * per);
    const float* p = part + (int64_t)which * cols + col;
#pragma unroll 8
    for (int i = wave * per; i < last; ++i) sum += p[(int64_t)i * 2 * cols];
  }
  sums[wave][lane] = sum;
  __syncthreads();
  if (wave != 0 || col >= cols || out == nullptr) return;
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) sum += sums[i][lane];
  static_cast<typename P::bits*>(out)[col] = P::pack1(sum);
}

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// How a row's pieces are shared out: threads to a row and pieces to a thread, by the number of pieces.  Zero threads: longer
// than the registers of a workgroup hold.
struct Shape {
  int threads, pieces;
};
Shape norm_shape(int cols, int type) {
  const int pieces = ceil_div(cols, type == FP8GMM_TYPE_FP32 ? 4 : 8);
  if (pieces <= 16) return {16, 1};
  if (pieces <= 64) return {64, 1};
  if (pieces <= 128) return {64, 2};
  if (pieces <= 256) return {64, 4};
  if (pieces <= 512) return {256, 2};
  if (pieces <= 1024) return {256, 4};
  if (pieces <= 2048) return {1024, 2};
  if (pieces <= 4096) return {1024, 4};
  return {0, 0};
}
// Workgroups of a backward pass: partial sums that its parameters' gradients have.
int backward_blocks(int rows, int cols, int type) {
  const Shape s = norm_shape(cols, type);
  if (s.threads == 0) return std::min(rows, 64);
  const int block = std::max(s.threads, backward_threads(s.pieces));
  return std::min(ceil_div(rows, block / s.threads), kNormMaxBlocks * 512 / block);
}

#define FP8GMM_NORM_SHAPES(X) X(16, 1) X(64, 1) X(64, 2) X(64, 4) X(256, 2) X(256, 4) X(1024, 2) X(1024, 4)

// calls f(TYPE, PTYPE) with the two as integral constants
template <class F>
void with_types(int type, int param_type, F&& f) {
  constexpr std::integral_constant<int, FP8GMM_TYPE_BF16> bf16{};
  constexpr std::integral_constant<int, FP8GMM_TYPE_FP16> fp16{};
  constexpr std::integral_constant<int, FP8GMM_TYPE_FP32> fp32{};
  if (type == FP8GMM_TYPE_FP32) f(fp32, fp32);
  else if (type == FP8GMM_TYPE_BF16) param_type == FP8GMM_TYPE_FP32 ? f(bf16, fp32) : f(bf16, bf16);
  else param_type == FP8GMM_TYPE_FP32 ? f(fp16, fp32) : f(fp16, fp16);
}

int check_norm(int64_t rows, int cols, int64_t ldx, int type, int param_type) {
  if (!known_type(type) || (param_type != type && param_type != FP8GMM_TYPE_FP32)) return FP8GMM_ERR_BAD_FORMAT;
  // a row's offsets in 32 bits, with room for the last piece's
  if (rows < 0 || rows > INT32_MAX || cols < 1 || cols > (1 << 30) || ldx < cols) return FP8GMM_ERR_BAD_SHAPE;
  return FP8GMM_OK;
}

}  // namespace
}  // namespace fp8gmm

extern "C" {

int fp8gmm_layer_norm(const void* x, int64_t ldx, const void* weight, const void* bias, void* y, float* mean, float* rstd,
                      int64_t rows, int cols, float eps, int type, int param_type, void* stream) {
  using namespace fp8gmm;
  const int rc = check_norm(rows, cols, ldx, type, param_type);
  if (rc != FP8GMM_OK) return rc;
  if (!(eps >= 0.f)) return FP8GMM_ERR_BAD_ARGUMENT;
  if (rows == 0) return FP8GMM_OK;
  if (x == nullptr || weight == nullptr || y == nullptr || (mean == nullptr) != (rstd == nullptr)) return FP8GMM_ERR_NULL_POINTER;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const Shape shape = norm_shape(cols, type);
  for (int64_t r0 = 0; r0 < rows; r0 += kNormSlab) {
    const int n = (int)std::min<int64_t>(kNormSlab, rows - r0), size = type_bytes(type);
    const void* const xs = static_cast<const char*>(x) + r0 * ldx * size;
    void* const ys = static_cast<char*>(y) + r0 * cols * size;
    float* const ms = mean != nullptr ? mean + r0 : nullptr;
    float* const rs = rstd != nullptr ? rstd + r0 : nullptr;
    with_types(type, param_type, [&](auto tc, auto pc) {
      constexpr int T = decltype(tc)::value, P = decltype(pc)::value;
#define FP8GMM_LAUNCH(THREADS, C)                                                                                       \
  if (shape.threads == THREADS && shape.pieces == C)                                                                    \
    hipLaunchKernelGGL((layer_norm_kernel<T, P, THREADS, C>), dim3(ceil_div(n, THREADS < 256 ? 256 / THREADS : 1)),     \
                       dim3(THREADS < 256 ? 256 : THREADS), 0, s, xs, ldx, weight, bias, ys, ms, rs, n, cols, eps);
      FP8GMM_NORM_SHAPES(FP8GMM_LAUNCH)
#undef FP8GMM_LAUNCH
      if (shape.threads == 0)
        hipLaunchKernelGGL((layer_norm_long_kernel<T, P>), dim3(n), dim3(kNormLongThreads), 0, s, xs, ldx, weight, bias, ys, ms,
                           rs, cols, eps);
    });
  }
  return hipGetLastError() == hipSuccess ? FP8GMM_OK : FP8GMM_ERR_LAUNCH;
}

size_t fp8gmm_layer_norm_workspace_bytes(int64_t rows, int cols, int type) {
  using namespace fp8gmm;
  if (check_norm(rows, cols, cols, type, type) != FP8GMM_OK) return 0;
  return (size_t)backward_blocks((int)rows, cols, type) * 2 * cols * sizeof(float);
}

int fp8gmm_layer_norm_backward(const void* dy, int64_t ldy, const void* x, int64_t ldx, const void* weight, const float* mean,
                               const float* rstd, void* dx, void* dweight, void* dbias, int64_t rows, int cols, int type,
                               int param_type, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace fp8gmm;
  const int rc = check_norm(rows, cols, std::min(ldx, ldy), type, param_type);
  if (rc != FP8GMM_OK) return rc;
  const bool params = dweight != nullptr || dbias != nullptr;
  if (rows > 0 && (dy == nullptr || x == nullptr || weight == nullptr || mean == nullptr || rstd == nullptr))
    return FP8GMM_ERR_NULL_POINTER;
  if (params && rows > 0) {
    if (workspace == nullptr) return FP8GMM_ERR_NULL_POINTER;
    if (workspace_bytes < fp8gmm_layer_norm_workspace_bytes(rows, cols, type)) return FP8GMM_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return FP8GMM_ERR_ALIGNMENT;
  }
  if (!params && (dx == nullptr || rows == 0)) return FP8GMM_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  float* const part = params ? static_cast<float*>(workspace) : nullptr;
  const int blocks = backward_blocks((int)rows, cols, type), bias = dbias != nullptr;
  const Shape shape = norm_shape(cols, type);
  with_types(type, param_type, [&](auto tc, auto pc) {
    constexpr int T = decltype(tc)::value, P = decltype(pc)::value;
    if (rows > 0) {
#define FP8GMM_LAUNCH(THREADS, C)                                                                                       \
  if (shape.threads == THREADS && shape.pieces == C)                                                                    \
    hipLaunchKernelGGL((layer_norm_backward_kernel<T, P, THREADS, C>), dim3(blocks),                                    \
                       dim3(THREADS > backward_threads(C) ? THREADS : backward_threads(C)), 0, s, dy, ldy, x, ldx, weight, \
                       mean, rstd, dx, part, bias, (int)rows, cols);
      FP8GMM_NORM_SHAPES(FP8GMM_LAUNCH)
#undef FP8GMM_LAUNCH
      if (shape.threads == 0) {
        for (int64_t r0 = 0; dx != nullptr && r0 < rows; r0 += kNormSlab) {
          const int size = type_bytes(type);
          hipLaunchKernelGGL((layer_norm_long_dx_kernel<T, P>), dim3((unsigned)std::min<int64_t>(kNormSlab, rows - r0)),
                             dim3(kNormLongThreads), 0, s, static_cast<const char*>(dy) + r0 * ldy * size, ldy,
                             static_cast<const char*>(x) + r0 * ldx * size, ldx, weight, mean + r0, rstd + r0,
                             static_cast<char*>(dx) + r0 * cols * size, cols);
        }
        if (params)
          hipLaunchKernelGGL((layer_norm_long_params_kernel<T>), dim3(ceil_div(cols, 256 * Elements<T>::kVec), blocks), dim3(256),
                             0, s, dy, ldy, x, ldx, mean, rstd, part, bias, (int)rows, cols);
      }
    }
    if (params)
      hipLaunchKernelGGL((layer_norm_params_kernel<P>), dim3(ceil_div(cols, 64), dbias != nullptr ? 2 : 1), dim3(1024), 0, s,
                         part, blocks, cols, dweight, dbias);
  });
  return hipGetLastError() == hipSuccess ? FP8GMM_OK : FP8GMM_ERR_LAUNCH;
}

}  // extern "C"
