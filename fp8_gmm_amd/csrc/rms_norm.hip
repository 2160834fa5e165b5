// Root-mean-square norm over the columns of rows of bf16, fp16 or fp32, for gfx950, with the addition of a residual in front, a result
// in 8 bits, and the backward pass: the norm in front of a routed layer (moe.py, rms_norm=True) or of a product in 8 bits.
//
//   h = x + residual, rounded (without a residual x itself), r = 1 / sqrt(mean(h^2) + eps), z = h r, y = z w
//   g = dy w, dx = dh + r (g - z mean(g z)), dw = sum over rows of dy z
//   in 8 bits: q = fp8(y s) by the tensor's scale s, with the largest |y| recorded, or by the row's, s = most / max |y|
//
// The norm is that of the rows as h is returned, so that the backward pass starts from what the forward pass ended with.  Bound by
// memory: every row passes once in and once out.  Sums are taken in fp32, a result is rounded once.
#include <algorithm>

#include "norm_rows.h"

namespace fp8gmm {
namespace {

constexpr int kBackwardThreads = 1024;   // of a workgroup of the backward pass: as many rows at a time as fit, since every workgroup
constexpr int kBackwardBlocks = 256;     // leaves one partial sum of the weight's gradient in memory; one per compute unit
constexpr int kBackwardAlone = 2;        // turns of one workgroup that take less than a second launch for the sums of several
constexpr int kForwardThreads = 256;     // of a workgroup of the forward pass, where a row needs no more
// What a forward pass writes: the normed rows (of x, or of the sum with a residual, which it writes as well), or these in 8 bits
enum { kRows, kSums, kBits8 };
// Threads of its launch, which go on to other rows.  With 8 bits what the compute units hold at a time, three times that where they would go
// on more than five times; else four times as many (16384 x 4096, bf16, with a residual 89.5 us, what they hold alone 90.5; without one 44.3
// and 46.7; 16384 x 4093 92.9 and 97.0; but in 8 bits 81.4 and 79.2).
constexpr int kForwardAll = 256 * 2048, kForwardTurns = 5, kForwardMore = 3, kForwardFour = 4;

// The least magnitude that a row's scale is made of: what is smaller is zero in 8 bits, and no scale is zero.
constexpr float kLeast = 0x1p-100f;

__device__ __forceinline__ float most_of(int fmt) { return fmt == FP8GMM_E4M3 ? Fp8Limits<FP8GMM_E4M3>::kMax : Fp8Limits<FP8GMM_E5M2>::kMax; }

// The first n of V values in 8 bits, at any byte
typedef uint32_t u32_any1 __attribute__((aligned(1)));
typedef uint32_t u32x2_any1 __attribute__((ext_vector_type(2), aligned(1)));
template <int V>
__device__ __forceinline__ void store8(uint8_t* p, int n, const float (&f)[V], int fmt) {
  uint32_t w[V / 4];
#pragma unroll
  for (int i = 0; i < V / 4; ++i)
    w[i] = fmt == FP8GMM_E4M3 ? cvt4_fp8<FP8GMM_E4M3>(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3])
                              : cvt4_fp8<FP8GMM_E5M2>(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
  if (n >= V) {
    if constexpr (V == 8) *reinterpret_cast<u32x2_any1*>(p) = u32x2{w[0], w[1]};
    else *reinterpret_cast<u32_any1*>(p) = w[0];
    return;
  }
#pragma unroll
  for (int i = 0; i < V - 1; ++i)
    if (i < n) p[i] = (uint8_t)(w[i / 4] >> i % 4 * 8);
}

// The largest over the workgroup's threads; `slot` as of row_sum
template <int THREADS>
__device__ __forceinline__ float row_max(float v, float* slot) {
  v = wave_max(v);
  if (threadIdx.x % 64 == 0) slot[threadIdx.x / 64] = v;
  __syncthreads();
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < THREADS / 64; ++i) most = fmaxf(most, slot[i]);
  return most;
}

// Where an 8-bit result goes, and its scales: `scale` and `amax` (may be NULL) of the tensor, or `scale_inv` of every row
struct Bits8 {
  uint8_t* q;
  const float* scale;
  float* amax;
  float* scale_inv;
  int fmt;
};

// A workgroup takes ROWS rows at a time, LANES * waves threads to a row and C pieces to a thread, and goes on to other rows by the grid:
// the next rows are loaded before the sums of the present ones are shared, and the weight stays in registers.
template <int TYPE, int PTYPE, int LANES, int C, int MODE, int MOST, int KIND>
__global__ __launch_bounds__(MOST) void rms_norm_kernel(
    const void* __restrict__ x_, int64_t ldx, const void* __restrict__ residual_, int64_t ldr, const void* __restrict__ w,
    void* __restrict__ y_, const Bits8 bits8, void* __restrict__ h_, float* __restrict__ rstd_out, int rows, int cols, float eps, int waves,
    bool stream) {
  typedef Elements<TYPE> E;
  constexpr int V = E::kVec;
  // With the streaming hint, but for rows that are the residual stream themselves (16384 x 4096, bf16, with a residual 89.5 us, without the
  // hint 93.0; in 8 bits 74 and 84; without a residual 45.0 and 44.3).
  constexpr bool BITS8 = KIND == kBits8, STREAM = KIND != kRows;
  __shared__ float slots[2][kNormWaves][kNormWaves], tops[2][kNormWaves][kNormWaves];
  const int THREADS = LANES * waves, ROWS = blockDim.x / THREADS;
  int group = threadIdx.x / THREADS;
  if constexpr (LANES == 64) group = __builtin_amdgcn_readfirstlane(group);
  const int t = threadIdx.x - group * THREADS;
  int at[C];
#pragma unroll
  for (int c = 0; c < C; ++c) at[c] = (c * THREADS + t) * V;
  const int skip = piece_skip<MODE, V>(at[C - 1], cols);   // the pieces before the last one are there in whole
  at[C - 1] = piece_begin<MODE, V>(at[C - 1], cols);
  const bool added = KIND == kSums || (BITS8 && residual_ != nullptr);
  u32x4 nx[C], nr[C];
  const auto load = [&](int64_t row) {
    const RowAccess<TYPE, MODE> x(x_, row, rows, ldx, cols);
#pragma unroll
    for (int c = 0; c < C; ++c) nx[c] = x.template load<STREAM>(at[c]);
    if (added) {
      const RowAccess<TYPE, MODE> residual(residual_, row, rows, ldr, cols);
#pragma unroll
      for (int c = 0; c < C; ++c) nr[c] = residual.template load<STREAM>(at[c]);
    }
  };
  const int64_t stride = (int64_t)gridDim.x * ROWS;
  int64_t row = (int64_t)blockIdx.x * ROWS + group;
  load(row);
  Parameters<TYPE, PTYPE> pw[C];
#pragma unroll
  for (int c = 0; c < C; ++c) pw[c].load(w, at[c], cols - at[c]);
  const int wave = LANES == 64 ? __builtin_amdgcn_readfirstlane(t / 64) : 0;
  const int peer = threadIdx.x % 16;   // the wavefront whose share this lane takes up where they meet
  const float count = (float)cols;
  float top = 0.f;   // of all rows
  const float tensor_scale = BITS8 && bits8.scale != nullptr ? *bits8.scale : 0.f;
  int turn = 0;
  for (int64_t first = (int64_t)blockIdx.x * ROWS; first < rows; first += stride, row += stride, turn ^= 1) {
    u32x4 x[C];
#pragma unroll
    for (int c = 0; c < C; ++c) x[c] = nx[c];
    if (added) {
      const RowAccess<TYPE, MODE> h(h_, row, rows, cols, cols);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float f[V], a[V];
        E::unpack(x[c], f);
        E::unpack(nr[c], a);
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] += a[i];
        x[c] = E::pack(f);
        h.store(at[c], x[c], stream);
      }
    }
    if (first + stride < rows) load(row + stride);
    float squares = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float f[V];
      E::unpack(x[c], f);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float v = !is_edge(MODE) || c < C - 1 || i >= skip ? f[i] : 0.f;
        squares = __builtin_fmaf(v, v, squares);
      }
    }
    squares = lanes_sum<LANES>(squares);
    if (LANES == 64 && waves > 1) {   // the other turn's slots are read before the next barrier
      if (threadIdx.x % 64 == 0) slots[turn][group][wave] = squares;
      __syncthreads();
      squares = lanes_sum<16>(peer < waves ? slots[turn][group][peer] : 0.f);
    }
    const float rstd = 1.0f / sqrtf(squares / count + eps);
    if (rstd_out != nullptr && t == 0 && row < rows) rstd_out[row] = rstd;
    const auto normed = [&](int c, float (&f)[V]) {
      float fw[V];
      E::unpack(x[c], f);
      pw[c].get(fw);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = f[i] * rstd * fw[i];
    };
    if constexpr (BITS8) {
      float scale = tensor_scale, most = 0.f;
      if (bits8.scale == nullptr || bits8.amax != nullptr) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
          float f[V];
          normed(c, f);
#pragma unroll
          for (int i = 0; i < V; ++i)   // (a piece behind the end is zeros times the row's factor, be that infinite)
            if (is_edge(MODE) || at[c] + i < cols) most = amax_step(most, f[i]);
        }
        if (bits8.scale != nullptr) top = fmaxf(top, most);
      }
      if (bits8.scale == nullptr) {
        most = lanes_max<LANES>(most);
        if (LANES == 64 && waves > 1) {
          if (threadIdx.x % 64 == 0) tops[turn][group][wave] = most;
          __syncthreads();
          most = lanes_max<16>(peer < waves ? tops[turn][group][peer] : 0.f);
        }
        most = fmaxf(most, kLeast);
        scale = most_of(bits8.fmt) / most;
        if (t == 0 && row < rows) bits8.scale_inv[row] = most / most_of(bits8.fmt);
      }
      if (is_edge(MODE) || row < rows) {
        uint8_t* const q = bits8.q + (row < rows ? row : rows - 1) * (int64_t)cols;
#pragma unroll
        for (int c = 0; c < C; ++c) {
          float f[V];
          normed(c, f);
#pragma unroll
          for (int i = 0; i < V; ++i) f[i] *= scale;
          if (is_edge(MODE) || at[c] < cols) store8<V>(q + at[c], MODE == kShort ? cols - at[c] : V, f, bits8.fmt);
        }
      }
    } else {
      const RowAccess<TYPE, MODE> y(y_, row, rows, cols, cols);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float f[V];
        normed(c, f);
        y.store(at[c], E::pack(f), stream);
      }
    }
  }
  if (BITS8 && bits8.amax != nullptr) {
    __syncthreads();
    top = lanes_max<64>(top);
    float* const meet = &tops[0][0][0];
    if (threadIdx.x % 64 == 0) meet[threadIdx.x / 64] = top;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int i = 1; i < (int)(blockDim.x / 64); ++i) top = fmaxf(top, meet[i]);
    if (!(__builtin_nontemporal_load(bits8.amax) >= top)) atomic_max_nonneg(bits8.amax, top);
  }
}

// The backward pass in the same way, with the sums of dy z for the columns of its threads.  `part`: [workgroup][cols]; NULL where the
// weight takes no gradient.  dx may be NULL.  A single workgroup writes the gradient itself.
template <int TYPE, int PTYPE, int LANES, int C, int MODE>
__global__ __launch_bounds__(kBackwardThreads) void rms_norm_backward_kernel(
    const void* __restrict__ dy_, int64_t ldy, const void* __restrict__ dh_, int64_t ldd, const void* __restrict__ h_, int64_t ldh,
    const void* __restrict__ w, const float* __restrict__ rstd_in, void* __restrict__ dx_, float* __restrict__ part,
    void* __restrict__ dweight, int rows, int cols, int waves, bool stream) {
  typedef Elements<TYPE> E;
  constexpr int V = E::kVec;
  __shared__ float slots[2][kNormWaves][kNormWaves];
  __shared__ float sums[kBackwardThreads * V];
  const int THREADS = LANES * waves, ROWS = blockDim.x / THREADS;
  int group = threadIdx.x / THREADS;
  if constexpr (LANES == 64) group = __builtin_amdgcn_readfirstlane(group);
  const int t = threadIdx.x - group * THREADS;
  const int wave = LANES == 64 ? __builtin_amdgcn_readfirstlane(t / 64) : 0, peer = threadIdx.x % 16;
  int at[C];
#pragma unroll
  for (int c = 0; c < C; ++c) at[c] = (c * THREADS + t) * V;
  const int skip = piece_skip<MODE, V>(at[C - 1], cols);   // the pieces before the last one are there in whole
  at[C - 1] = piece_begin<MODE, V>(at[C - 1], cols);
  Parameters<TYPE, PTYPE> pw[C];
#pragma unroll
  for (int c = 0; c < C; ++c) pw[c].load(w, at[c], cols - at[c]);
  float dw[C][V] = {};
  u32x4 nh[C], ny[C];
  float nr;
  const auto load = [&](int64_t row) {
    const RowAccess<TYPE, MODE> h(h_, row, rows, ldh, cols), y(dy_, row, rows, ldy, cols);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      nh[c] = h.template load<true>(at[c]);
      ny[c] = y.template load<true>(at[c]);
    }
    nr = row < rows ? rstd_in[row] : 0.f;
  };
  const int64_t stride = (int64_t)gridDim.x * ROWS;
  int64_t row = (int64_t)blockIdx.x * ROWS + group;
  load(row);
  int turn = 0;
  for (int64_t first = (int64_t)blockIdx.x * ROWS; first < rows; first += stride, row += stride, turn ^= 1) {
    u32x4 h[C], y[C], d[C];   // d is wanted behind the sum alone: it comes with its own row, ahead of the next one's loads
#pragma unroll
    for (int c = 0; c < C; ++c) {
      h[c] = nh[c];
      y[c] = ny[c];
      d[c] = u32x4{0u, 0u, 0u, 0u};
    }
    if (dh_ != nullptr) {
      const RowAccess<TYPE, MODE> from(dh_, row, rows, ldd, cols);
#pragma unroll
      for (int c = 0; c < C; ++c) d[c] = from.template load<true>(at[c]);
    }
    const float rstd = nr;
    if (first + stride < rows) load(row + stride);
    float s = 0.f;
    if (!is_edge(MODE) || row < rows) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float fh[V], fy[V], fw[V];
        E::unpack(h[c], fh);
        E::unpack(y[c], fy);
        pw[c].get(fw);
        float u = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if (is_edge(MODE) && c == C - 1 && i < skip) fy[i] = 0.f;   // elsewhere they are zeros
          const float z = MODE != kShort || i < cols ? fh[i] * rstd : 0.f;
          u = __builtin_fmaf(fy[i] * fw[i], z, u);
          dw[c][i] = __builtin_fmaf(fy[i], z, dw[c][i]);
        }
        s += c < C - 1 || skip < V ? u : 0.f;   // nothing of a piece behind the end, whose zeros meet the row's factor, be that infinite
      }
    }
    if (dx_ == nullptr) continue;
    s = lanes_sum<LANES>(s);
    if (LANES == 64 && waves > 1) {   // the other turn's slots are read before the next barrier
      if (threadIdx.x % 64 == 0) slots[turn][group][wave] = s;
      __syncthreads();
      s = lanes_sum<16>(peer < waves ? slots[turn][group][peer] : 0.f);
    }
    if (is_edge(MODE) && row >= rows) continue;   // its sums leave no row out
    const float mean = s / (float)cols;
    const RowAccess<TYPE, MODE> dx(dx_, row, rows, cols, cols);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float fh[V], fy[V], fw[V], fd[V];
      E::unpack(h[c], fh);
      E::unpack(y[c], fy);
      E::unpack(d[c], fd);
      pw[c].get(fw);
#pragma unroll
      for (int i = 0; i < V; ++i)
        fd[i] = __builtin_fmaf(rstd, __builtin_fmaf(fy[i], fw[i], -(fh[i] * rstd) * mean), fd[i]);
      dx.store(at[c], E::pack(fd), stream);
    }
  }
  if (part == nullptr) return;
  // the workgroup's rows together, in their order: THREADS * V columns at a time
  float* const out = part + (int64_t)blockIdx.x * cols;
  const auto write = [&](int64_t col, float sum) {
    typedef Elements<PTYPE> P;
    if (gridDim.x > 1) out[col] = sum;
    else static_cast<typename P::bits*>(dweight)[col] = P::pack1(sum);
  };
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (ROWS > 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < V; ++i) sums[threadIdx.x * V + i] = dw[c][i];
      __syncthreads();
      for (int k = threadIdx.x; k < THREADS * V; k += blockDim.x) {
        float sum = 0.f;
        for (int r = 0; r < ROWS; ++r) sum += sums[r * THREADS * V + k];
        const int piece = (c * THREADS + k / V) * V;
        if (own<MODE>(k % V, piece_skip<MODE, V>(piece, cols), cols)) write(piece_begin<MODE, V>(piece, cols) + k % V, sum);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (c < C - 1 || own<MODE>(i, skip, cols)) write(at[c] + i, dw[c][i]);
    }
  }
}

// Rows that no workgroup's registers hold are read up to three times, from the cache the second and third time.
template <int TYPE, int PTYPE, bool BITS8>
__global__ __launch_bounds__(kNormLongThreads) void rms_norm_long_kernel(
    const void* __restrict__ x_, int64_t ldx, const void* __restrict__ residual_, int64_t ldr, const void* __restrict__ w,
    void* __restrict__ y_, const Bits8 bits8, void* __restrict__ h_, float* __restrict__ rstd_out, int64_t first, int cols, float eps) {
  typedef Elements<TYPE> E;
  typedef typename E::bits bits;
  constexpr int V = E::kVec, STEP = kNormLongThreads * V;
  __shared__ float slots[2][kNormLongThreads / 64];
  const int64_t row = first + blockIdx.x;
  const int t = threadIdx.x;
  const bits* const x = static_cast<const bits*>(x_) + row * ldx;
  const bits* const residual = residual_ != nullptr ? static_cast<const bits*>(residual_) + row * ldr : nullptr;
  bits* const h = residual != nullptr ? static_cast<bits*>(h_) + row * cols : nullptr;
  float squares = 0.f;
  for (int64_t at = t * V; at < cols; at += STEP) {
    const int n = (int)(cols - at);
    float f[V];
    E::unpack(E::load(x + at, n), f);
    if (residual != nullptr) {
      float a[V];
      E::unpack(E::load(residual + at, n), a);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] += a[i];
      const u32x4 sum = E::pack(f);
      E::store(h + at, n, sum);
      E::unpack(sum, f);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) squares = __builtin_fmaf(f[i], f[i], squares);
  }
  const float rstd = 1.0f / sqrtf(row_sum<kNormLongThreads>(squares, slots[0]) / (float)cols + eps);
  if (rstd_out != nullptr && t == 0) rstd_out[row] = rstd;
  const bits* const rows = residual != nullptr ? h : x;   // a thread reads what it has written
  const auto normed = [&](int64_t at, float (&f)[V]) {
    const int n = (int)(cols - at);
    Parameters<TYPE, PTYPE> pw;
    pw.load(w, (int)at, n);
    float fw[V];
    E::unpack(E::load(rows + at, n), f);
    pw.get(fw);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = f[i] * rstd * fw[i];
  };
  if constexpr (BITS8) {
    float scale = bits8.scale != nullptr ? *bits8.scale : 0.f;
    if (bits8.scale == nullptr || bits8.amax != nullptr) {
      float most = 0.f;
      for (int64_t at = t * V; at < cols; at += STEP) {
        float f[V];
        normed(at, f);
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (i < cols - at) most = amax_step(most, f[i]);
      }
      most = row_max<kNormLongThreads>(most, slots[1]);
      if (bits8.scale == nullptr) {
        most = fmaxf(most, kLeast);
        scale = most_of(bits8.fmt) / most;
        if (t == 0) bits8.scale_inv[row] = most / most_of(bits8.fmt);
      } else if (t == 0 && !(__builtin_nontemporal_load(bits8.amax) >= most)) {
        atomic_max_nonneg(bits8.amax, most);
      }
    }
    for (int64_t at = t * V; at < cols; at += STEP) {
      float f[V];
      normed(at, f);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] *= scale;
      store8<V>(bits8.q + row * cols + at, (int)(cols - at < V ? cols - at : V), f, bits8.fmt);
    }
  } else {
    bits* const y = static_cast<bits*>(y_) + row * cols;
    for (int64_t at = t * V; at < cols; at += STEP) {
      float f[V];
      normed(at, f);
      E::store(y + at, (int)(cols - at), E::pack(f));
    }
  }
}

template <int TYPE, int PTYPE>
__global__ __launch_bounds__(kNormLongThreads) void rms_norm_long_dx_kernel(
    const void* __restrict__ dy_, int64_t ldy, const void* __restrict__ dh_, int64_t ldd, const void* __restrict__ h_, int64_t ldh,
    const void* __restrict__ w, const float* __restrict__ rstd_in, void* __restrict__ dx_, int64_t first, int cols) {
  typedef Elements<TYPE> E;
  typedef typename E::bits bits;
  constexpr int V = E::kVec, STEP = kNormLongThreads * V;
  __shared__ float slots[kNormLongThreads / 64];
  const int64_t row = first + blockIdx.x;
  const int t = threadIdx.x;
  const bits* const h = static_cast<const bits*>(h_) + row * ldh;
  const bits* const dy = static_cast<const bits*>(dy_) + row * ldy;
  const bits* const dh = dh_ != nullptr ? static_cast<const bits*>(dh_) + row * ldd : nullptr;
  bits* const dx = static_cast<bits*>(dx_) + row * cols;
  const float rstd = rstd_in[row];
  float s = 0.f, c = 0.f;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    for (int64_t at = t * V; at < cols; at += STEP) {
      const int n = (int)(cols - at);
      Parameters<TYPE, PTYPE> pw;
      pw.load(w, (int)at, n);
      float fh[V], fy[V], fw[V], fd[V] = {};
      E::unpack(E::load(h + at, n), fh);
      E::unpack(E::load(dy + at, n), fy);
      if (pass == 1 && dh != nullptr) E::unpack(E::load(dh + at, n), fd);
      pw.get(fw);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float z = i < n ? fh[i] * rstd : 0.f, g = fy[i] * fw[i];   // (behind the row's end an infinite rstd times zero)
        s = __builtin_fmaf(g, z, s);
        fd[i] = __builtin_fmaf(rstd, g - z * c, fd[i]);
      }
      if (pass == 1) E::store(dx + at, n, E::pack(fd));
    }
    if (pass == 0) c = row_sum<kNormLongThreads>(s, slots) / (float)cols;
  }
}

// The weight's gradient: a thread keeps one piece of the columns for a slice of the rows.
template <int TYPE>
__global__ __launch_bounds__(256) void rms_norm_long_weight_kernel(
    const void* __restrict__ dy_, int64_t ldy, const void* __restrict__ h_, int64_t ldh, const float* __restrict__ rstd_in,
    float* __restrict__ part, int rows, int cols) {
  typedef Elements<TYPE> E;
  typedef typename E::bits bits;
  constexpr int V = E::kVec;
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
  if (at >= cols) return;
  const int n = (int)(cols - at);
  float dw[V] = {};
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const float rstd = rstd_in[row];
    float fh[V], fy[V];
    E::unpack(E::load(static_cast<const bits*>(h_) + row * ldh + at, n), fh);
    E::unpack(E::load(static_cast<const bits*>(dy_) + row * ldy + at, n), fy);
#pragma unroll
    for (int i = 0; i < V; ++i) dw[i] = __builtin_fmaf(fy[i], fh[i] * rstd, dw[i]);
  }
  float* const out = part + (int64_t)blockIdx.y * cols + at;
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < n) out[i] = dw[i];
}

// Forward, 4 pieces to a thread, as in the layer norm; 2 of aligned rows in 8 bits, whose conversions want more wavefronts (4096 x 4096, bf16,
// 22.8 us, with 4 pieces 26.6; 256 rows 5.2 and 6.1; 16384 rows 74.0 and 76.3; but 16384 x 4093 91.8 and 79.2).
Shape forward_shape(int cols, int type, bool two) {
  const int pieces = pieces_of(cols, type);
  Shape s = shape_of(pieces, two ? 2 : 4, 8, 4);
  if (s.lanes == 0) s = shape_of(pieces, 4, 8, 4);
  return s.lanes != 0 ? s : widest(cols, type);
}
// Backward, 2, or 1 of aligned rows that leave a workgroup two of them (16384 x 4096, bf16, 91.7 us, with 2 pieces 93.7; 65536 x 1024 90.7 and
// 94.7; 256 x 4096 9.1 and 10.6; 4096 x 4096 30.2 and 29.5; 64 x 8192, one row, 10.9 and 9.9).  The widest rows of fp32 spill some registers
// and are ahead all the same (4096 x 16384 208 us, by the kernels for longer rows 325; 4096 x 10000 139 and 202).
Shape backward_shape(int cols, int type, bool aligned) {
  const int pieces = pieces_of(cols, type);
  const Shape one = shape_of(pieces, 1, kNormWaves / 2, 2), s = shape_of(pieces, 2, kNormWaves, 2);
  if (aligned && one.lanes == 64 && kBackwardThreads % one.threads() == 0) return one;
  return s.lanes != 0 ? s : widest(cols, type);
}
// Workgroups of a backward pass: partial sums that its weight's gradient has.  Of aligned rows no fewer than of others.
int backward_blocks(int64_t rows, int cols, int type, bool aligned) {
  const Shape s = backward_shape(cols, type, aligned);
  if (s.lanes == 0) return (int)std::min<int64_t>(rows, 64);
  const int blocks = ceil_div(rows, kBackwardThreads / s.threads());
  return blocks <= kBackwardAlone ? std::min(blocks, 1) : std::min(blocks, kBackwardBlocks);
}

int check_rms(int64_t rows, int cols, int type, int param_type) {
  if (!known_type(type) || (param_type != type && param_type != FP8GMM_TYPE_FP32)) return FP8GMM_ERR_BAD_FORMAT;
  // a row's offsets in 32 bits, with room for the last piece's
  if (rows < 0 || rows > INT32_MAX || cols < 1 || cols > (1 << 30)) return FP8GMM_ERR_BAD_SHAPE;
  return FP8GMM_OK;
}

struct Rows {
  const void* x;
  int64_t ldx;
  const void* residual;
  int64_t ldr;
  const void* weight;
  void* h;
  int64_t rows;
  int cols;
  float eps;
  int type, param_type;
};

// What both forward passes ask of their rows; 1: nothing to do
int check_forward(const Rows& a) {
  const int rc = check_rms(a.rows, a.cols, a.type, a.param_type);
  if (rc != FP8GMM_OK) return rc;
  if (a.ldx < a.cols || (a.residual != nullptr && a.ldr < a.cols)) return FP8GMM_ERR_BAD_SHAPE;
  if (!(a.eps >= 0.f)) return FP8GMM_ERR_BAD_ARGUMENT;
  if (a.rows == 0) return 1;
  if (a.x == nullptr || a.weight == nullptr || (a.residual != nullptr && a.h == nullptr)) return FP8GMM_ERR_NULL_POINTER;
  return FP8GMM_OK;
}

template <int KIND>
int launch_forward(const Rows& a, void* y, const Bits8& bits8, float* rstd, hipStream_t s) {
  constexpr bool BITS8 = KIND == kBits8;
  const bool aligned = whole(a.x, a.ldx, a.cols, a.type) && (a.residual == nullptr || (whole(a.residual, a.ldr, a.cols, a.type) &&
                       whole(a.h, a.cols, a.cols, a.type))) && (BITS8 || whole(y, a.cols, a.cols, a.type));
  const Shape shape = forward_shape(a.cols, a.type, BITS8 && aligned);
  const int threads = shape.lanes == 0 ? 0 : std::max(shape.threads(), kForwardThreads / shape.threads() * shape.threads());
  const bool streaming = streams(a.rows, a.cols, a.type);
  const auto blocks = [&] {
    const int groups = ceil_div(a.rows, threads / shape.threads()), all = kForwardAll / threads;   // rows that a workgroup takes at a time
    return std::min(groups, !BITS8 ? kForwardFour * all : groups > kForwardTurns * all ? kForwardMore * all : all);
  };
  const int mode = mode_of(a.cols, a.type, shape.lanes, aligned, streaming);
  bool known = true;   // a row's share of the registers that no launch below is for would leave the results unwritten
  with_types(a.type, a.param_type, [&](auto tc, auto pc) {
    constexpr int T = decltype(tc)::value, P = decltype(pc)::value;
#define FP8GMM_LAUNCH(LANES, C, MOST)                                                                                                \
  if (shape.lanes == LANES && shape.pieces == C && threads <= MOST) {                                                                \
    auto* kernel = mode == kEdge         ? &rms_norm_kernel<T, P, LANES, C, kEdge, MOST, KIND>                                      \
                   : mode == kEdgeStream ? &rms_norm_kernel<T, P, LANES, C, kEdgeStream, MOST, KIND>                                \
                                         : &rms_norm_kernel<T, P, LANES, C, LANES == 64 ? kWhole : C == 1 ? kShort : kEdge, MOST, KIND>; \
    hipLaunchKernelGGL(kernel, dim3(blocks()), dim3(threads), 0, s, a.x, a.ldx, a.residual, a.ldr, a.weight, y, bits8, a.h, rstd,     \
                       (int)a.rows, a.cols, a.eps, shape.waves, streaming);                                                          \
  } else
    FP8GMM_LAUNCH(16, 1, 256)
    FP8GMM_LAUNCH(16, 2, 256)
    FP8GMM_LAUNCH(16, 3, 256)
    FP8GMM_LAUNCH(16, 4, 256)
    FP8GMM_LAUNCH(64, 2, 512)   // (one piece to each of 64 lanes is 16 lanes' share)
    FP8GMM_LAUNCH(64, 3, 512)
    FP8GMM_LAUNCH(64, 4, 512)
    if constexpr (T == FP8GMM_TYPE_FP32) {
      FP8GMM_LAUNCH(64, 4, 1024) known = shape.lanes == 0;
    } else {
      known = shape.lanes == 0;
    }
#undef FP8GMM_LAUNCH
    for (int64_t r0 = 0; shape.lanes == 0 && r0 < a.rows; r0 += kNormSlab)
      hipLaunchKernelGGL((rms_norm_long_kernel<T, P, BITS8>), dim3((unsigned)std::min<int64_t>(kNormSlab, a.rows - r0)),
                         dim3(kNormLongThreads), 0, s, a.x, a.ldx, a.residual, a.ldr, a.weight, y, bits8, a.h, rstd, r0, a.cols, a.eps);
  });
  if (!known) return FP8GMM_ERR_LAUNCH;
  return hipGetLastError() == hipSuccess ? FP8GMM_OK : FP8GMM_ERR_LAUNCH;
}

}  // namespace
}  // namespace fp8gmm

extern "C" {

int fp8gmm_rms_norm(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight, void* y, void* h, float* rstd,
                    int64_t rows, int cols, float eps, int type, int param_type, void* stream) {
  using namespace fp8gmm;
  const Rows a = {x, ldx, residual, ldr, weight, h, rows, cols, eps, type, param_type};
  const int rc = check_forward(a);
  if (rc != FP8GMM_OK) return rc == 1 ? FP8GMM_OK : rc;
  if (y == nullptr) return FP8GMM_ERR_NULL_POINTER;
  return residual != nullptr ? launch_forward<kSums>(a, y, Bits8{}, rstd, static_cast<hipStream_t>(stream))
                             : launch_forward<kRows>(a, y, Bits8{}, rstd, static_cast<hipStream_t>(stream));
}

int fp8gmm_rms_norm_fp8(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight, void* q, void* h,
                        const float* scale, float* amax, float* scale_inv, int64_t rows, int cols, float eps, int type, int param_type,
                        int fmt, void* stream) {
  using namespace fp8gmm;
  const Rows a = {x, ldx, residual, ldr, weight, h, rows, cols, eps, type, param_type};
  const int rc = check_forward(a);
  if (rc < 0) return rc;
  if (fmt != FP8GMM_E4M3 && fmt != FP8GMM_E5M2) return FP8GMM_ERR_BAD_FORMAT;
  if (rc == 1) return FP8GMM_OK;
  if ((scale == nullptr) == (scale_inv == nullptr) || (scale == nullptr && amax != nullptr)) return FP8GMM_ERR_BAD_ARGUMENT;
  if (q == nullptr) return FP8GMM_ERR_NULL_POINTER;
  return launch_forward<kBits8>(a, nullptr, Bits8{static_cast<uint8_t*>(q), scale, amax, scale_inv, fmt}, nullptr,
                              static_cast<hipStream_t>(stream));
}

size_t fp8gmm_rms_norm_workspace_bytes(int64_t rows, int cols, int type) {
  using namespace fp8gmm;
  if (check_rms(rows, cols, type, type) != FP8GMM_OK) return 0;
  return (size_t)backward_blocks(rows, cols, type, true) * cols * sizeof(float);
}

int fp8gmm_rms_norm_backward(const void* dy, int64_t ldy, const void* dh, int64_t ldd, const void* h, int64_t ldh, const void* weight,
                             const float* rstd, void* dx, void* dweight, int64_t rows, int cols, int type, int param_type,
                             void* workspace, size_t workspace_bytes, void* stream) {
  using namespace fp8gmm;
  const int rc = check_rms(rows, cols, type, param_type);
  if (rc != FP8GMM_OK) return rc;
  if (ldy < cols || ldh < cols || (dh != nullptr && ldd < cols)) return FP8GMM_ERR_BAD_SHAPE;
  if (rows > 0 && (dy == nullptr || h == nullptr || weight == nullptr || rstd == nullptr)) return FP8GMM_ERR_NULL_POINTER;
  if (dweight != nullptr && rows > 0) {
    if (workspace == nullptr) return FP8GMM_ERR_NULL_POINTER;
    if (workspace_bytes < fp8gmm_rms_norm_workspace_bytes(rows, cols, type)) return FP8GMM_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return FP8GMM_ERR_ALIGNMENT;
  }
  if (dweight == nullptr && (dx == nullptr || rows == 0)) return FP8GMM_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  float* const part = dweight != nullptr ? static_cast<float*>(workspace) : nullptr;
  const bool aligned = whole(h, ldh, cols, type) && whole(dy, ldy, cols, type) && (dh == nullptr || whole(dh, ldd, cols, type)) &&
                       (dx == nullptr || whole(dx, cols, cols, type));
  const int blocks = backward_blocks(rows, cols, type, aligned);
  const Shape shape = backward_shape(cols, type, aligned);
  const bool streaming = streams(rows, cols, type);
  const int mode = mode_of(cols, type, shape.lanes, aligned, streaming && type == FP8GMM_TYPE_FP32);
  bool known = true;
  with_types(type, param_type, [&](auto tc, auto pc) {
    constexpr int T = decltype(tc)::value, P = decltype(pc)::value;
    constexpr int kStreamed = T == FP8GMM_TYPE_FP32 ? kEdgeStream : kEdge;
    if (rows > 0) {
#define FP8GMM_LAUNCH(LANES, C)                                                                                                      \
  if (shape.lanes == LANES && shape.pieces == C) {                                                                                   \
    auto* kernel = mode == kEdge         ? &rms_norm_backward_kernel<T, P, LANES, C, kEdge>                                          \
                   : mode == kEdgeStream ? &rms_norm_backward_kernel<T, P, LANES, C, kStreamed>                                      \
                                         : &rms_norm_backward_kernel<T, P, LANES, C, LANES == 64 ? kWhole : C == 1 ? kShort : kEdge>; \
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kBackwardThreads / shape.threads() * shape.threads()), 0, s, dy, ldy, dh, ldd, h, ldh, \
                       weight, rstd, dx, part, dweight, (int)rows, cols, shape.waves, streaming);                                    \
  } else
      FP8GMM_LAUNCH(16, 1)
      FP8GMM_LAUNCH(16, 2)
      FP8GMM_LAUNCH(64, 1)
      FP8GMM_LAUNCH(64, 2)
      if constexpr (T == FP8GMM_TYPE_FP32) {
        FP8GMM_LAUNCH(64, 4) known = shape.lanes == 0;
      } else {
        known = shape.lanes == 0;
      }
#undef FP8GMM_LAUNCH
      if (shape.lanes == 0) {
        for (int64_t r0 = 0; dx != nullptr && r0 < rows; r0 += kNormSlab)
          hipLaunchKernelGGL((rms_norm_long_dx_kernel<T, P>), dim3((unsigned)std::min<int64_t>(kNormSlab, rows - r0)),
                             dim3(kNormLongThreads), 0, s, dy, ldy, dh, ldd, h, ldh, weight, rstd, dx, r0, cols);
        if (dweight != nullptr)
          hipLaunchKernelGGL((rms_norm_long_weight_kernel<T>), dim3(ceil_div(cols, 256 * Elements<T>::kVec), blocks), dim3(256), 0, s, dy,
                             ldy, h, ldh, rstd, part, (int)rows, cols);
      }
    }
    if (dweight != nullptr && (blocks != 1 || shape.lanes == 0))
      launch_norm_params<P>(part, blocks, 1, cols, dweight, nullptr, s);
  });
  if (!known) return FP8GMM_ERR_LAUNCH;
  return hipGetLastError() == hipSuccess ? FP8GMM_OK : FP8GMM_ERR_LAUNCH;
}

}  // extern "C"
