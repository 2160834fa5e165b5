// Layer norm over the columns of rows of bf16, fp16 or fp32, and its backward pass, for gfx950: the norm in front of a
// routed layer (moe.py, layer_norm=True).
//
//   m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), z = (x - m) r, y = z w + b
//   g = dy w, dx = r (g - mean(g) - z mean(g z)), dw = sum over rows of dy z, db = sum over rows of dy
//
// Bound by memory: x and y pass once, and in the backward pass x, dy and dx.  A row stays in the registers of the threads
// that share it, so nothing is read twice, and the squares are taken around a mean that is already known (no cancellation where
// a row lies far off zero).  The statistics are kept in fp32 for the backward pass, m and r of every row; every sum is taken in
// fp32, and a result is rounded once.
//
// From call to call, with so many buffers in turn that the caches hold nothing of the next call's (1.3 GB of rows or more), in us
// and TB/s of what has to pass.  The figures below are taken in the same way.
//                          forward        backward
//   1 x 4096, bf16         4.4            8.0            one launch each, out of the caches
//   1024 x 4096, bf16      5.8            17             out of the caches
//   16384 x 4096, bf16     49     5.5     73     5.5     forward 43 where the caches hold a part of the rows
//   16384 x 4093, bf16     51     5.3     81     4.9     rows that begin at any element
//   65536 x 2048, fp32     185    5.8     259    6.2
//   8192 x 16384, bf16     101    5.3     157    5.1     the longest rows of 16 bits that stay in registers
//   262144 x 256, bf16     47     5.8     79     5.1     four rows to a wavefront
// A large copy reaches 5.3 here.
#include <algorithm>
#include <type_traits>

#include "elements.h"

namespace fp8gmm {
namespace {

constexpr int kBackwardThreads = 1024;   // of a workgroup of the backward pass: as many rows at a time as fit, since every workgroup
constexpr int kBackwardBlocks = 256;     // leaves one partial sum of the parameters' gradients in memory; one per compute unit
constexpr int kNormLongThreads = 1024;
constexpr int kNormSlab = 1 << 16;   // rows of a launch with a workgroup to a row, 2 GB at least: a grid has fewer than 2^32 threads

// So many turns of one workgroup take less than a second launch for the sums of several: 32 x 1024, bf16, 2 turns: 8.4 us, by two
// workgroups 8.8; 64 x 1024, 4 turns: 11.5 and 9.0; 16 x 4096, 4 turns: 14.2 and 10.7.
constexpr int kBackwardAlone = 2;
constexpr int kNormWaves = 16;           // the most wavefronts that share a row
constexpr int kForwardThreads = 256;     // of a workgroup of the forward pass, where a row needs no more
// Threads of its launch: what the compute units hold at a time, which go on to other rows; three times that where they would go on
// more than five times (24576 x 4096, bf16, 6 turns: 73 us, with three times as many 67, with all rows at once 77; 65536 x 2048, 8
// turns, 96, 88 and 99; fp32, 16 turns, 192, 185 and 182; 24576 x 2048, 3 turns, 36 and 40).  Not everywhere: 16384 x 4096, 4 turns, 49,
// with twice as many 46; 8192 x 16384, 8 turns, 92, with three times as many 101.
constexpr int kForwardAll = 256 * 2048, kForwardTurns = 5, kForwardMore = 3;

// The sum over the THREADS threads of a row, the same in all of them.  `slot`: THREADS / 64 floats of LDS per row that nobody
// uses before the next barrier but one.
template <int THREADS>
__device__ __forceinline__ float row_sum(float v, float* slot) {
  v = lanes_sum<64>(v);
  if (threadIdx.x % 64 == 0) slot[threadIdx.x / 64] = v;
  __syncthreads();
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < THREADS / 64; ++i) sum += slot[i];
  return sum;
}

// How the pieces of a row are reached, without a branch where that can be: the compiler then knows how many accesses are under
// way, and waits for the loads of the next row alone and not for the stores behind them.
//   kWhole  rows of whole pieces on 16 bytes: through a buffer descriptor of the row.  What lies behind its end, or belongs to no
//           row, reads as zeros and is not stored.
//   kEdge   other rows of at least one piece, at any element: the last piece ends where the row ends and begins inside the piece
//           before it, and threads behind the end have the last piece too.  What a thread has twice it leaves out of the sums and
//           stores all the same: the same bits to the same place.
//   kShort  shorter rows, element by element.
//   kEdgeStream  kEdge with its results written with the streaming hint: the compiler makes one store, without it, of two that are
//           chosen from at run time
enum { kWhole, kEdge, kEdgeStream, kShort };
constexpr bool is_edge(int mode) { return mode == kEdge || mode == kEdgeStream; }

// Where a thread's piece begins that begins at `at`, and how many of its elements are not its own
template <int MODE, int V>
__device__ __forceinline__ int piece_begin(int at, int cols) { return is_edge(MODE) ? min(at, cols - V) : at; }
template <int MODE, int V>
__device__ __forceinline__ int piece_skip(int at, int cols) {
  return is_edge(MODE) ? min(at - piece_begin<MODE, V>(at, cols), V) : at < cols ? 0 : V;
}
// Whether element i counts: of kShort, the row's first piece only
template <int MODE>
__device__ __forceinline__ bool own(int i, int skip, int cols) { return i >= skip && (MODE != kShort || i < cols); }

template <int TYPE, int MODE>
struct RowAccess {
  typedef Elements<TYPE> E;
  typedef typename E::bits bits;
  bits* p;
  __amdgpu_buffer_rsrc_t r;
  int cols;
  __device__ __forceinline__ RowAccess(const void* base, int64_t row, int64_t rows, int64_t pitch, int n) {
    const bool live = row < rows;
    cols = live || is_edge(MODE) ? n : 0;
    p = const_cast<bits*>(static_cast<const bits*>(base)) + (live ? row : rows - 1) * pitch;   // kEdge: the last row once more
    if constexpr (MODE == kWhole) r = make_rsrc(p, (uint32_t)cols * E::kBytes);
  }
  template <bool STREAM>
  __device__ __forceinline__ u32x4 load(int at) const {
    if constexpr (MODE == kWhole) return STREAM ? buf_load16_stream(r, (uint32_t)at * E::kBytes) : buf_load16(r, (uint32_t)at * E::kBytes);
    else return E::template load<STREAM>(p + at, is_edge(MODE) ? E::kVec : cols - at);
  }
  __device__ __forceinline__ void store(int at, u32x4 v, bool stream) const {
    if constexpr (MODE == kWhole) stream ? buf_store16_stream(v, r, (uint32_t)at * E::kBytes) : buf_store16(v, r, (uint32_t)at * E::kBytes);
    else E::template store<MODE == kEdgeStream>(p + at, is_edge(MODE) ? E::kVec : cols - at, v);
  }
};

// A workgroup takes ROWS rows at a time, THREADS threads to a row and C pieces to a thread, and goes on to other rows by the grid:
// the next rows are loaded before the statistics of the present ones are shared, and the parameters stay in registers.
// The wavefronts of a row meet once: each brings its sum and the squares around its own mean, which combine to those around the
// row's, sum (M2_w + n_w (m_w - m)^2).
template <int TYPE, int PTYPE, int LANES, int C, int MODE, int MOST>
__global__ __launch_bounds__(MOST) void layer_norm_kernel(
    const void* __restrict__ x_, int64_t ldx, const void* __restrict__ w, const void* __restrict__ b, void* __restrict__ y_,
    float* __restrict__ mean_out, float* __restrict__ rstd_out, int rows, int cols, float eps, int waves, bool stream) {
  typedef Elements<TYPE> E;
  constexpr int V = E::kVec;
  __shared__ float slots[2][2][kNormWaves][kNormWaves];
  const int THREADS = LANES * waves, ROWS = blockDim.x / THREADS;
  int group = threadIdx.x / THREADS;
  if constexpr (LANES == 64) group = __builtin_amdgcn_readfirstlane(group);
  const int t = threadIdx.x - group * THREADS;
  int at[C];
#pragma unroll
  for (int c = 0; c < C; ++c) at[c] = (c * THREADS + t) * V;
  const int skip = piece_skip<MODE, V>(at[C - 1], cols);   // the pieces before the last one are there in whole
  at[C - 1] = piece_begin<MODE, V>(at[C - 1], cols);
  u32x4 next[C];
  const auto load = [&](int64_t row) {
    const RowAccess<TYPE, MODE> from(x_, row, rows, ldx, cols);
#pragma unroll
    for (int c = 0; c < C; ++c) next[c] = from.template load<false>(at[c]);
  };
  const int64_t stride = (int64_t)gridDim.x * ROWS;
  int64_t row = (int64_t)blockIdx.x * ROWS + group;
  load(row);
  Parameters<TYPE, PTYPE> pw[C], pb[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    pw[c].load(w, at[c], cols - at[c]);
    if (b != nullptr) pb[c].load(b, at[c], cols - at[c]);
  }
  // elements of a row's wavefront (group of 16 lanes): its piece c covers columns from (c THREADS + first lane) V on
  const auto held = [&](int wave) {
    int n = 0;
#pragma unroll
    for (int c = 0; c < C; ++c) n += min(max(cols - (c * THREADS + wave * LANES) * V, 0), LANES * V);
    return (float)n;
  };
  const int wave = LANES == 64 ? __builtin_amdgcn_readfirstlane(t / 64) : 0;
  const float count = (float)cols, mine = held(wave);
  const int peer = threadIdx.x % 16;   // the wavefront whose share this lane takes up where they meet
  const float peer_count = peer < waves ? held(peer) : 0.f;
  int turn = 0;
  for (int64_t first = (int64_t)blockIdx.x * ROWS; first < rows; first += stride, row += stride, turn ^= 1) {
    u32x4 x[C];
#pragma unroll
    for (int c = 0; c < C; ++c) x[c] = next[c];
    if (first + stride < rows) load(row + stride);
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float f[V];
      E::unpack(x[c], f);
#pragma unroll
      for (int i = 0; i < V; ++i) sum += !is_edge(MODE) || c < C - 1 || i >= skip ? f[i] : 0.f;
    }
    sum = lanes_sum<LANES>(sum);
    float mean = sum / mine, squares = 0.f;   // every wavefront of a row has some of it
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float f[V];
      E::unpack(x[c], f);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = c < C - 1 || own<MODE>(i, skip, cols) ? f[i] - mean : 0.f;
        squares = __builtin_fmaf(d, d, squares);
      }
    }
    squares = lanes_sum<LANES>(squares);
    if (LANES == 64 && waves > 1) {   // the other turn's slots are read before the next barrier
      if (threadIdx.x % 64 == 0) {
        slots[turn][0][group][wave] = mean;
        slots[turn][1][group][wave] = squares;
      }
      __syncthreads();
      const float m = peer < waves ? slots[turn][0][group][peer] : 0.f, q = peer < waves ? slots[turn][1][group][peer] : 0.f;
      mean = lanes_sum<16>(peer_count * m) / count;
      squares = lanes_sum<16>(__builtin_fmaf(peer_count * (m - mean), m - mean, q));
    }
    const float rstd = 1.0f / sqrtf(squares / count + eps);
    if (mean_out != nullptr && t == 0 && row < rows) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
    const RowAccess<TYPE, MODE> y(y_, row, rows, cols, cols);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float f[V], fw[V], fb[V];
      E::unpack(x[c], f);
      pw[c].get(fw);
      if (b != nullptr) pb[c].get(fb);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = __builtin_fmaf((f[i] - mean) * rstd, fw[i], b != nullptr ? fb[i] : 0.f);
      y.store(at[c], E::pack(f), stream);
    }
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

// The backward pass in the same way, with the sums of dy z and dy for the columns of its threads.  `part`: [workgroup][2][cols], the
// second without a bias left out; NULL where the parameters take no gradients.  dx may be NULL.  A single workgroup writes the
// gradients themselves.
template <int TYPE, int PTYPE, int LANES, int C, int MODE>
__global__ __launch_bounds__(kBackwardThreads) void layer_norm_backward_kernel(
    const void* __restrict__ dy_, int64_t ldy, const void* __restrict__ x_, int64_t ldx, const void* __restrict__ w,
    const float* __restrict__ mean_in, const float* __restrict__ rstd_in, void* __restrict__ dx_, float* __restrict__ part,
    void* __restrict__ dweight, void* __restrict__ dbias, int rows, int cols, int waves, bool stream) {
  typedef Elements<TYPE> E;
  constexpr int V = E::kVec;
  __shared__ float slots[2][2][kNormWaves][kNormWaves];
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
  float dw[C][V] = {}, db[C][V] = {};
  u32x4 nx[C], ny[C];
  float nm, nr;
  const auto load = [&](int64_t row) {
    const RowAccess<TYPE, MODE> x(x_, row, rows, ldx, cols), y(dy_, row, rows, ldy, cols);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      nx[c] = x.template load<true>(at[c]);
      ny[c] = y.template load<true>(at[c]);
    }
    nm = row < rows ? mean_in[row] : 0.f;
    nr = row < rows ? rstd_in[row] : 0.f;
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
    if (first + stride < rows) load(row + stride);
    float s1 = 0.f, s2 = 0.f;
    if (!is_edge(MODE) || row < rows) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float fx[V], fy[V], fw[V];
        E::unpack(x[c], fx);
        E::unpack(y[c], fy);
        pw[c].get(fw);
        float u1 = 0.f, u2 = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if (is_edge(MODE) && c == C - 1 && i < skip) fy[i] = 0.f;   // elsewhere they are zeros
          const float z = MODE != kShort || i < cols ? (fx[i] - mean) * rstd : 0.f, g = fy[i] * fw[i];
          u1 += g;
          u2 = __builtin_fmaf(g, z, u2);
          dw[c][i] = __builtin_fmaf(fy[i], z, dw[c][i]);
          db[c][i] += fy[i];
        }
        // nothing of a piece behind the end, whose zeros have a z of minus the mean times rstd, be that infinite
        s1 += c < C - 1 || skip < V ? u1 : 0.f;
        s2 += c < C - 1 || skip < V ? u2 : 0.f;
      }
    }
    if (dx_ == nullptr) continue;
    s1 = lanes_sum<LANES>(s1);
    s2 = lanes_sum<LANES>(s2);
    if (LANES == 64 && waves > 1) {   // the other turn's slots are read before the next barrier
      if (threadIdx.x % 64 == 0) {
        slots[turn][0][group][wave] = s1;
        slots[turn][1][group][wave] = s2;
      }
      __syncthreads();
      s1 = lanes_sum<16>(peer < waves ? slots[turn][0][group][peer] : 0.f);
      s2 = lanes_sum<16>(peer < waves ? slots[turn][1][group][peer] : 0.f);
    }
    if (is_edge(MODE) && row >= rows) continue;   // its sums leave no row out
    const float c1 = -rstd * (s1 / (float)cols), c2 = -rstd * (s2 / (float)cols);
    const RowAccess<TYPE, MODE> dx(dx_, row, rows, cols, cols);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float fx[V], fy[V], fw[V];
      E::unpack(x[c], fx);
      E::unpack(y[c], fy);
      pw[c].get(fw);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float z = (fx[i] - mean) * rstd;
        fx[i] = __builtin_fmaf(fy[i], fw[i] * rstd, __builtin_fmaf(z, c2, c1));
      }
      dx.store(at[c], E::pack(fx), stream);
    }
  }
  if (part == nullptr) return;
  // the workgroup's rows together, in their order: THREADS * V columns at a time
  float* const out = part + (int64_t)blockIdx.x * 2 * cols;
  const auto write = [&](int which, int64_t col, float sum) {
    typedef Elements<PTYPE> P;
    void* const to = which == 0 ? dweight : dbias;
    if (gridDim.x > 1) out[(int64_t)which * cols + col] = sum;
    else if (to != nullptr) static_cast<typename P::bits*>(to)[col] = P::pack1(sum);
  };
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      if (which == 1 && dbias == nullptr) continue;
      if (ROWS > 1) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) sums[threadIdx.x * V + i] = which == 0 ? dw[c][i] : db[c][i];
        __syncthreads();
        for (int k = threadIdx.x; k < THREADS * V; k += blockDim.x) {
          float sum = 0.f;
          for (int r = 0; r < ROWS; ++r) sum += sums[r * THREADS * V + k];
          const int piece = (c * THREADS + k / V) * V;
          if (own<MODE>(k % V, piece_skip<MODE, V>(piece, cols), cols))
            write(which, piece_begin<MODE, V>(piece, cols) + k % V, sum);
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (c < C - 1 || own<MODE>(i, skip, cols)) write(which, at[c] + i, which == 0 ? dw[c][i] : db[c][i]);
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
        // behind the row's end x is a zero, whose z is minus the mean times rstd, be that infinite
        const float z = i < n ? (fx[i] - mean) * rstd : 0.f, g = fy[i] * fw[i];
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

// How a row is shared out: `lanes` * `waves` threads, `pieces` 16-byte pieces to each.  No lanes: longer than the registers of a
// workgroup hold.
struct Shape {
  int lanes, waves, pieces;
  int threads() const { return lanes * waves; }
};
int pieces_of(int cols, int type) { return ceil_div(cols, 16 / type_bytes(type)); }
// Up to `most` pieces to a thread, as few threads as that allows, and then as few pieces: a thread behind the row's end works for
// nothing.  `waves`: the most of them.  A row's first 64 * waves pieces are there, so that every wavefront has some of the row.
// `narrow`: the most pieces of a thread where 16 lanes have a row.  4 forward (262144 x 256, bf16, 70 us by 64 lanes, 47 so; 131072 x
// 384, 39.5 and 35.7; 131072 x 512, 48.6 and 46.7), 2 backward (262144 x 256, 87 and 79; with 3, 131072 x 384, 55 and 161: spills).
Shape shape_of(int pieces, int most, int waves, int narrow) {
  if (pieces <= 16 * narrow) return {16, 1, ceil_div(pieces, 16)};
  const int w = ceil_div(pieces, 64 * most);
  return w <= waves ? Shape{64, w, ceil_div(pieces, 64 * w)} : Shape{0, 0, 0};
}
// The longest rows that stay in registers have 4 pieces in each of 1024 threads, which fits fp32 alone: a 16-bit type has twice
// the elements and spills backward (4096 x 32768, bf16: 103 and 781 us forward and backward, by the kernels for longer rows 146 and
// 296; 4096 x 16384, fp32: 92 and 174, by those 142 and 287).
Shape widest(int cols, int type) {
  const int w = ceil_div(pieces_of(cols, type), 64 * 4);
  return type == FP8GMM_TYPE_FP32 && w <= kNormWaves ? Shape{64, w, 4} : Shape{0, 0, 0};
}
// Forward, 4 pieces to a thread: few barriers and many loads under way (65536 x 2048, fp32: 185 us, with 2 pieces 193; 8192 x 16384,
// bf16: 101 and 120; 16384 x 1536: 21.2 and 23.0; 16384 x 4093: 51 and 58, but 16384 x 4096 49 and 48).
Shape forward_shape(int cols, int type) {
  const Shape s = shape_of(pieces_of(cols, type), 4, 8, 4);
  return s.lanes != 0 ? s : widest(cols, type);
}
// Backward, 2: the sums of the parameters' gradients take registers as well.  Of fp32 rows of whole pieces 1, where that fills the
// workgroup (65536 x 2048: 259 us, with 2 pieces 273; 32768 x 4096: 261 and 272; but 32768 x 3000, in 12 wavefronts, 220 and 207,
// and 60001 x 2047, with edges, 271 and 260; 16384 x 4096, bf16: 73 and 73).
Shape backward_shape(int cols, int type, bool aligned) {
  const int pieces = pieces_of(cols, type);
  const Shape one = shape_of(pieces, 1, kNormWaves, 1), s = shape_of(pieces, 2, kNormWaves, 2);
  if (type == FP8GMM_TYPE_FP32 && aligned && s.lanes != 16 && one.lanes != 0 && kBackwardThreads % one.threads() == 0) return one;
  return s.lanes != 0 ? s : widest(cols, type);
}
// Rows of whole pieces on 16 bytes
bool whole(const void* p, int64_t pitch, int cols, int type) {
  const int pieces = 16 / type_bytes(type);
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && pitch % pieces == 0 && cols % pieces == 0;
}
// Whether a result is written with the streaming hint: one that outgrows the cache is not found there by whoever reads it.  With it
// and without: 16384 x 4096, bf16, forward 49 and 49 us, backward 73 and 78; 65536 x 2048, fp32, 185 and 191, 259 and 269; 24576 x
// 2048, bf16, 36.4 and 37.2, 55.5 and 57.9.
bool streams(int64_t rows, int cols, int type) { return rows * cols * type_bytes(type) > (int64_t)64 << 20; }
// A descriptor is a wavefront's, which has four rows where 16 lanes have one: these have edges, if empty ones.
int mode_of(int cols, int type, int lanes, bool aligned, bool stream_edges) {
  return cols < 16 / type_bytes(type) ? kShort : aligned && lanes == 64 ? kWhole : stream_edges ? kEdgeStream : kEdge;
}
// Workgroups of a backward pass: partial sums that its parameters' gradients have.  Of aligned rows no fewer than of others.
int backward_blocks(int rows, int cols, int type, bool aligned) {
  const Shape s = backward_shape(cols, type, aligned);
  if (s.lanes == 0) return std::min(rows, 64);
  const int blocks = ceil_div(rows, kBackwardThreads / s.threads());
  return blocks <= kBackwardAlone ? std::min(blocks, 1) : std::min(blocks, kBackwardBlocks);
}

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
  const Shape shape = forward_shape(cols, type);
  const int threads = shape.lanes == 0 ? 0 : std::max(shape.threads(), kForwardThreads / shape.threads() * shape.threads());
  const bool streaming = streams(rows, cols, type);
  const auto blocks = [&] {
    const int groups = ceil_div(rows, threads / shape.threads()), all = kForwardAll / threads;   // rows that a workgroup takes at a time
    return std::min(groups, groups > kForwardTurns * all ? kForwardMore * all : all);
  };
  const int mode = mode_of(cols, type, shape.lanes, whole(x, ldx, cols, type) && whole(y, cols, cols, type), streaming);
  bool known = true;   // a row's share of the registers that no launch below is for would leave y unwritten
  with_types(type, param_type, [&](auto tc, auto pc) {
    constexpr int T = decltype(tc)::value, P = decltype(pc)::value;
#define FP8GMM_LAUNCH(LANES, C, MOST)                                                                                         \
  if (shape.lanes == LANES && shape.pieces == C && threads <= MOST) {                                                         \
    auto* kernel = mode == kEdge         ? &layer_norm_kernel<T, P, LANES, C, kEdge, MOST>                                    \
                   : mode == kEdgeStream ? &layer_norm_kernel<T, P, LANES, C, kEdgeStream, MOST>                              \
                                         : &layer_norm_kernel<T, P, LANES, C, LANES == 64 ? kWhole : C == 1 ? kShort : kEdge, MOST>; \
    hipLaunchKernelGGL(kernel, dim3(blocks()), dim3(threads), 0, s, x, ldx, weight, bias, y, mean, rstd, (int)rows, cols, eps, \
                       shape.waves, streaming);                                                                               \
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
    for (int64_t r0 = 0; shape.lanes == 0 && r0 < rows; r0 += kNormSlab) {
      const int size = type_bytes(type);
      hipLaunchKernelGGL((layer_norm_long_kernel<T, P>), dim3((unsigned)std::min<int64_t>(kNormSlab, rows - r0)),
                         dim3(kNormLongThreads), 0, s, static_cast<const char*>(x) + r0 * ldx * size, ldx, weight, bias,
                         static_cast<char*>(y) + r0 * cols * size, mean != nullptr ? mean + r0 : nullptr,
                         rstd != nullptr ? rstd + r0 : nullptr, cols, eps);
    }
  });
  if (!known) return FP8GMM_ERR_LAUNCH;
  return hipGetLastError() == hipSuccess ? FP8GMM_OK : FP8GMM_ERR_LAUNCH;
}

size_t fp8gmm_layer_norm_workspace_bytes(int64_t rows, int cols, int type) {
  using namespace fp8gmm;
  if (check_norm(rows, cols, cols, type, type) != FP8GMM_OK) return 0;
  return (size_t)backward_blocks((int)rows, cols, type, true) * 2 * cols * sizeof(float);
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
  const bool aligned = whole(x, ldx, cols, type) && whole(dy, ldy, cols, type) && (dx == nullptr || whole(dx, cols, cols, type));
  const int blocks = backward_blocks((int)rows, cols, type, aligned), bias = dbias != nullptr;
  const Shape shape = backward_shape(cols, type, aligned);
  const bool streaming = streams(rows, cols, type);
  // of a 16-bit type, edges are written without the hint (16384 x 4093, bf16: 81 us, with it 79, but 76 and 80 where the caches hold a
  // part of the rows; 60001 x 2047, fp32: 282 and 260)
  const int mode = mode_of(cols, type, shape.lanes, aligned, streaming && type == FP8GMM_TYPE_FP32);
  bool known = true;
  with_types(type, param_type, [&](auto tc, auto pc) {
    constexpr int T = decltype(tc)::value, P = decltype(pc)::value;
    constexpr int kStreamed = T == FP8GMM_TYPE_FP32 ? kEdgeStream : kEdge;
    if (rows > 0) {
#define FP8GMM_LAUNCH(LANES, C)                                                                                               \
  if (shape.lanes == LANES && shape.pieces == C) {                                                                            \
    auto* kernel = mode == kEdge         ? &layer_norm_backward_kernel<T, P, LANES, C, kEdge>                                 \
                   : mode == kEdgeStream ? &layer_norm_backward_kernel<T, P, LANES, C, kStreamed>                             \
                                         : &layer_norm_backward_kernel<T, P, LANES, C, LANES == 64 ? kWhole : C == 1 ? kShort : kEdge>; \
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kBackwardThreads / shape.threads() * shape.threads()), 0, s, dy, ldy, x, ldx, \
                       weight, mean, rstd, dx, part, dweight, dbias, (int)rows, cols, shape.waves, streaming);                 \
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
    if (params && (blocks != 1 || shape.lanes == 0))
      hipLaunchKernelGGL((layer_norm_params_kernel<P>), dim3(ceil_div(cols, 64), dbias != nullptr ? 2 : 1), dim3(1024), 0, s,
                         part, blocks, cols, dweight, dbias);
  });
  if (!known) return FP8GMM_ERR_LAUNCH;
  return hipGetLastError() == hipSuccess ? FP8GMM_OK : FP8GMM_ERR_LAUNCH;
}

}  // extern "C"
