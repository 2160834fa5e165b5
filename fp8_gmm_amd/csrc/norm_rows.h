// What the norms of rows share (layer_norm.hip, rms_norm.hip): how a row of any length and alignment is shared out to threads and
// reached by them, and the sum of the workgroups' shares of the parameters' gradients.
#pragma once

#include <algorithm>

#include "elements.h"

namespace fp8gmm {
namespace {

constexpr int kNormLongThreads = 1024;
constexpr int kNormSlab = 1 << 16;   // rows of a launch with a workgroup to a row, 2 GB at least: a grid has fewer than 2^32 threads
constexpr int kNormColumns = 1 << 27;   // of a launch that adds up parameters' gradients, 16 threads to a column
constexpr int kNormWaves = 16;       // the most wavefronts that share a row

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

// The workgroups' partial sums, [workgroup][outputs][cols], in their order: 64 columns a workgroup, a sixteenth of the sums a wavefront.  Without any
// (no rows) the gradients are zeros.  From column `first` on.
template <int PTYPE>
__global__ __launch_bounds__(1024) void norm_params_kernel(const float* __restrict__ part, int blocks, int outputs, int first, int cols,
                                                          void* __restrict__ dweight, void* __restrict__ dbias) {
  typedef Elements<PTYPE> P;
  __shared__ float sums[16][64];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, which = blockIdx.y;
  const int64_t col = first + (int64_t)blockIdx.x * 64 + lane;
  void* const out = which == 0 ? dweight : dbias;
  float sum = 0.f;
  if (col < cols) {
    const int per = (blocks + 15) / 16, last = min(blocks, (wave + 1) * per);
    const float* p = part + (int64_t)which * cols + col;
#pragma unroll 8
    for (int i = wave * per; i < last; ++i) sum += p[(int64_t)i * outputs * cols];
  }
  sums[wave][lane] = sum;
  __syncthreads();
  if (wave != 0 || col >= cols || out == nullptr) return;
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) sum += sums[i][lane];
  static_cast<typename P::bits*>(out)[col] = P::pack1(sum);
}

[[maybe_unused]] int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

template <int PTYPE>
void launch_norm_params(const float* part, int blocks, int outputs, int cols, void* dweight, void* dbias, hipStream_t s) {
  for (int64_t first = 0; first < cols; first += kNormColumns)
    hipLaunchKernelGGL((norm_params_kernel<PTYPE>), dim3(ceil_div(std::min<int64_t>(cols - first, kNormColumns), 64), dbias != nullptr ? 2 : 1),
                       dim3(1024), 0, s, part, blocks, outputs, (int)first, cols, dweight, dbias);
}

// How a row is shared out: `lanes` * `waves` threads, `pieces` 16-byte pieces to each.  No lanes: longer than the registers of a
// workgroup hold.
struct Shape {
  int lanes, waves, pieces;
  int threads() const { return lanes * waves; }
};
[[maybe_unused]] int pieces_of(int cols, int type) { return ceil_div(cols, 16 / type_bytes(type)); }
// Up to `most` pieces to a thread, as few threads as that allows, and then as few pieces: a thread behind the row's end works for
// nothing.  `waves`: the most of them.  A row's first 64 * waves pieces are there, so that every wavefront has some of the row.
// `narrow`: the most pieces of a thread where 16 lanes have a row.  4 forward (262144 x 256, bf16, 70 us by 64 lanes, 47 so; 131072 x
// 384, 39.5 and 35.7; 131072 x 512, 48.6 and 46.7), 2 backward (262144 x 256, 87 and 79; with 3, 131072 x 384, 55 and 161: spills).
[[maybe_unused]] Shape shape_of(int pieces, int most, int waves, int narrow) {
  if (pieces <= 16 * narrow) return {16, 1, ceil_div(pieces, 16)};
  const int w = ceil_div(pieces, 64 * most);
  return w <= waves ? Shape{64, w, ceil_div(pieces, 64 * w)} : Shape{0, 0, 0};
}
// The longest rows that stay in registers have 4 pieces in each of 1024 threads, which fits fp32 alone: a 16-bit type has twice
// the elements and spills backward (4096 x 32768, bf16: 103 and 781 us forward and backward, by the kernels for longer rows 146 and
// 296; 4096 x 16384, fp32: 92 and 174, by those 142 and 287).
[[maybe_unused]] Shape widest(int cols, int type) {
  const int w = ceil_div(pieces_of(cols, type), 64 * 4);
  return type == FP8GMM_TYPE_FP32 && w <= kNormWaves ? Shape{64, w, 4} : Shape{0, 0, 0};
}
// Whether a result is written with the streaming hint: one that outgrows the cache is not found there by whoever reads it.  With it
// and without: 16384 x 4096, bf16, forward 49 and 49 us, backward 73 and 78; 65536 x 2048, fp32, 185 and 191, 259 and 269; 24576 x
// 2048, bf16, 36.4 and 37.2, 55.5 and 57.9.
[[maybe_unused]] bool streams(int64_t rows, int cols, int type) { return rows * cols * type_bytes(type) > (int64_t)64 << 20; }
// Rows of whole pieces on 16 bytes
[[maybe_unused]] bool whole(const void* p, int64_t pitch, int cols, int type) {
  const int pieces = 16 / type_bytes(type);
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && pitch % pieces == 0 && cols % pieces == 0;
}
// A descriptor is a wavefront's, which has four rows where 16 lanes have one: these have edges, if empty ones.
[[maybe_unused]] int mode_of(int cols, int type, int lanes, bool aligned, bool stream_edges) {
  return cols < 16 / type_bytes(type) ? kShort : aligned && lanes == 64 ? kWhole : stream_edges ? kEdgeStream : kEdge;
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

}  // namespace
}  // namespace fp8gmm
