// The global norm of many tensors, and their scaling by it, for gfx950: the gradients of a step are clipped before the optimizer
// takes them (backend.multi_norm, multi_clip).
//
//   norm = sqrt(sum over all tensors and elements of g^2),  out = g * min(1, max_norm / (norm + 1e-6))
//
// Bound by memory: the norm reads everything once, the scaling once more, and writes.  The squares are taken and added in 64
// bits, which the memory hides (two conversions and a multiply-add per value, a third of the time that its bytes take): no
// magnitude that a gradient can have overflows or vanishes, and the order of the sums does not show in 32 bits.
//
// The tensors travel as the launch's own arguments, 128 of them at a time, so nothing is uploaded, and a captured launch holds
// its table.  Every tensor is cut into chunks; a workgroup takes a contiguous range of all chunks of its launch.  The partial
// sums, one per workgroup, are added up by every workgroup of the scaling for itself, in the same order.  The scaling goes
// backwards through the launches and chunks, from what the norm has read last and the caches still hold.
#include <algorithm>
#include <vector>

#include "elements.h"

namespace fp8gmm {
namespace {

constexpr int kTensors = 128;        // of a launch
constexpr int kThreads = 256;
constexpr int kPieces = 4;           // of 16 bytes per thread and chunk
constexpr int kNormBlocks = 1024;    // workgroups of a launch: four per compute unit
constexpr int kManyPartials = 4096;  // more than these are added up by a launch of their own

struct NormTable {
  const void* in[kTensors];
  int64_t count[kTensors];
  uint32_t begin[kTensors + 1];   // first chunk of every tensor; behind the last one, the launch's chunks
  int n;
};
struct ClipTable {
  const void* in[kTensors];
  void* out[kTensors];
  int64_t count[kTensors];
  uint32_t begin[kTensors + 1];
  int n;
};
static_assert(sizeof(NormTable) <= 4000 && sizeof(ClipTable) <= 4000, "the arguments of a launch");

template <int TYPE>
constexpr int chunk_elements() { return kThreads * kPieces * Elements<TYPE>::kVec; }

template <class Table>
__device__ __forceinline__ int tensor_of(const Table& t, uint32_t chunk) {
  return upper_slot(t.n, (int)chunk, [&](int i) { return (int)t.begin[i]; });
}

__device__ __forceinline__ double lanes_sum64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}
// The sum over a workgroup of WAVES wavefronts, the same in all of its threads
template <int WAVES>
__device__ __forceinline__ double block_sum(double v, double* slots) {
  v = lanes_sum64(v);
  if (threadIdx.x % 64 == 0) slots[threadIdx.x / 64] = v;
  __syncthreads();
  double sum = 0.;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) sum += slots[i];
  return sum;
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void multi_norm_kernel(const NormTable t, double* __restrict__ partials) {
  typedef Elements<TYPE> E;
  typedef typename E::bits bits;
  constexpr int V = E::kVec, CHUNK = chunk_elements<TYPE>();
  __shared__ double slots[kThreads / 64];
  const uint32_t chunks = t.begin[t.n];
  const uint32_t lo = (uint32_t)((uint64_t)chunks * blockIdx.x / gridDim.x), hi = (uint32_t)((uint64_t)chunks * (blockIdx.x + 1) / gridDim.x);
  double sum[2] = {0., 0.};
  int i = tensor_of(t, lo);
  for (uint32_t c = lo; c < hi; ++c) {
    while (c >= t.begin[i + 1]) ++i;
    const int64_t first = (int64_t)(c - t.begin[i]) * CHUNK, left = t.count[i] - first;
    const int n = (int)(left < CHUNK ? left : CHUNK);
    const bits* const p = static_cast<const bits*>(t.in[i]) + first;
    u32x4 raw[kPieces];
#pragma unroll
    for (int u = 0; u < kPieces; ++u) {
      const int at = (u * kThreads + threadIdx.x) * V;
      raw[u] = E::load(p + at, n - at);
    }
#pragma unroll
    for (int u = 0; u < kPieces; ++u) {
      float f[V];
      E::unpack(raw[u], f);
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j & 1] = __builtin_fma((double)f[j], (double)f[j], sum[j & 1]);
    }
  }
  const double total = block_sum<kThreads / 64>(sum[0] + sum[1], slots);
  if (threadIdx.x == 0) partials[blockIdx.x] = total;
}

// norm = sqrt of the sum; `sum` (may be NULL, may be partials): the sum itself
__global__ __launch_bounds__(1024) void multi_norm_finish_kernel(const double* __restrict__ partials, int n,
                                                                 float* __restrict__ norm, double* __restrict__ sum) {
  __shared__ double slots[16];
  double v = 0.;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += 1024) v += partials[i];
  v = block_sum<16>(v, slots);
  if (threadIdx.x != 0) return;
  if (norm != nullptr) *norm = (float)sqrt(v);
  if (sum != nullptr) *sum = v;
}

template <int TYPE, int OUT>
__global__ __launch_bounds__(kThreads) void multi_clip_kernel(const ClipTable t, const double* __restrict__ partials, int n_partials,
                                                              double max_norm, float* __restrict__ norm) {
  typedef Elements<TYPE> E;
  typedef Elements<OUT> O;
  typedef typename E::bits bits;
  constexpr int V = E::kVec, CHUNK = chunk_elements<TYPE>();
  __shared__ double slots[kThreads / 64];
  double v = 0.;
#pragma unroll 4
  for (int i = threadIdx.x; i < n_partials; i += kThreads) v += partials[i];
  const double total = sqrt(block_sum<kThreads / 64>(v, slots));
  if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
  const double ratio = max_norm / (total + 1e-6);
  const float factor = ratio > 1. ? 1.f : (float)ratio;   // a NaN stays one
  const uint32_t chunks = t.begin[t.n], block = gridDim.x - 1 - blockIdx.x;   // backwards
  const uint32_t lo = (uint32_t)((uint64_t)chunks * block / gridDim.x), hi = (uint32_t)((uint64_t)chunks * (block + 1) / gridDim.x);
  if (lo == hi) return;
  int i = tensor_of(t, hi - 1);
  for (uint32_t c = hi; c-- > lo;) {
    while (c < t.begin[i]) --i;
    if (factor == 1.f && t.in[i] == t.out[i]) {   // gradients within the bound stay as they are, in place
      if (t.begin[i] <= lo) return;
      c = t.begin[i];
      continue;
    }
    const int64_t first = (int64_t)(c - t.begin[i]) * CHUNK, left = t.count[i] - first;
    const int n = (int)(left < CHUNK ? left : CHUNK);
    const bits* const p = static_cast<const bits*>(t.in[i]) + first;
    typename O::bits* const out = static_cast<typename O::bits*>(t.out[i]) + first;
    u32x4 raw[kPieces];
#pragma unroll
    for (int u = 0; u < kPieces; ++u) {
      const int at = (u * kThreads + threadIdx.x) * V;
      raw[u] = E::load(p + at, n - at);
    }
#pragma unroll
    for (int u = 0; u < kPieces; ++u) {
      const int at = (u * kThreads + threadIdx.x) * V;
      float f[V];
      E::unpack(raw[u], f);
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] *= factor;
      if constexpr (O::kVec >= V) {   // fp32 gradients stay in fp32
        O::store(out + at, n - at, O::pack(f));
      } else {
#pragma unroll
        for (int q = 0; q < V / O::kVec; ++q) {
          float part[O::kVec];
#pragma unroll
          for (int j = 0; j < O::kVec; ++j) part[j] = f[q * O::kVec + j];
          O::store(out + at + q * O::kVec, n - at - q * O::kVec, O::pack(part));
        }
      }
    }
  }
}

uint32_t chunks_of(int64_t count, int type) {
  const int64_t chunk = (int64_t)kThreads * kPieces * 16 / type_bytes(type);
  return (uint32_t)((count + chunk - 1) / chunk);
}

int check_tensors(const fp8gmm_norm_tensor* tensors, int n, bool out) {
  if (n < 0) return FP8GMM_ERR_BAD_ARGUMENT;
  if (n > 0 && tensors == nullptr) return FP8GMM_ERR_NULL_POINTER;
  int64_t all = 0;   // bounds the chunks of a launch
  for (int i = 0; i < n; ++i) {
    const fp8gmm_norm_tensor& t = tensors[i];
    if (!known_type(t.type) || (out && t.out_type != t.type && t.out_type != FP8GMM_TYPE_FP32)) return FP8GMM_ERR_BAD_FORMAT;
    if (t.count < 0 || t.count > ((int64_t)1 << 40) - all) return FP8GMM_ERR_BAD_SHAPE;
    all += t.count;
    if (t.count > 0 && (t.in == nullptr || (out && t.out == nullptr))) return FP8GMM_ERR_NULL_POINTER;
    const int64_t mask = type_bytes(t.type) - 1, out_mask = out ? type_bytes(t.out_type) - 1 : 0;
    if ((reinterpret_cast<uintptr_t>(t.in) & mask) || (out && (reinterpret_cast<uintptr_t>(t.out) & out_mask)))
      return FP8GMM_ERR_ALIGNMENT;
  }
  return FP8GMM_OK;
}

// Nothing is written that another tensor of the call reads or writes: a result lies apart from all else, or in the place of its own tensor.
int check_apart(const fp8gmm_norm_tensor* tensors, int n) {
  struct Range {
    uintptr_t begin, end;
    int which, writes;
  };
  std::vector<Range> ranges;
  ranges.reserve(2 * (size_t)n);
  for (int i = 0; i < n; ++i) {
    const fp8gmm_norm_tensor& t = tensors[i];
    if (t.count == 0) continue;
    const uintptr_t in = reinterpret_cast<uintptr_t>(t.in), out = reinterpret_cast<uintptr_t>(t.out);
    ranges.push_back({out, out + (uintptr_t)t.count * type_bytes(t.out_type), i, 1});
    if (in != out || t.type != t.out_type) ranges.push_back({in, in + (uintptr_t)t.count * type_bytes(t.type), i, 0});
  }
  std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
  uintptr_t written = 0, read = 0;   // ends of what the ranges so far write and read
  for (const Range& r : ranges) {
    if (r.begin < written || (r.writes && r.begin < read)) return FP8GMM_ERR_BAD_ARGUMENT;
    (r.writes ? written : read) = std::max(r.writes ? written : read, r.end);
  }
  return FP8GMM_OK;
}

struct Part {   // of a list: up to kTensors tensors of one type (of one pair of types)
  std::vector<int> which;
  uint32_t chunks = 0;
};
std::vector<Part> parts_of(const fp8gmm_norm_tensor* tensors, int n, int type, int out_type) {
  std::vector<Part> parts;
  for (int i = 0; i < n; ++i) {
    const fp8gmm_norm_tensor& t = tensors[i];
    if (t.count == 0 || t.type != type || (out_type >= 0 && t.out_type != out_type)) continue;
    const uint32_t chunks = chunks_of(t.count, type);
    if (parts.empty() || parts.back().which.size() == kTensors) parts.emplace_back();
    parts.back().which.push_back(i);
    parts.back().chunks += chunks;
  }
  return parts;
}

constexpr int kAllTypes[] = {FP8GMM_TYPE_BF16, FP8GMM_TYPE_FP16, FP8GMM_TYPE_FP32};

// Enqueues the partial sums; how many there are.
int launch_norms(const fp8gmm_norm_tensor* tensors, int n, double* partials, hipStream_t s) {
  int total = 0;
  for (const int type : kAllTypes)
    for (const Part& part : parts_of(tensors, n, type, -1)) {
      NormTable t;
      t.n = (int)part.which.size();
      uint32_t at = 0;
      for (int i = 0; i < t.n; ++i) {
        const fp8gmm_norm_tensor& from = tensors[part.which[i]];
        t.in[i] = from.in;
        t.count[i] = from.count;
        t.begin[i] = at;
        at += chunks_of(from.count, type);
      }
      t.begin[t.n] = at;
      const int blocks = (int)std::min<uint32_t>(kNormBlocks, part.chunks);
      auto* kernel = type == FP8GMM_TYPE_BF16   ? &multi_norm_kernel<FP8GMM_TYPE_BF16>
                     : type == FP8GMM_TYPE_FP16 ? &multi_norm_kernel<FP8GMM_TYPE_FP16>
                                                : &multi_norm_kernel<FP8GMM_TYPE_FP32>;
      hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kThreads), 0, s, t, partials + total);
      total += blocks;
    }
  return total;
}

template <int TYPE, int OUT>
void launch_clips(const fp8gmm_norm_tensor* tensors, int n, const double* partials, int n_partials, double max_norm, float** norm,
                  hipStream_t s) {
  const std::vector<Part> parts = parts_of(tensors, n, TYPE, OUT);
  for (auto part = parts.rbegin(); part != parts.rend(); ++part) {
    ClipTable t;
    t.n = (int)part->which.size();
    uint32_t at = 0;
    for (int i = 0; i < t.n; ++i) {
      const fp8gmm_norm_tensor& from = tensors[part->which[i]];
      t.in[i] = from.in;
      t.out[i] = from.out;
      t.count[i] = from.count;
      t.begin[i] = at;
      at += chunks_of(from.count, TYPE);
    }
    t.begin[t.n] = at;
    hipLaunchKernelGGL((multi_clip_kernel<TYPE, OUT>), dim3(std::min<uint32_t>(2 * kNormBlocks, part->chunks)), dim3(kThreads), 0,
                       s, t, partials, n_partials, max_norm, *norm);
    *norm = nullptr;   // by the first launch
  }
}

int check_workspace(int n, void* workspace, size_t bytes) {
  if (workspace == nullptr) return FP8GMM_ERR_NULL_POINTER;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return FP8GMM_ERR_ALIGNMENT;
  return bytes < fp8gmm_multi_norm_workspace_bytes(n) ? FP8GMM_ERR_WORKSPACE : FP8GMM_OK;
}

int multi_norm(const fp8gmm_norm_tensor* tensors, int n, float* norm, void* workspace, size_t bytes, hipStream_t s) {
  int rc = check_tensors(tensors, n, false);
  if (rc == FP8GMM_OK) rc = norm == nullptr ? FP8GMM_ERR_NULL_POINTER : check_workspace(n, workspace, bytes);
  if (rc != FP8GMM_OK) return rc;
  double* const partials = static_cast<double*>(workspace);
  const int total = launch_norms(tensors, n, partials, s);
  hipLaunchKernelGGL(multi_norm_finish_kernel, dim3(1), dim3(1024), 0, s, partials, total, norm, static_cast<double*>(nullptr));
  return hipGetLastError() == hipSuccess ? FP8GMM_OK : FP8GMM_ERR_LAUNCH;
}

int multi_clip(const fp8gmm_norm_tensor* tensors, int n, double max_norm, float* norm, void* workspace, size_t bytes,
               hipStream_t s) {
  int rc = check_tensors(tensors, n, true);
  if (rc == FP8GMM_OK) rc = norm == nullptr ? FP8GMM_ERR_NULL_POINTER : check_workspace(n, workspace, bytes);
  if (rc == FP8GMM_OK && !(max_norm >= 0.)) rc = FP8GMM_ERR_BAD_ARGUMENT;
  if (rc == FP8GMM_OK) rc = check_apart(tensors, n);
  if (rc != FP8GMM_OK) return rc;
  double* partials = static_cast<double*>(workspace);
  int total = launch_norms(tensors, n, partials, s);
  if (total == 0 || total > kManyPartials) {
    double* const sum = partials + total;
    hipLaunchKernelGGL(multi_norm_finish_kernel, dim3(1), dim3(1024), 0, s, partials, total, norm, sum);
    partials = sum;
    total = 1;
    norm = nullptr;   // written
  }
  launch_clips<FP8GMM_TYPE_FP32, FP8GMM_TYPE_FP32>(tensors, n, partials, total, max_norm, &norm, s);
  launch_clips<FP8GMM_TYPE_FP16, FP8GMM_TYPE_FP32>(tensors, n, partials, total, max_norm, &norm, s);
  launch_clips<FP8GMM_TYPE_FP16, FP8GMM_TYPE_FP16>(tensors, n, partials, total, max_norm, &norm, s);
  launch_clips<FP8GMM_TYPE_BF16, FP8GMM_TYPE_FP32>(tensors, n, partials, total, max_norm, &norm, s);
  launch_clips<FP8GMM_TYPE_BF16, FP8GMM_TYPE_BF16>(tensors, n, partials, total, max_norm, &norm, s);
  return hipGetLastError() == hipSuccess ? FP8GMM_OK : FP8GMM_ERR_LAUNCH;
}

// The host's lists are the only thing here that can fail by an exception, which ends at this border.
template <class F>
int without_exceptions(F&& f) noexcept {
  try {
    return f();
  } catch (...) {
    return FP8GMM_ERR_BAD_ARGUMENT;
  }
}

}  // namespace
}  // namespace fp8gmm

extern "C" {

size_t fp8gmm_multi_norm_workspace_bytes(int n) {
  using namespace fp8gmm;
  // a launch per kTensors tensors and one more that is not full for every type, and the sum
  return n < 0 ? 0 : ((size_t)(n / kTensors + 4) * kNormBlocks + 2) * sizeof(double);
}

int fp8gmm_multi_norm(const fp8gmm_norm_tensor* tensors, int n, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  return fp8gmm::without_exceptions(
      [&] { return fp8gmm::multi_norm(tensors, n, norm, workspace, workspace_bytes, static_cast<hipStream_t>(stream)); });
}

int fp8gmm_multi_clip(const fp8gmm_norm_tensor* tensors, int n, double max_norm, float* norm, void* workspace,
                      size_t workspace_bytes, void* stream) {
  return fp8gmm::without_exceptions([&] {
    return fp8gmm::multi_clip(tensors, n, max_norm, norm, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
  });
}

}  // extern "C"
