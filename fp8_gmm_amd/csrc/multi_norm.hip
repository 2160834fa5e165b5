// The global norm of many tensors, and their scaling by it, for gfx950: the gradients of a step are clipped before the optimizer
// takes them (backend.multi_norm, multi_clip).
//
//   norm = sqrt(sum over all tensors and elements of g^2),  out = g * min(1, max_norm / (norm + 1e-6))
//
// Bound by memory: the norm reads everything once, the scaling once more, and writes.  The squares are taken and added in 64
// bits, which the memory hides (two conversions and a multiply-add per value, a third of the time that its bytes take): no
// magnitude that a gradient can have overflows or vanishes, and the order of the sums does not show in 32 bits.
//
// Every tensor is cut into chunks of 16 KB, and a workgroup takes a contiguous range of all chunks.  The table of the tensors of a
// short list travels in the launches' arguments (96 tensors, 290 MB of bf16, clipped: 150.8 us, through memory 152.6; 112 short ones
// 14.7, 113 of them 19.6); that of a longer one is written to the workspace first, 200 tensors to a launch, by their arguments too -
// so nothing is uploaded, and a captured call holds its table.  The partial sums, one per workgroup of the norm, are added up by every
// workgroup of the scaling for itself, in the same order, or in a launch of their own where they are many.  The scaling goes
// backwards, from what the norm has read last and the caches still hold.
#include <algorithm>
#include <vector>

#include "elements.h"

namespace fp8gmm {
namespace {

constexpr int kTensors = 112;        // of a launch's arguments
constexpr int kThreads = 256;
constexpr int kPieces = 4;           // of 16 bytes per thread and chunk
constexpr int kChunkBytes = kThreads * kPieces * 16;
// Chunks of a workgroup of the norm, and more of very long lists.  Norms of 96 tensors, 290 MB of bf16, by 1, 4 and 16 chunks:
// 50.6, 51.8 and 53.5 us; of 24 tensors, 67 MB of fp32, by 1 and 4: 17.4 and 15.9 (more workgroups, more partial sums).
constexpr int kRun = 4;
constexpr int kNormBlocks = 8192;    // the most workgroups of a launch
// Partial sums that every workgroup of the scaling adds up for itself; more have a launch for that.  Clipping of 24 tensors of
// 87381 fp32 elements (129 sums) 13.0 us, with the launch 15.7; of 349525 (516) 22.0 without it and 23.1; of 300 MB (4600) 182
// and 151.
constexpr int kFewPartials = 512;
constexpr int kClipBlocks = 1 << 20; // of the scaling, a chunk or half of one to each but for lists of 8 GB and more
// Halves of a chunk to a workgroup of the scaling where some results are fp32 of 16 bits, twice what is read: 1.9 GB to 3.8 1224 us, by
// whole chunks 1331; 305 MB to 610, 400 tensors, 215.5 and 217.  Results of the same type by halves: 160 us, and 171.
constexpr int kWiderParts = 2;
// Gradients are read with the streaming hint where nothing of them would be found in the caches by a second pass, 512 MB on (1.9
// GB to 3.8 by whole chunks: 1332 us, without the hint 1346; 270 MB: 159, with it 163), or where there is none (norm of 290 MB:
// 52 us, without 58).  Results are written with it where whoever reads them does not find them there (290 MB clipped: 151 us,
// without 182).
constexpr int64_t kStreamTwice = (int64_t)512 << 20, kStreamOnce = (int64_t)32 << 20, kStreamOut = (int64_t)64 << 20;
static_assert(kStreamTwice >= kStreamOut, "results are no fewer bytes than what is read: the hint on the reads means both");

struct Entry {
  const void* in;
  void* out;
  int64_t count;
  uint32_t begin;   // first chunk
  uint16_t type, out_type;
};
static_assert(sizeof(Entry) == 32, "two to a cache line's half");
struct Part {
  Entry e[kTensors];
};
static_assert(sizeof(Part) <= 3600, "the arguments of a launch");

// The tensors of a call: in the arguments, or in memory.
template <bool DIRECT>
struct Table {
  const Part& part;
  const Entry* memory;
  int n;
  uint32_t chunks;
  __device__ __forceinline__ const Entry& operator[](int i) const { return DIRECT ? part.e[i] : memory[i]; }
  __device__ __forceinline__ uint32_t end(int i) const { return i + 1 < n ? (*this)[i + 1].begin : chunks; }
  // The tensor that a chunk is of: every thread looks at tensors of its own
  __device__ __forceinline__ int of(uint32_t chunk) const {
    __shared__ int found;
    for (int i = threadIdx.x; i < n; i += kThreads)
      if ((*this)[i].begin <= chunk && chunk < end(i)) found = i;
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(found);
  }
};

// The table of a longer list: an entry travels in 18 bytes, 48 bits of each address, 40 of the count, and the types.  400 short
// tensors, norm: 21.5 us with these, 28.4 with entries as they are in memory, 112 to a launch.
struct Packed {
  uint16_t part[9];
};
constexpr int kPacked = 200, kPackedThreads = 256;   // of a launch
struct PackedPart {
  Packed e[kPacked];
};
static_assert(sizeof(PackedPart) <= 3600, "the arguments of a launch");

__host__ __device__ inline uint32_t chunks_of(int64_t count, int type) {
  return (uint32_t)((count * (type == FP8GMM_TYPE_FP32 ? 4 : 2) + kChunkBytes - 1) / kChunkBytes);
}

__global__ __launch_bounds__(kPackedThreads) void multi_norm_table_kernel(const PackedPart part, int n, uint32_t begin,
                                                                          Entry* __restrict__ table) {
  __shared__ uint32_t sums[kPackedThreads / 64];
  const int i = threadIdx.x, lane = i % 64, wave = i / 64;
  Entry e = {};
  uint32_t chunks = 0;
  if (i < n) {
    uint64_t word[9];
#pragma unroll
    for (int k = 0; k < 9; ++k) word[k] = part.e[i].part[k];
    e.in = reinterpret_cast<const void*>(word[0] | word[1] << 16 | word[2] << 32);
    e.out = reinterpret_cast<void*>(word[3] | word[4] << 16 | word[5] << 32);
    e.count = (int64_t)(word[6] | word[7] << 16 | (word[8] & 0xff) << 32);
    e.type = (uint16_t)(word[8] >> 8 & 0xf);
    e.out_type = (uint16_t)(word[8] >> 12);
    chunks = chunks_of(e.count, e.type);
  }
  uint32_t incl = chunks;   // the first chunks: prefix sums
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t other = __shfl_up(incl, d, 64);
    if (lane >= d) incl += other;
  }
  if (lane == 63) sums[wave] = incl;
  __syncthreads();
  e.begin = begin + incl - chunks;
#pragma unroll
  for (int w = 0; w < kPackedThreads / 64; ++w)
    if (w < wave) e.begin += sums[w];
  if (i < n) table[i] = e;
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

// f(TYPE, elements of a chunk) for a tensor's type
template <class F>
__device__ __forceinline__ void with_type(int type, F&& f) {
  if (type == FP8GMM_TYPE_BF16) f(std::integral_constant<int, FP8GMM_TYPE_BF16>{});
  else if (type == FP8GMM_TYPE_FP16) f(std::integral_constant<int, FP8GMM_TYPE_FP16>{});
  else f(std::integral_constant<int, FP8GMM_TYPE_FP32>{});
}

// The pieces of a thread of the chunk, or share of one, at `p`, of which `n` elements are the tensor's
template <int TYPE, bool STREAM, int PIECES>
__device__ __forceinline__ void load_chunk(const typename Elements<TYPE>::bits* p, int n, int t, u32x4 (&raw)[PIECES]) {
  typedef Elements<TYPE> E;
  constexpr int V = E::kVec;
  if (n == kThreads * PIECES * V) {
#pragma unroll
    for (int u = 0; u < PIECES; ++u) raw[u] = E::template load<STREAM>(p + (u * kThreads + t) * V, V);
  } else {
#pragma unroll
    for (int u = 0; u < PIECES; ++u) raw[u] = E::load(p + (u * kThreads + t) * V, n - (u * kThreads + t) * V);
  }
}

// The elements of a tensor in front of the first 16 bytes that are aligned.  They belong to its first chunk, and the chunks' pieces
// are aligned (270 MB in tensors at any element: norm 65 us with chunks from the first element on, 58 with these; clipped 169 and
// 161).  A tensor's last chunk may be left without elements.
template <int SIZE>
__device__ __forceinline__ int head_of(const void* p, int64_t count) {
  const int head = (int)(-reinterpret_cast<uintptr_t>(p) & 15) / SIZE;
  return count < head ? (int)count : head;
}
template <int TYPE>
__device__ __forceinline__ float element(const typename Elements<TYPE>::bits* p) {
  float f[Elements<TYPE>::kVec];
  Elements<TYPE>::unpack(Elements<TYPE>::load(p, 1), f);
  return f[0];
}

// The squares of thread t's share of chunk c, added to `sum`
template <int TYPE, bool STREAM>
__device__ __forceinline__ void add_squares(const Entry& e, uint32_t c, int t, double (&sum)[2]) {
  typedef Elements<TYPE> E;
  constexpr int V = E::kVec, CHUNK = kThreads * kPieces * V;
  const typename E::bits* const p = static_cast<const typename E::bits*>(e.in);
  const int head = head_of<E::kBytes>(p, e.count);
  const int64_t first = head + (int64_t)(c - e.begin) * CHUNK, left = e.count - first;
  u32x4 raw[kPieces];
  load_chunk<TYPE, STREAM>(p + first, (int)(left < CHUNK ? left : CHUNK), t, raw);
  if (c == e.begin && t < head) {
    const float f = element<TYPE>(p + t);
    sum[0] = __builtin_fma((double)f, (double)f, sum[0]);
  }
#pragma unroll
  for (int u = 0; u < kPieces; ++u) {
    float f[V];
    E::unpack(raw[u], f);
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j & 1] = __builtin_fma((double)f[j], (double)f[j], sum[j & 1]);
  }
}

template <bool DIRECT, bool STREAM>
__global__ __launch_bounds__(kThreads) void multi_norm_kernel(const Part part, const Entry* __restrict__ memory, int n, uint32_t chunks,
                                                              double* __restrict__ partials) {
  __shared__ double slots[kThreads / 64];
  const Table<DIRECT> table = {part, memory, n, chunks};
  const uint32_t lo = (uint32_t)((uint64_t)chunks * blockIdx.x / gridDim.x), hi = (uint32_t)((uint64_t)chunks * (blockIdx.x + 1) / gridDim.x);
  double sum[2] = {0., 0.};
  int i = table.of(lo);
  for (uint32_t c = lo; c < hi; ++i) {
    const Entry e = table[i];
    const uint32_t last = min(table.end(i), hi);
    with_type(e.type, [&](auto type) {
      for (; c < last; ++c) add_squares<decltype(type)::value, STREAM>(e, c, threadIdx.x, sum);
    });
  }
  const double total = block_sum<kThreads / 64>(sum[0] + sum[1], slots);
  if (threadIdx.x == 0) partials[blockIdx.x] = total;
}

// The factor of the scaling: 1 within the bound; a norm that is a NaN stays one, an infinite one makes it 0.
__device__ __forceinline__ float factor_of(double norm, double max_norm) {
  const double ratio = max_norm / (norm + 1e-6);
  return ratio > 1. ? 1.f : (float)ratio;
}

// The norm, and the factor behind it where a scaling follows.
__global__ __launch_bounds__(1024) void multi_norm_finish_kernel(const double* __restrict__ partials, int n, double max_norm,
                                                                 float* __restrict__ norm, float* __restrict__ factor) {
  __shared__ double slots[16];
  double v = 0.;
#pragma unroll 8
  for (int i = threadIdx.x; i < n; i += 1024) v += partials[i];
  v = sqrt(block_sum<16>(v, slots));
  if (threadIdx.x != 0) return;
  *norm = (float)v;
  if (factor != nullptr) *factor = factor_of(v, max_norm);
}

// A chunk's pieces times the factor.  fp32 results of a 16-bit type: pieces of four elements, 8 bytes read and 16 written, so
// that a store instruction writes whole lines (with 8 elements a thread, whose two stores share lines, the streaming hint made
// 1.9 GB to 3.8 take 2440 us; without it 1544).
template <int TYPE, int OUT, bool STREAM, bool STREAM_OUT, int PIECES>
__device__ __forceinline__ void scale_chunk(const typename Elements<TYPE>::bits* p, typename Elements<OUT>::bits* out, int n, int t,
                                            float factor) {
  typedef Elements<TYPE> E;
  typedef Elements<OUT> O;
  if constexpr (TYPE == OUT) {
    constexpr int V = E::kVec;
    const bool all = n == kThreads * PIECES * V;
    u32x4 raw[PIECES];
    load_chunk<TYPE, STREAM>(p, n, t, raw);
#pragma unroll
    for (int u = 0; u < PIECES; ++u) {
      float f[V];
      E::unpack(raw[u], f);
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] *= factor;
      raw[u] = E::pack(f);
    }
    if (all) {
#pragma unroll
      for (int u = 0; u < PIECES; ++u) O::template store<STREAM_OUT>(out + (u * kThreads + t) * V, V, raw[u]);
    } else {
#pragma unroll
      for (int u = 0; u < PIECES; ++u)
        O::store(out + (u * kThreads + t) * V, n - (u * kThreads + t) * V, raw[u]);
    }
  } else {
    constexpr int V = 4, COUNT = PIECES * E::kVec / V;
    typedef uint32_t half_piece __attribute__((ext_vector_type(2), aligned(2)));
    const auto scaled = [&](u32x2 raw) {
      float f[E::kVec];
      E::unpack(u32x4{raw.x, raw.y, 0u, 0u}, f);
      return u32x4{__float_as_uint(f[0] * factor), __float_as_uint(f[1] * factor), __float_as_uint(f[2] * factor),
                   __float_as_uint(f[3] * factor)};
    };
    if (n == kThreads * COUNT * V) {
      u32x2 raw[COUNT];
#pragma unroll
      for (int u = 0; u < COUNT; ++u) {
        const half_piece* const at = reinterpret_cast<const half_piece*>(p + (u * kThreads + t) * V);
        raw[u] = STREAM ? __builtin_nontemporal_load(at) : *at;
      }
#pragma unroll
      for (int u = 0; u < COUNT; ++u) O::template store<STREAM_OUT>(out + (u * kThreads + t) * V, V, scaled(raw[u]));
    } else {
      for (int at = t * V; at < n; at += kThreads * V) {
        const u32x4 raw = E::load(p + at, min(n - at, V));
        O::store(out + at, n - at, scaled(u32x2{raw.x, raw.y}));
      }
    }
  }
}

// Thread t's share of a part of chunk c of a tensor, scaled; the chunks as the result is aligned
template <int TYPE, int OUT, bool STREAM, bool STREAM_OUT, int PARTS>
__device__ __forceinline__ void scale_as(const Entry& e, uint32_t c, int part, int t, float factor) {
  typedef Elements<TYPE> E;
  typedef Elements<OUT> O;
  constexpr int CHUNK = kThreads * kPieces * E::kVec, SHARE = CHUNK / PARTS;
  const typename E::bits* const p = static_cast<const typename E::bits*>(e.in);
  typename O::bits* const out = static_cast<typename O::bits*>(e.out);
  const int head = head_of<O::kBytes>(out, e.count);
  const int64_t at = head + (int64_t)(c - e.begin) * CHUNK + part * SHARE, left = e.count - at;
  scale_chunk<TYPE, OUT, STREAM, STREAM_OUT, kPieces / PARTS>(p + at, out + at, (int)(left < SHARE ? left : SHARE), t, factor);
  if (c == e.begin && part == 0 && t < head) out[t] = O::pack1(element<TYPE>(p + t) * factor);
}
template <int TYPE, bool STREAM, bool STREAM_OUT, int PARTS>
__device__ __forceinline__ void scale(const Entry& e, uint32_t c, int part, int t, float factor) {
  if (TYPE != FP8GMM_TYPE_FP32 && e.out_type == FP8GMM_TYPE_FP32)
    scale_as<TYPE, FP8GMM_TYPE_FP32, STREAM, STREAM_OUT, PARTS>(e, c, part, t, factor);
  else
    scale_as<TYPE, TYPE, STREAM, STREAM_OUT, PARTS>(e, c, part, t, factor);
}

template <bool DIRECT, bool STREAM, bool STREAM_OUT, int PARTS>
__global__ __launch_bounds__(kThreads) void multi_clip_kernel(const Part part, const Entry* __restrict__ memory, int n, uint32_t chunks,
                                                              const double* __restrict__ partials, int n_partials, double max_norm,
                                                              const float* __restrict__ finished, bool in_place, float* __restrict__ norm) {
  __shared__ double slots[kThreads / 64];
  float factor;
  if (finished != nullptr) {
    factor = *finished;
  } else {
    double v = 0.;
    for (int i = threadIdx.x; i < n_partials; i += kThreads) v += partials[i];
    const double total = sqrt(block_sum<kThreads / 64>(v, slots));
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
    factor = factor_of(total, max_norm);
  }
  if (in_place && factor == 1.f) return;   // all of them
  const Table<DIRECT> table = {part, memory, n, chunks};
  const uint32_t block = gridDim.x - 1 - blockIdx.x;      // backwards
  const uint64_t parts = (uint64_t)chunks * PARTS;
  const uint32_t lo = (uint32_t)(parts * block / gridDim.x), hi = (uint32_t)(parts * (block + 1) / gridDim.x);
  if (lo == hi) return;
  int i = table.of((hi - 1) / PARTS);
  for (uint32_t c = hi; c > lo; --i) {
    const Entry e = table[i];
    const uint32_t first = max(e.begin * PARTS, lo);
    if (factor == 1.f && e.in == e.out) {   // gradients within the bound stay as they are, in place
      c = first;
      continue;
    }
    with_type(e.type, [&](auto type) {
      for (; c > first; --c)
        scale<decltype(type)::value, STREAM, STREAM_OUT, PARTS>(e, (c - 1) / PARTS, (c - 1) % PARTS, threadIdx.x, factor);
    });
  }
}

// A short list in one launch of one workgroup, and one pass over memory: cut into units of 4 KB, up to four of them to a wavefront,
// which stay in its registers while the workgroup shares the norm.  Bound by the latency of a launch and of one access: 24 tensors
// of 1300 fp32 take 8.3 us from call to call, by two launches over chunks 12.6; 64 units 8.4, and 13.
constexpr int kUnitWaves = 16, kUnitsEach = 4, kUnits = kUnitWaves * kUnitsEach;
struct Unit {
  const void* in;
  void* out;
  int32_t count;   // elements, at most kPieces 16-byte pieces of every lane
  uint16_t type, out_type;
};
struct Units {
  Unit u[kUnits];
};
static_assert(sizeof(Units) <= 1600, "the arguments of a launch");

__global__ __launch_bounds__(kUnitWaves * 64) void multi_small_kernel(const Units units, int n, bool clip, double max_norm,
                                                                      float* __restrict__ norm) {
  __shared__ double slots[kUnitWaves];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  u32x4 raw[kUnitsEach][kPieces];
#pragma unroll
  for (int r = 0; r < kUnitsEach; ++r) {
    const int k = wave + r * kUnitWaves;
    if (k >= n) continue;
    const Unit& u = units.u[k];
    if (u.type == FP8GMM_TYPE_FP32) {
      typedef Elements<FP8GMM_TYPE_FP32> E;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int at = (i * 64 + lane) * E::kVec;
        raw[r][i] = E::load(static_cast<const uint32_t*>(u.in) + at, u.count - at);
      }
    } else {   // the bits of either 16-bit type
      typedef Elements<FP8GMM_TYPE_BF16> E;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int at = (i * 64 + lane) * E::kVec;
        raw[r][i] = E::load(static_cast<const uint16_t*>(u.in) + at, u.count - at);
      }
    }
  }
  double sum = 0.;
#pragma unroll
  for (int r = 0; r < kUnitsEach; ++r) {
    const int k = wave + r * kUnitWaves;
    if (k >= n) continue;
    with_type(units.u[k].type, [&](auto type) {
      typedef Elements<decltype(type)::value> E;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        float f[E::kVec];
        E::unpack(raw[r][i], f);
#pragma unroll
        for (int j = 0; j < E::kVec; ++j) sum = __builtin_fma((double)f[j], (double)f[j], sum);
      }
    });
  }
  const double total = sqrt(block_sum<kUnitWaves>(sum, slots));
  if (threadIdx.x == 0) *norm = (float)total;
  if (!clip) return;
  const float factor = factor_of(total, max_norm);
#pragma unroll
  for (int r = 0; r < kUnitsEach; ++r) {
    const int k = wave + r * kUnitWaves;
    if (k >= n) continue;
    const Unit& u = units.u[k];
    if (factor == 1.f && u.in == u.out) continue;   // gradients within the bound stay as they are, in place
    with_type(u.type, [&](auto type) {
      typedef Elements<decltype(type)::value> E;
      typedef Elements<FP8GMM_TYPE_FP32> F;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int at = (i * 64 + lane) * E::kVec;
        float f[E::kVec];
        E::unpack(raw[r][i], f);
#pragma unroll
        for (int j = 0; j < E::kVec; ++j) f[j] *= factor;
        if (u.out_type == u.type) {
          E::store(static_cast<typename E::bits*>(u.out) + at, u.count - at, E::pack(f));
        } else {
#pragma unroll
          for (int q = 0; q < E::kVec; q += 4)
            F::store(static_cast<uint32_t*>(u.out) + at + q, u.count - at - q,
                     u32x4{__float_as_uint(f[q]), __float_as_uint(f[q + 1]), __float_as_uint(f[q + 2]), __float_as_uint(f[q + 3])});
        }
      }
    });
  }
}

int check_tensors(const fp8gmm_norm_tensor* tensors, int n, bool out) {
  if (n < 0) return FP8GMM_ERR_BAD_ARGUMENT;
  if (n > 0 && tensors == nullptr) return FP8GMM_ERR_NULL_POINTER;
  int64_t all = 0;   // bounds the chunks of a launch, and fits the table's bits, as an address has to
  for (int i = 0; i < n; ++i) {
    const fp8gmm_norm_tensor& t = tensors[i];
    if (!known_type(t.type) || (out && t.out_type != t.type && t.out_type != FP8GMM_TYPE_FP32)) return FP8GMM_ERR_BAD_FORMAT;
    if (t.count < 0 || t.count >= ((int64_t)1 << 40) - all) return FP8GMM_ERR_BAD_SHAPE;
    all += t.count;
    if (t.count > 0 && (t.in == nullptr || (out && t.out == nullptr))) return FP8GMM_ERR_NULL_POINTER;
    const int64_t mask = type_bytes(t.type) - 1, out_mask = out ? type_bytes(t.out_type) - 1 : 0;
    if ((reinterpret_cast<uintptr_t>(t.in) & mask) || (out && (reinterpret_cast<uintptr_t>(t.out) & out_mask)))
      return FP8GMM_ERR_ALIGNMENT;
    if (reinterpret_cast<uintptr_t>(t.in) >> 48 || (out && reinterpret_cast<uintptr_t>(t.out) >> 48)) return FP8GMM_ERR_BAD_ARGUMENT;
  }
  return FP8GMM_OK;
}

// Nothing is written that another tensor of the call reads or writes: a result lies apart from all else, or in the place of its own
// tensor.
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
  const auto before = [](const Range& a, const Range& b) { return a.begin < b.begin; };
  if (!std::is_sorted(ranges.begin(), ranges.end(), before)) std::sort(ranges.begin(), ranges.end(), before);   // buckets are
  uintptr_t written = 0, read = 0;   // ends of what the ranges so far write and read
  for (const Range& r : ranges) {
    if (r.begin < written || (r.writes && r.begin < read)) return FP8GMM_ERR_BAD_ARGUMENT;
    (r.writes ? written : read) = std::max(r.writes ? written : read, r.end);
  }
  return FP8GMM_OK;
}

// The tensors with elements, as the launches take them.
struct List {
  std::vector<Entry> entries;
  uint32_t chunks = 0;
  int64_t bytes_in = 0, bytes_out = 0;
  bool in_place = true;   // all of them
  bool wider = false;     // some in fp32 of 16 bits
  List(const fp8gmm_norm_tensor* tensors, int n) {
    entries.reserve((size_t)n);
    for (int i = 0; i < n; ++i) {
      const fp8gmm_norm_tensor& t = tensors[i];
      if (t.count == 0) continue;
      entries.push_back({t.in, t.out, t.count, chunks, (uint16_t)t.type, (uint16_t)t.out_type});
      chunks += chunks_of(t.count, t.type);
      bytes_in += t.count * type_bytes(t.type);
      bytes_out += t.count * type_bytes(t.out_type);
      in_place = in_place && t.in == t.out;
      wider = wider || t.out_type != t.type;
    }
  }
  int n() const { return (int)entries.size(); }
  bool direct() const { return n() <= kTensors; }
  // The list in units, where there are no more than one workgroup takes: their number, or -1.
  int small(Units* units) const {
    int k = 0;
    for (const Entry& e : entries) {
      const int size = type_bytes(e.type), most = 64 * kPieces * 16 / size;
      if (e.count > (int64_t)(kUnits - k) * most) return -1;
      for (int64_t at = 0; at < e.count; at += most)
        units->u[k++] = {static_cast<const char*>(e.in) + at * size, static_cast<char*>(e.out) + at * type_bytes(e.out_type),
                         (int32_t)std::min<int64_t>(most, e.count - at), e.type, e.out_type};
    }
    return k;
  }
  int blocks() const { return (int)std::min<uint32_t>(kNormBlocks, (chunks + kRun - 1) / kRun); }
  Part part() const {
    Part p = {};
    std::copy(entries.begin(), entries.end(), p.e);
    return p;
  }
  PackedPart packed(int first) const {
    PackedPart p = {};
    for (int i = 0; i < std::min(kPacked, n() - first); ++i) {
      const Entry& e = entries[first + i];
      const uint64_t in = reinterpret_cast<uintptr_t>(e.in), out = reinterpret_cast<uintptr_t>(e.out);
      for (int k = 0; k < 3; ++k) {
        p.e[i].part[k] = (uint16_t)(in >> 16 * k);
        p.e[i].part[3 + k] = (uint16_t)(out >> 16 * k);
        p.e[i].part[6 + k] = (uint16_t)((uint64_t)e.count >> 16 * k);
      }
      p.e[i].part[8] |= (uint16_t)(e.type << 8 | e.out_type << 12);
    }
    return p;
  }
};

// The workspace: the partial sums, the factor, and the table behind them.
double* partials_of(void* workspace) { return static_cast<double*>(workspace); }
float* factor_at(void* workspace) { return reinterpret_cast<float*>(partials_of(workspace) + kNormBlocks); }
Entry* table_of(void* workspace) { return reinterpret_cast<Entry*>(partials_of(workspace) + kNormBlocks + 2); }

// Enqueues the partial sums of a list that is not empty; the table of a short one, for the scaling.
Part launch_norm(const List& list, bool stream, void* workspace, hipStream_t s) {
  if (!list.direct())
    for (int first = 0; first < list.n(); first += kPacked)
      hipLaunchKernelGGL(multi_norm_table_kernel, dim3(1), dim3(kPackedThreads), 0, s, list.packed(first),
                         std::min(kPacked, list.n() - first), list.entries[first].begin, table_of(workspace) + first);
  const Part part = list.direct() ? list.part() : Part{};
  auto* kernel = list.direct() ? stream ? &multi_norm_kernel<true, true> : &multi_norm_kernel<true, false>
                 : stream      ? &multi_norm_kernel<false, true>
                               : &multi_norm_kernel<false, false>;
  hipLaunchKernelGGL(kernel, dim3(list.blocks()), dim3(kThreads), 0, s, part, table_of(workspace), list.n(), list.chunks,
                     partials_of(workspace));
  return part;
}

void launch_finish(const List& list, double max_norm, float* norm, float* factor, void* workspace, hipStream_t s) {
  hipLaunchKernelGGL(multi_norm_finish_kernel, dim3(1), dim3(1024), 0, s, partials_of(workspace), list.blocks(), max_norm, norm, factor);
}

// Whether the list was a short one, which is enqueued then
bool launch_small(const List& list, bool clip, double max_norm, float* norm, hipStream_t s) {
  Units units = {};
  const int n = list.small(&units);
  if (n >= 0) hipLaunchKernelGGL(multi_small_kernel, dim3(1), dim3(kUnitWaves * 64), 0, s, units, n, clip, max_norm, norm);
  return n >= 0;
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
  const List list(tensors, n);
  if (!launch_small(list, false, 0., norm, s)) {
    launch_norm(list, list.bytes_in > kStreamOnce, workspace, s);
    launch_finish(list, 0., norm, nullptr, workspace, s);
  }
  return hipGetLastError() == hipSuccess ? FP8GMM_OK : FP8GMM_ERR_LAUNCH;
}

int multi_clip(const fp8gmm_norm_tensor* tensors, int n, double max_norm, float* norm, void* workspace, size_t bytes,
               hipStream_t s) {
  int rc = check_tensors(tensors, n, true);
  if (rc == FP8GMM_OK) rc = norm == nullptr ? FP8GMM_ERR_NULL_POINTER : check_workspace(n, workspace, bytes);
  if (rc == FP8GMM_OK && !(max_norm >= 0.)) rc = FP8GMM_ERR_BAD_ARGUMENT;
  if (rc == FP8GMM_OK) rc = check_apart(tensors, n);
  if (rc != FP8GMM_OK) return rc;
  const List list(tensors, n);
  if (launch_small(list, true, max_norm, norm, s)) return hipGetLastError() == hipSuccess ? FP8GMM_OK : FP8GMM_ERR_LAUNCH;
  const bool in = list.bytes_in > kStreamTwice, out = list.bytes_out > kStreamOut;
  const Part part = launch_norm(list, in, workspace, s);
  float* const finished = list.blocks() > kFewPartials ? factor_at(workspace) : nullptr;
  if (finished != nullptr) launch_finish(list, max_norm, norm, finished, workspace, s);
  const auto launch = [&](auto parts) {
    constexpr int PARTS = decltype(parts)::value;
    auto* kernel = list.direct() ? in    ? &multi_clip_kernel<true, true, true, PARTS>
                                   : out ? &multi_clip_kernel<true, false, true, PARTS>
                                         : &multi_clip_kernel<true, false, false, PARTS>
                   : in  ? &multi_clip_kernel<false, true, true, PARTS>
                   : out ? &multi_clip_kernel<false, false, true, PARTS>
                         : &multi_clip_kernel<false, false, false, PARTS>;
    hipLaunchKernelGGL(kernel, dim3(std::min<uint32_t>(list.chunks, kClipBlocks / PARTS) * PARTS), dim3(kThreads), 0, s, part,
                       table_of(workspace), list.n(), list.chunks, partials_of(workspace), list.blocks(), max_norm, finished,
                       list.in_place, norm);
  };
  list.wider ? launch(std::integral_constant<int, kWiderParts>{}) : launch(std::integral_constant<int, 1>{});
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
  return n < 0 ? 0 : (kNormBlocks + 2) * sizeof(double) + (n > kTensors ? (size_t)n * sizeof(Entry) : 0);
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
