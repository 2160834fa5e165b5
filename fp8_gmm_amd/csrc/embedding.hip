// Rows of a table by token id, scaled, and the table's gradient by sorted tokens, for gfx950: what stands in front of the
// first routed layer of a model (layers.py, embedding).
//
//   y[t, :] = s w[id t, :]        dw[v, :] = s * (sum of dy[t, :] over the tokens t with id v)
//
// An id outside the table has a row of zeros and no gradient; the padding id has its row and no gradient.
//
// The lookup is bound by memory: every row passes once.  So is the gradient, by the table, which is written whole, and the
// rows of dy.  Its sums have an order that does not change from run to run: the tokens are sorted by id (stable, a radix sort
// of digits of at most 9 bits), a wavefront takes a chunk of neighbouring sorted tokens and 64 pieces of 16 bytes of
// their columns and keeps the sum of the present id in fp32.  A run of one id inside a chunk is rounded and written at once;
// one that crosses chunks leaves fp32 partial sums, which a second launch adds up in order.  The zeros of the rows without
// tokens are written by workgroups that ride along with the launches of the sort: the sort is bound by latency and leaves the
// memory idle.
#include <algorithm>

#include "elements.h"

namespace fp8gmm {
namespace {

constexpr int kMaxDigit = 9;                        // bits of a pass of the sort
constexpr int kBins = 1 << kMaxDigit;
constexpr int kSortWaves = 16;                      // the sort in one workgroup: so many wavefronts ..
constexpr int kSortSteps = 16;                      // .. that hold so many tokens per lane
constexpr int kSortMax = kSortWaves * kSortSteps * 64;
constexpr int kSortPlaceBits = 14;                  // of a token's place there, packed with its id into 32 bits
static_assert(kSortMax == 1 << kSortPlaceBits, "a place of the list in its bits");
constexpr int kPlaceWaves = 4;                      // longer lists: wavefronts of a workgroup
constexpr int kPlaceChunk = kPlaceWaves * kSortSteps * 64;
constexpr int kScanThreads = kBins;
constexpr int kFillBlocks = 1024;                   // workgroups of 256 threads that write zeros beside a launch of the sort
constexpr int kLookupPieces = 4;                    // pieces per lane of the lookup
constexpr int kSumWaves = 4;
constexpr int kSumMaxChunk = 32;                    // sorted tokens of a wavefront
constexpr int kSumMinChunk = 8;

// The id's key in the sort: `table` (the last one) for what takes no part.
template <typename Id>
__device__ __forceinline__ uint32_t key_of(Id id, int64_t table, int64_t padding) {
  return id >= 0 && (int64_t)id < table && (int64_t)id != padding ? (uint32_t)id : (uint32_t)table;
}

// ---- lookup ----------------------------------------------------------------------------------------------------------
template <int TYPE, typename Id, int LANES>   // lanes to a row
__global__ __launch_bounds__(256) void embedding_kernel(const Id* __restrict__ ids, int64_t n, const void* __restrict__ weight,
                                                        int64_t table, int cols, float scale, void* __restrict__ y) {
  typedef Elements<TYPE> E;
  typedef typename E::bits bits;
  constexpr int V = E::kVec, ROWS = 256 / LANES;
  const int lane = threadIdx.x % LANES;
  const int64_t t = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES;
  if (t >= n) return;
  const int64_t id = ids[t];
  const bool in = id >= 0 && id < table;
  const bits* const w = static_cast<const bits*>(weight) + (in ? id : 0) * cols;
  bits* const out = static_cast<bits*>(y) + t * cols;
  const int first = blockIdx.y * LANES * kLookupPieces;
  u32x4 raw[kLookupPieces];
#pragma unroll
  for (int u = 0; u < kLookupPieces; ++u) {
    const int at = (first + u * LANES + lane) * V;
    raw[u] = E::load(w + at, in ? cols - at : 0);
  }
#pragma unroll
  for (int u = 0; u < kLookupPieces; ++u) {
    const int at = (first + u * LANES + lane) * V;
    if (scale != 1.f && in) {
      float f[V];
      E::unpack(raw[u], f);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] *= scale;
      raw[u] = E::pack(f);
    }
    E::store(out + at, cols - at, raw[u]);
  }
}

// ---- zeros -----------------------------------------------------------------------------------------------------------
struct Fill {
  u32x4* base;          // on 16 bytes
  int64_t first, last;  // pieces of 16 bytes
  int tail;             // bytes behind `last`, of the last share
};

__device__ __forceinline__ void fill_zeros(const Fill& f, int block, int blocks) {
  const int64_t step = (int64_t)blocks * blockDim.x;
  int64_t i = f.first + (int64_t)block * blockDim.x + threadIdx.x;
  const u32x4 zero = {0u, 0u, 0u, 0u};
  for (; i + 3 * step < f.last; i += 4 * step) {
#pragma unroll
    for (int u = 0; u < 4; ++u) f.base[i + u * step] = zero;
  }
  for (; i < f.last; i += step) f.base[i] = zero;
  if (block == 0 && (int)threadIdx.x < f.tail) reinterpret_cast<uint8_t*>(f.base + f.last)[threadIdx.x] = 0;
}

__global__ __launch_bounds__(256) void embedding_fill_kernel(Fill fill) { fill_zeros(fill, blockIdx.x, gridDim.x); }

// ---- sort ------------------------------------------------------------------------------------------------------------
// The lanes that hold the same digit as this one
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, bool valid, int bits) {
  uint64_t same = __ballot(valid);
  for (int k = 0; k < bits; ++k) {
    const bool set = (digit >> k) & 1;
    const uint64_t has = __ballot(valid && set);
    same &= set ? has : ~has;
  }
  return same;
}

// Where this lane's entry goes: `next` is the wavefront's own table of the next place of every digit, which moves on.  The
// wavefront's LDS operations are carried out in their order; the fences keep the compiler to it.
__device__ __forceinline__ int place_of(int* next, uint32_t digit, bool valid, int bits, uint64_t below) {
  const uint64_t same = same_digit(digit, valid, bits);
  const int before = __popcll(same & below);
  const int place = valid ? next[digit] + before : 0;
  asm volatile("" ::: "memory");
  if (valid && before == 0) next[digit] = place + __popcll(same);
  asm volatile("" ::: "memory");
  return place;
}

// Exclusive prefix sums over the 512 bins, one to a thread of the first 512; every thread of the workgroup calls it.
__device__ __forceinline__ int bins_before(int count, int* wave_sums) {
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  int incl = count;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int other = __shfl_up(incl, d, 64);
    if (lane >= d) incl += other;
  }
  if (wave < kBins / 64 && lane == 63) wave_sums[wave] = incl;
  __syncthreads();
  int before = incl - count;
#pragma unroll
  for (int w = 0; w < kBins / 64; ++w)
    if (w < wave) before += wave_sums[w];
  return before;
}

// A list of at most kSortMax tokens and 18 bits of id, by the first workgroup: the entries stay in registers, (id, place)
// packed into a word, and go through LDS once a pass.  The other workgroups write zeros.
template <typename Id>
__global__ __launch_bounds__(kSortWaves * 64) void embedding_sort_kernel(const Id* __restrict__ ids, int n, int64_t table,
                                                                         int64_t padding, int passes, int digit_bits,
                                                                         int32_t* __restrict__ keys, int32_t* __restrict__ places,
                                                                         Fill fill) {
  __shared__ int next[kSortWaves][kBins];
  __shared__ uint32_t entries[kSortMax];
  __shared__ int wave_sums[kBins / 64];
  if (blockIdx.x > 0) {
    fill_zeros(fill, blockIdx.x - 1, gridDim.x - 1);
    return;
  }
  const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const int steps = (n + kSortWaves * 64 - 1) / (kSortWaves * 64);   // at most kSortSteps
  const int base = wave * steps * 64 + lane;
  const uint64_t below = (1ull << lane) - 1ull;
  const uint32_t mask = (1u << digit_bits) - 1u;
  uint32_t v[kSortSteps];
#pragma unroll
  for (int r = 0; r < kSortSteps; ++r) {
    const int i = base + r * 64;
    v[r] = r < steps && i < n ? key_of(ids[i], table, padding) << kSortPlaceBits | (uint32_t)i : 0u;
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = kSortPlaceBits + pass * digit_bits;
    for (int b = lane; b < kBins; b += 64) next[wave][b] = 0;
    asm volatile("" ::: "memory");   // the wavefront's own table, in its own order
#pragma unroll
    for (int r = 0; r < kSortSteps; ++r)
      if (r < steps && base + r * 64 < n) atomicAdd(&next[wave][v[r] >> shift & mask], 1);
    __syncthreads();
    int run = 0;
    if (tid < kBins) {
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) {
        const int c = next[w][tid];
        next[w][tid] = run;
        run += c;
      }
    }
    const int before = bins_before(tid < kBins ? run : 0, wave_sums);
    if (tid < kBins) {
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) next[w][tid] += before;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortSteps; ++r) {
      if (r >= steps) continue;
      const bool valid = base + r * 64 < n;
      const int place = place_of(next[wave], v[r] >> shift & mask, valid, digit_bits, below);
      if (valid) entries[place] = v[r];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortSteps; ++r)
      if (r < steps && base + r * 64 < n) v[r] = entries[base + r * 64];
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < kSortSteps; ++r)
    if (r < steps && base + r * 64 < n) {
      keys[base + r * 64] = (int32_t)(v[r] >> kSortPlaceBits);
      places[base + r * 64] = (int32_t)(v[r] & (uint32_t)(kSortMax - 1));
    }
}

// One pass of the sort of a longer list in three launches, as the router's (router.hip): the digits of every chunk are counted,
// the counts become starts, and a stable placement.  `keys_in` == NULL: the first pass, on the ids themselves.
template <typename Id>
struct PassInput {
  const Id* ids;
  const int32_t *keys, *places;
  int64_t table, padding;
  __device__ __forceinline__ uint32_t key(int64_t i) const { return keys != nullptr ? (uint32_t)keys[i] : key_of(ids[i], table, padding); }
  __device__ __forceinline__ int32_t place(int64_t i) const { return keys != nullptr ? places[i] : (int32_t)i; }
};

template <typename Id>
__global__ __launch_bounds__(kPlaceWaves * 64) void embedding_count_kernel(PassInput<Id> in, int n, int chunks, int shift,
                                                                           int digit_bits, int32_t* __restrict__ counts, Fill fill) {
  __shared__ int bins[kBins];
  if ((int)blockIdx.x >= chunks) {
    fill_zeros(fill, blockIdx.x - chunks, gridDim.x - chunks);
    return;
  }
  for (int b = threadIdx.x; b < kBins; b += kPlaceWaves * 64) bins[b] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kPlaceChunk + threadIdx.x;
  const uint32_t mask = (1u << digit_bits) - 1u;
#pragma unroll
  for (int r = 0; r < kSortSteps; ++r) {
    const int64_t i = base + r * kPlaceWaves * 64;
    if (i < n) atomicAdd(&bins[in.key(i) >> shift & mask], 1);
  }
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += kPlaceWaves * 64) counts[(int64_t)blockIdx.x * kBins + b] = bins[b];
}

// counts[chunk][bin] becomes the place of the chunk's first entry of that digit
__global__ __launch_bounds__(kScanThreads) void embedding_scan_kernel(int32_t* __restrict__ counts, int chunks, Fill fill) {
  __shared__ int wave_sums[kBins / 64];
  if (blockIdx.x > 0) {
    fill_zeros(fill, blockIdx.x - 1, gridDim.x - 1);
    return;
  }
  const int bin = threadIdx.x;
  int total = 0;
#pragma unroll 16
  for (int c = 0; c < chunks; ++c) total += counts[(int64_t)c * kBins + bin];
  int run = bins_before(total, wave_sums);
#pragma unroll 16
  for (int c = 0; c < chunks; ++c) {
    const int count = counts[(int64_t)c * kBins + bin];
    counts[(int64_t)c * kBins + bin] = run;
    run += count;
  }
}

template <typename Id>
__global__ __launch_bounds__(kPlaceWaves * 64) void embedding_place_kernel(PassInput<Id> in, int n, int chunks, int shift,
                                                                           int digit_bits, const int32_t* __restrict__ starts,
                                                                           int32_t* __restrict__ keys, int32_t* __restrict__ places,
                                                                           Fill fill) {
  __shared__ int next[kPlaceWaves][kBins];
  if ((int)blockIdx.x >= chunks) {
    fill_zeros(fill, blockIdx.x - chunks, gridDim.x - chunks);
    return;
  }
  const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const int64_t base = (int64_t)blockIdx.x * kPlaceChunk + wave * kSortSteps * 64 + lane;   // a wavefront's entries are neighbours
  const uint64_t below = (1ull << lane) - 1ull;
  const uint32_t mask = (1u << digit_bits) - 1u;
  uint32_t key[kSortSteps];
  int32_t from[kSortSteps];
#pragma unroll
  for (int r = 0; r < kSortSteps; ++r) {
    const int64_t i = base + r * 64;
    key[r] = i < n ? in.key(i) : 0u;
    from[r] = i < n ? in.place(i) : 0;
  }
  for (int b = lane; b < kBins; b += 64) next[wave][b] = 0;
  asm volatile("" ::: "memory");   // the wavefront's own table, in its own order
#pragma unroll
  for (int r = 0; r < kSortSteps; ++r)
    if (base + r * 64 < n) atomicAdd(&next[wave][key[r] >> shift & mask], 1);
  __syncthreads();
  for (int b = tid; b < kBins; b += kPlaceWaves * 64) {
    int run = starts[(int64_t)blockIdx.x * kBins + b];
#pragma unroll
    for (int w = 0; w < kPlaceWaves; ++w) {
      const int c = next[w][b];
      next[w][b] = run;
      run += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kSortSteps; ++r) {
    const bool valid = base + r * 64 < n;
    const int place = place_of(next[wave], key[r] >> shift & mask, valid, digit_bits, below);
    if (valid) {
      keys[place] = (int32_t)key[r];
      places[place] = from[r];
    }
  }
}

// ---- sums ------------------------------------------------------------------------------------------------------------
// parts: [chunk][2][cols], fp32: of the run that comes in from the chunk before, and of the one that goes on into the next.
template <int TYPE>
__global__ __launch_bounds__(kSumWaves * 64) void embedding_sum_kernel(const int32_t* __restrict__ keys,
                                                                       const int32_t* __restrict__ places, int n, int chunk,
                                                                       int slices, const void* __restrict__ dy_, int64_t table,
                                                                       int cols, float scale, void* __restrict__ dw_,
                                                                       float* __restrict__ parts) {
  typedef Elements<TYPE> E;
  typedef typename E::bits bits;
  constexpr int V = E::kVec, AHEAD = kSumMinChunk;
  const int lane = threadIdx.x % 64;
  const uint32_t unit = blockIdx.x * kSumWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int c = unit / slices, slice = unit - c * slices;
  const int64_t p0 = (int64_t)c * chunk;
  if (p0 >= n) return;
  const int count = min((int64_t)chunk, n - p0);
  const int at = (slice * 64 + lane) * V;
  const int mine = cols - at;   // elements of the row from here on
  const int32_t key = lane < count ? keys[p0 + lane] : (int32_t)table;
  const int32_t place = lane < count ? places[p0 + lane] : 0;
  const int32_t before = p0 > 0 ? keys[p0 - 1] : -1, behind = p0 + count < n ? keys[p0 + count] : -1;
  const bits* const dy = static_cast<const bits*>(dy_) + at;
  float sum[V] = {};
  int32_t id = __builtin_amdgcn_readfirstlane(key);
  int from = 0;   // the present run's first entry
  const auto flush = [&](int to) {
    if (id == (int32_t)table) return;
    const bool comes = from == 0 && before == id, goes = to == count && behind == id;
    if (!comes && !goes) {
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] *= scale;
      E::store(static_cast<bits*>(dw_) + (int64_t)id * cols + at, mine, E::pack(sum));
    } else {
      float* const out = parts + ((int64_t)c * 2 + (comes ? 0 : 1)) * cols + at;
#pragma unroll
      for (int q = 0; q < V / 4; ++q)
        Elements<FP8GMM_TYPE_FP32>::store(reinterpret_cast<uint32_t*>(out) + q * 4, mine - q * 4,
                                          u32x4{__float_as_uint(sum[4 * q]), __float_as_uint(sum[4 * q + 1]),
                                                __float_as_uint(sum[4 * q + 2]), __float_as_uint(sum[4 * q + 3])});
    }
  };
#pragma unroll 1
  for (int i0 = 0; i0 < count; i0 += AHEAD) {
    u32x4 raw[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const bool live = __builtin_amdgcn_readlane(key, i0 + j) != (int32_t)table;   // entries past the end are none's
      raw[j] = E::load(dy + (int64_t)__builtin_amdgcn_readlane(place, i0 + j) * cols, live ? mine : 0);
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int32_t next = __builtin_amdgcn_readlane(key, i0 + j);
      if (i0 + j < count && next != id) {
        flush(i0 + j);
        id = next;
        from = i0 + j;
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] = 0.f;
      }
      float f[V];
      E::unpack(raw[j], f);
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] += f[i];
    }
  }
  flush(count);
}

// A run that crosses chunks: the workgroup of the chunk that it begins in adds its partial sums up, a quarter of them to a
// wavefront, and the quarters in their order.
template <int TYPE>
__global__ __launch_bounds__(kSumWaves * 64) void embedding_join_kernel(const int32_t* __restrict__ keys, int n, int chunk,
                                                                        int64_t table, int cols, float scale,
                                                                        const float* __restrict__ parts, void* __restrict__ dw_) {
  typedef Elements<TYPE> E;
  typedef typename E::bits bits;
  __shared__ float quarters[kSumWaves][64];
  const int64_t p0 = (int64_t)blockIdx.x * chunk, p1 = p0 + chunk;
  if (p1 >= n) return;
  const int32_t id = keys[p1 - 1];
  if (id == (int32_t)table || keys[p1] != id || (p0 > 0 && keys[p0 - 1] == id)) return;
  int64_t lo = p1, hi = n - 1;   // the run's last entry
  while (lo < hi) {
    const int64_t mid = (lo + hi + 1) / 2;
    if (keys[mid] <= id) lo = mid;
    else hi = mid - 1;
  }
  const int more = (int)(lo / chunk - blockIdx.x);   // chunks behind this one
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int per = (more + 1 + kSumWaves - 1) / kSumWaves, last = min(more + 1, (wave + 1) * per);
  for (int64_t col = blockIdx.y * 64 + lane; col - lane < cols; col += (int64_t)gridDim.y * 64) {
    float sum = 0.f;
    if (col < cols) {
#pragma unroll 8
      for (int k = wave * per; k < last; ++k) sum += parts[((int64_t)(blockIdx.x + k) * 2 + (k == 0 ? 1 : 0)) * cols + col];
    }
    quarters[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && col < cols) {
#pragma unroll
      for (int w = 1; w < kSumWaves; ++w) sum += quarters[w][lane];
      static_cast<bits*>(dw_)[(int64_t)id * cols + col] = E::pack1(sum * scale);
    }
    __syncthreads();
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int check_embedding(int64_t n, int64_t table, int cols, int type) {
  if (!known_type(type)) return FP8GMM_ERR_BAD_FORMAT;
  // keys below 2^31, offsets of a row in 32 bits, a grid of fewer than 2^32 threads
  if (n < 0 || n > (1 << 28) || table < 0 || table >= INT32_MAX || cols < 0 || cols > (1 << 24)) return FP8GMM_ERR_BAD_SHAPE;
  return FP8GMM_OK;
}

int slices_of(int cols, int type) { return (int)ceil_div(cols, 64 * 16 / type_bytes(type)); }

// Sorted tokens of a wavefront: few where longer chunks would leave the chip short of wavefronts.
int chunk_of(int64_t n, int cols, int type) {
  return ceil_div(n, kSumMaxChunk) * slices_of(cols, type) >= 4096 ? kSumMaxChunk : kSumMinChunk;
}

struct Layout {   // of the workspace
  int key_bits, passes, digit_bits, chunk;
  bool one;   // the sort in one workgroup
  int64_t chunks, sort_chunks;
  size_t list, counts, parts, bytes;   // bytes of a list of the sort; offsets of the counts and the partial sums
};
Layout layout_of(int64_t n, int64_t table, int cols, int type) {
  Layout l{};
  while (l.key_bits < 31 && (table >> l.key_bits) != 0) ++l.key_bits;   // keys of 0 .. table
  l.one = n <= kSortMax && l.key_bits + kSortPlaceBits <= 32;
  l.passes = (int)ceil_div(l.key_bits, kMaxDigit);
  l.digit_bits = (int)ceil_div(l.key_bits, std::max(l.passes, 1));
  l.chunk = chunk_of(n, cols, type);
  l.chunks = ceil_div(n, l.chunk);
  l.sort_chunks = ceil_div(n, kPlaceChunk);
  l.list = (size_t)ceil_div(n * 4, 256) * 256;
  l.counts = l.list * (l.one ? 2 : 4);   // keys and places, twice where a pass reads from memory what another wrote
  l.parts = l.counts + (l.one ? 0 : (size_t)l.sort_chunks * kBins * 4);
  l.bytes = l.parts + (size_t)l.chunks * 2 * cols * 4;
  return l;
}

}  // namespace
}  // namespace fp8gmm

extern "C" {

int fp8gmm_embedding(const void* ids, int ids64, int64_t n, const void* weight, int64_t table, int cols, float scale, int type,
                     void* y, void* stream) {
  using namespace fp8gmm;
  const int rc = check_embedding(n, table, cols, type);
  if (rc != FP8GMM_OK) return rc;
  if (n == 0 || cols == 0) return FP8GMM_OK;
  if (ids == nullptr || y == nullptr || (weight == nullptr && table > 0)) return FP8GMM_ERR_NULL_POINTER;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t pieces = ceil_div(cols, 16 / type_bytes(type));
  const int lanes = pieces <= 16 * kLookupPieces ? 16 : 64;
  const unsigned segments = (unsigned)ceil_div(pieces, lanes * kLookupPieces);
  const int64_t slab = 1 << 22;   // tokens of a launch: a grid has fewer than 2^32 threads
  for (int64_t t0 = 0; t0 < n; t0 += slab) {
    const int64_t m = std::min(slab, n - t0);
    const dim3 grid((unsigned)ceil_div(m, 256 / lanes), segments);
    const void* const from = static_cast<const char*>(ids) + t0 * (ids64 ? 8 : 4);
    void* const to = static_cast<char*>(y) + t0 * cols * type_bytes(type);
#define FP8GMM_LOOKUP(TYPE, ID, LANES)                                                                                   \
  hipLaunchKernelGGL((embedding_kernel<TYPE, ID, LANES>), grid, dim3(256), 0, s, static_cast<const ID*>(from), m, weight, \
                     table, cols, scale, to)
#define FP8GMM_LOOKUP_OF(TYPE)                           \
  if (type == TYPE) {                                    \
    if (ids64) {                                         \
      if (lanes == 16) FP8GMM_LOOKUP(TYPE, int64_t, 16); \
      else FP8GMM_LOOKUP(TYPE, int64_t, 64);             \
    } else {                                             \
      if (lanes == 16) FP8GMM_LOOKUP(TYPE, int32_t, 16); \
      else FP8GMM_LOOKUP(TYPE, int32_t, 64);             \
    }                                                    \
  }
    FP8GMM_LOOKUP_OF(FP8GMM_TYPE_BF16)
    FP8GMM_LOOKUP_OF(FP8GMM_TYPE_FP16)
    FP8GMM_LOOKUP_OF(FP8GMM_TYPE_FP32)
#undef FP8GMM_LOOKUP_OF
#undef FP8GMM_LOOKUP
  }
  return hipGetLastError() == hipSuccess ? FP8GMM_OK : FP8GMM_ERR_LAUNCH;
}

size_t fp8gmm_embedding_workspace_bytes(int64_t n, int64_t table, int cols, int type) {
  using namespace fp8gmm;
  if (check_embedding(n, table, cols, type) != FP8GMM_OK || n == 0 || cols == 0 || table == 0) return 0;
  return layout_of(n, table, cols, type).bytes;
}

int fp8gmm_embedding_backward(const void* ids, int ids64, int64_t n, const void* dy, void* dweight, int64_t table, int cols,
                              float scale, int64_t padding, int type, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace fp8gmm;
  const int rc = check_embedding(n, table, cols, type);
  if (rc != FP8GMM_OK) return rc;
  if (table == 0 || cols == 0) return FP8GMM_OK;
  if (dweight == nullptr || (n > 0 && (ids == nullptr || dy == nullptr || workspace == nullptr))) return FP8GMM_ERR_NULL_POINTER;
  if ((reinterpret_cast<uintptr_t>(dweight) & 15) || (reinterpret_cast<uintptr_t>(workspace) & 15)) return FP8GMM_ERR_ALIGNMENT;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t bytes = table * cols * type_bytes(type), pieces = bytes / 16;
  if (n == 0) {
    const Fill all = {static_cast<u32x4*>(dweight), 0, pieces, (int)(bytes % 16)};
    hipLaunchKernelGGL(embedding_fill_kernel, dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>(2048, ceil_div(pieces, 1024)))),
                       dim3(256), 0, s, all);
    return hipGetLastError() == hipSuccess ? FP8GMM_OK : FP8GMM_ERR_LAUNCH;
  }
  const Layout l = layout_of(n, table, cols, type);
  if (workspace_bytes < l.bytes) return FP8GMM_ERR_WORKSPACE;
  char* const work = static_cast<char*>(workspace);
  int32_t* lists[2][2];
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2; ++j) lists[i][j] = reinterpret_cast<int32_t*>(work + l.list * (l.one ? j : 2 * i + j));
  const int launches = l.one ? 1 : 3 * l.passes;
  int launch = 0;
  // a launch's share of the zeros, and the workgroups of `threads` threads that write it
  const auto share = [&](int threads, unsigned* blocks) {
    const Fill f = {static_cast<u32x4*>(dweight), pieces * launch / launches, pieces * (launch + 1) / launches,
                    launch + 1 == launches ? (int)(bytes % 16) : 0};
    ++launch;
    *blocks = (unsigned)std::max<int64_t>(1, std::min<int64_t>(kFillBlocks * 256 / threads - 1, ceil_div(f.last - f.first, threads * 4)));
    return f;
  };
  const auto sort = [&](auto* typed) {
    typedef std::remove_const_t<std::remove_pointer_t<decltype(typed)>> Id;
    unsigned extra;
    if (l.one) {
      const Fill f = share(kSortWaves * 64, &extra);
      hipLaunchKernelGGL(embedding_sort_kernel<Id>, dim3(1 + extra), dim3(kSortWaves * 64), 0, s, typed, (int)n, table, padding,
                         l.passes, l.digit_bits, lists[0][0], lists[0][1], f);
      return 0;
    }
    int32_t* const counts = reinterpret_cast<int32_t*>(work + l.counts);
    const int chunks = (int)l.sort_chunks;
    PassInput<Id> in = {typed, nullptr, nullptr, table, padding};
    int to = 0;
    for (int pass = 0; pass < l.passes; ++pass) {
      const int shift = pass * l.digit_bits;
      Fill f = share(kPlaceWaves * 64, &extra);
      hipLaunchKernelGGL(embedding_count_kernel<Id>, dim3(chunks + extra), dim3(kPlaceWaves * 64), 0, s, in, (int)n, chunks, shift,
                         l.digit_bits, counts, f);
      f = share(kScanThreads, &extra);
      hipLaunchKernelGGL(embedding_scan_kernel, dim3(1 + extra), dim3(kScanThreads), 0, s, counts, chunks, f);
      f = share(kPlaceWaves * 64, &extra);
      hipLaunchKernelGGL(embedding_place_kernel<Id>, dim3(chunks + extra), dim3(kPlaceWaves * 64), 0, s, in, (int)n, chunks, shift,
                         l.digit_bits, counts, lists[to][0], lists[to][1], f);
      in.keys = lists[to][0];
      in.places = lists[to][1];
      to ^= 1;
    }
    return to ^ 1;
  };
  const int at = ids64 ? sort(static_cast<const int64_t*>(ids)) : sort(static_cast<const int32_t*>(ids));
  const int32_t *const keys = lists[at][0], *const places = lists[at][1];
  float* const parts = reinterpret_cast<float*>(work + l.parts);
  const int slices = slices_of(cols, type);
  const unsigned sums = (unsigned)ceil_div(l.chunks * slices, kSumWaves);
  const dim3 joins((unsigned)l.chunks, (unsigned)std::min<int64_t>(64, ceil_div(cols, 64)));
#define FP8GMM_SUMS(TYPE)                                                                                                     \
  if (type == TYPE) {                                                                                                         \
    hipLaunchKernelGGL(embedding_sum_kernel<TYPE>, dim3(sums), dim3(kSumWaves * 64), 0, s, keys, places, (int)n, l.chunk, slices, \
                       dy, table, cols, scale, dweight, parts);                                                               \
    if (l.chunks > 1)                                                                                                         \
      hipLaunchKernelGGL(embedding_join_kernel<TYPE>, joins, dim3(kSumWaves * 64), 0, s, keys, (int)n, l.chunk, table, cols,  \
                         scale, parts, dweight);                                                                              \
  }
  FP8GMM_SUMS(FP8GMM_TYPE_BF16)
  FP8GMM_SUMS(FP8GMM_TYPE_FP16)
  FP8GMM_SUMS(FP8GMM_TYPE_FP32)
#undef FP8GMM_SUMS
  return hipGetLastError() == hipSuccess ? FP8GMM_OK : FP8GMM_ERR_LAUNCH;
}

}  // extern "C"
