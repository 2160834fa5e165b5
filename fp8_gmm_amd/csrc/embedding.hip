// Rows of a table by token id, scaled, and the table's gradient by sorted tokens, for gfx950: what stands in front of the
// first routed layer of a model (layers.py, embedding).
//
//   y[t, :] = s w[id t, :]        dw[v, :] = s * (sum of dy[t, :] over the tokens t with id v)
//
// An id outside the table has a row of zeros and no gradient; the padding id has its row and no gradient.
//
// The lookup is bound by memory: every row passes once.  So is the gradient, by the table, which is written whole, and the
// rows of dy.  Its sums have an order that does not change from run to run: the tokens are sorted by id (stable, a radix sort
// of digits of at most 9 bits), and a wavefront takes the runs of one id that begin in its chunk of neighbouring sorted tokens, for
// 64 pieces of 16 bytes of their columns, and keeps the present run's sum in fp32.  A run of up to 32 tokens is its wavefront's
// to the end, and is rounded and written at once; a longer one leaves fp32 partial sums of every chunk that it crosses, which a
// second launch adds up in order.  The zeros of the rows without tokens are written by workgroups that ride along with the
// launches of the sort: the sort is bound by latency and leaves the memory idle.
#include <algorithm>

#include "elements.h"

namespace fp8gmm {
namespace {

constexpr int kFewTokens = 1024;                    // of a batch whose gradient is one launch,
constexpr int64_t kFewTokenBytes = 1 << 20;         // .. and its bytes, which one row's may all be,
constexpr int64_t kFewTableBytes = 128 << 20;       // .. and the table's
constexpr int kFewRows = 4096;                      // the most rows of the table of a workgroup of it ..
constexpr int64_t kFewBytes = 32 << 10;             // .. and their bytes, but for a single row
constexpr int kMaxDigit = 9;                        // bits of a pass of the sort
constexpr int kBins = 1 << kMaxDigit;
constexpr int kSortWaves = 16;                      // the sort in one workgroup: so many wavefronts ..
constexpr int kSortSteps = 16;                      // .. that hold so many tokens per lane
constexpr int kSortMax = kSortWaves * kSortSteps * 64;
constexpr int kSortPlaceBits = 14;                  // of a token's place there, packed with its id into 32 bits
static_assert(kSortMax == 1 << kSortPlaceBits, "a place of the list in its bits");
constexpr int64_t kSortZeros = 128 << 20;           // the least bytes of a table whose zeros outlast the sort of more than half of those
constexpr int kPlaceWaves = 16;                     // longer lists: wavefronts of a workgroup, and their tokens per lane
constexpr int kPlaceSteps = 2;
constexpr int kPlaceChunk = kPlaceWaves * kPlaceSteps * 64;
constexpr int kScanThreads = kBins;
// Chunks of which every workgroup adds the counts up for itself; those of more have a launch for that.  Gradients of rows of 16
// columns without it and with it: 196608 tokens (96 chunks) 57 and 67 us, 2^20 188 and 224, 3/2 2^20 (768) 323 and 323, 2^22 1160
// and 785.
constexpr int kManyChunks = 768;
constexpr int kFillBlocks = 16384;                  // the most workgroups of 256 threads that write zeros beside a launch of the sort
constexpr int kLookupPieces = 4;                    // pieces per lane of the lookup
constexpr int kSumWaves = 4;
constexpr int kSumMaxChunk = 32;                    // sorted tokens of a wavefront
constexpr int kSumMinChunk = 8;
// Tokens: a run of more is shared out by chunks (65536 tokens of a text, table 8000 x 1024, bf16: 62 us; with runs of 8 and more
// shared out 64).
constexpr int kLongRun = 32;
// Chunks whose long runs a workgroup of the join looks for, and its wavefronts, to which it shares a run out: 16384 tokens of one id,
// 1024 columns, 56 us; by 1 chunk 66, by 16 chunks 81, by 4 wavefronts 112.  30000 of a text over 100 ids, 2048 columns: 60; 75,
// 56, 65.
constexpr int kJoinChunks = 4;
constexpr int kJoinWaves = 16;
// Of a result that outgrows the cache: written with the streaming hint (16384 rows of 4096, bf16, 134 MB: 32 us, without it 40).
constexpr int64_t kStreamBytes = (int64_t)64 << 20;

// The id's key in the sort: `table` (the last one) for what takes no part.
template <typename Id>
__device__ __forceinline__ uint32_t key_of(Id id, int64_t table, int64_t padding) {
  return id >= 0 && (int64_t)id < table && (int64_t)id != padding ? (uint32_t)id : (uint32_t)table;
}

// ---- lookup ----------------------------------------------------------------------------------------------------------
// Where the piece of a lane begins, and how many elements it has.  Rows of at least one piece: the last piece ends where the row
// ends, and lanes behind the end have it too - what is loaded and stored twice are the same bits, and nothing branches.
template <int V, bool SHORT>
__device__ __forceinline__ int piece_at(int at, int cols) { return SHORT ? at : min(at, cols - V); }
template <int V, bool SHORT>
__device__ __forceinline__ int piece_size(int at, int cols) { return SHORT ? cols - at : V; }

// LANES lanes to a row, PIECES of a row's pieces to each, of as many rows as make kLookupPieces together (2^20 rows of 64 columns,
// bf16: 50 us, with 4 pieces of one row, most of them the last one again, 93; 2^19 of 256 columns 43 and 55).  A row behind the last
// one is the last one once more.
template <int TYPE, typename Id, int LANES, int PIECES, bool SHORT, bool STREAM>
__global__ __launch_bounds__(256) void embedding_kernel(const Id* __restrict__ ids, int64_t n, const void* __restrict__ weight,
                                                        int64_t table, int cols, float scale, void* __restrict__ y) {
  typedef Elements<TYPE> E;
  typedef typename E::bits bits;
  constexpr int V = E::kVec, ROWS = 256 / LANES, TURNS = kLookupPieces / PIECES;
  const int lane = threadIdx.x % LANES;
  const int first = blockIdx.y * LANES * PIECES;
  int64_t row[TURNS], id[TURNS];
#pragma unroll
  for (int k = 0; k < TURNS; ++k) {
    row[k] = min((int64_t)blockIdx.x * ROWS * TURNS + k * ROWS + threadIdx.x / LANES, n - 1);
    id[k] = ids[row[k]];
  }
  u32x4 raw[TURNS][PIECES];
#pragma unroll
  for (int k = 0; k < TURNS; ++k) {
    const bool in = id[k] >= 0 && id[k] < table;
    const bits* const w = static_cast<const bits*>(weight) + (in ? id[k] : 0) * cols;
    if (in) {
#pragma unroll
      for (int u = 0; u < PIECES; ++u) {
        const int at = piece_at<V, SHORT>((first + u * LANES + lane) * V, cols);
        raw[k][u] = E::load(w + at, piece_size<V, SHORT>(at, cols));
      }
    } else {
#pragma unroll
      for (int u = 0; u < PIECES; ++u) raw[k][u] = u32x4{0u, 0u, 0u, 0u};
    }
  }
#pragma unroll
  for (int k = 0; k < TURNS; ++k)
#pragma unroll
    for (int u = 0; u < PIECES; ++u) {
      const int at = piece_at<V, SHORT>((first + u * LANES + lane) * V, cols);
      if (scale != 1.f) {
        float f[V];
        E::unpack(raw[k][u], f);
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] *= scale;
        raw[k][u] = E::pack(f);
      }
      E::template store<STREAM>(static_cast<bits*>(y) + row[k] * cols + at, piece_size<V, SHORT>(at, cols), raw[k][u]);
    }
}

// ---- zeros -----------------------------------------------------------------------------------------------------------
struct Fill {
  u32x4* base;          // on 16 bytes
  int64_t first, last;  // pieces of 16 bytes
  int tail;             // bytes behind `last`, of the last share
};

// With the streaming hint: 32000 x 4096, bf16, 262 MB: 32 us, without it 49.
__device__ __forceinline__ void fill_zeros(const Fill& f, int block, int blocks) {
  const int threads = blockDim.x;
  const u32x4 zero = {0u, 0u, 0u, 0u};
  for (int64_t at = f.first + (int64_t)block * threads * 4; at < f.last; at += (int64_t)blocks * threads * 4) {
    u32x4* const p = f.base + at + threadIdx.x;
    if (at + threads * 4 <= f.last) {
#pragma unroll
      for (int u = 0; u < 4; ++u) __builtin_nontemporal_store(zero, p + u * threads);
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (at + u * threads + (int)threadIdx.x < f.last) p[u * threads] = zero;
    }
  }
  if (block == 0 && (int)threadIdx.x < f.tail) reinterpret_cast<uint8_t*>(f.base + f.last)[threadIdx.x] = 0;
}

__global__ __launch_bounds__(256) void embedding_fill_kernel(Fill fill) { fill_zeros(fill, blockIdx.x, gridDim.x); }

// ---- sort ------------------------------------------------------------------------------------------------------------
// The lanes that hold the same digit as this one, found bit by bit: one ballot for each.
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, bool valid, int bits) {
  uint64_t same = __ballot(valid);
#pragma unroll
  for (int k = 0; k < kMaxDigit; ++k)
    if (k < bits) same &= ~(__ballot((digit >> k & 1) != 0) ^ (0ull - (uint64_t)(digit >> k & 1)));
  return same;
}

// How many of the wavefront's entries so far have this lane's digit: `count` is the wavefront's own table, which moves on.  One of
// the lanes with the same digit counts for all (a few frequent ids make most lanes the same: 16384 tokens of a text took 64 us to
// sort with an atomic for each, of evenly spread ids 45).  The wavefront's LDS operations are carried out in their order; the
// fences keep the compiler to it.
__device__ __forceinline__ int rank_of(int* count, uint32_t digit, bool valid, int bits, uint64_t below) {
  const uint64_t same = same_digit(digit, valid, bits);
  const int before = __popcll(same & below);
  const int rank = valid ? count[digit] + before : 0;
  asm volatile("" ::: "memory");
  if (valid && before == 0) count[digit] = rank + __popcll(same);
  asm volatile("" ::: "memory");
  return rank;
}

// Exclusive prefix sums over the workgroup's threads, of which the first 512 count; every thread calls it.
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
// packed into a word, and go through LDS once a pass.  The other workgroups write zeros.  Gradients by this sort and by the next
// one, whose passes are two launches each: 2048 tokens, table 8000 x 1024, bf16, 21.6 and 28.3 us; 4096, 50000 x 1024, 28.6 and 36.9;
// 8192, 38 and 41; 10000, 42.6 and 43.9; 12000, 8000 x 512, 36.7 and 32.4; 16384, 44 and 35 - but where there are zeros enough to
// write meanwhile, 32000 x 4096, 90.5 and 102.
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
    int rank[kSortSteps];
#pragma unroll
    for (int r = 0; r < kSortSteps; ++r)
      if (r < steps) rank[r] = rank_of(next[wave], v[r] >> shift & mask, base + r * 64 < n, digit_bits, below);
    __syncthreads();
    int run = 0;
    if (tid < kBins) {   // a digit's entries: the wavefronts' one behind the other
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
      if (r < steps && base + r * 64 < n) entries[next[wave][v[r] >> shift & mask] + rank[r]] = v[r];
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

// One pass of the sort of a longer list: the digits of every chunk are counted, and a stable placement.  Every workgroup of the
// placement adds the counts up for itself; those of many chunks become starts in a launch of their own.  Without `keys`: the first
// pass, on the ids themselves.
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
  const uint64_t below = (1ull << (threadIdx.x % 64)) - 1ull;
  const uint32_t mask = (1u << digit_bits) - 1u;
  uint32_t key[kPlaceSteps];
#pragma unroll
  for (int r = 0; r < kPlaceSteps; ++r) {
    const int64_t i = base + r * kPlaceWaves * 64;
    key[r] = i < n ? in.key(i) : 0u;
  }
#pragma unroll
  for (int r = 0; r < kPlaceSteps; ++r) {
    const bool valid = base + r * kPlaceWaves * 64 < n;
    const uint32_t digit = key[r] >> shift & mask;
    const uint64_t same = same_digit(digit, valid, digit_bits);
    if (valid && (same & below) == 0) atomicAdd(&bins[digit], __popcll(same));
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
                                                                           int digit_bits, const int32_t* __restrict__ counts,
                                                                           bool scanned, int32_t* __restrict__ keys,
                                                                           int32_t* __restrict__ places, Fill fill) {
  __shared__ int next[kPlaceWaves][kBins];
  __shared__ int wave_sums[kBins / 64];
  if ((int)blockIdx.x >= chunks) {
    fill_zeros(fill, blockIdx.x - chunks, gridDim.x - chunks);
    return;
  }
  const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const int64_t base = (int64_t)blockIdx.x * kPlaceChunk + wave * kPlaceSteps * 64 + lane;   // a wavefront's entries are neighbours
  const uint64_t below = (1ull << lane) - 1ull;
  const uint32_t mask = (1u << digit_bits) - 1u;
  uint32_t key[kPlaceSteps];
  int32_t from[kPlaceSteps];
#pragma unroll
  for (int r = 0; r < kPlaceSteps; ++r) {
    const int64_t i = base + r * 64;
    key[r] = i < n ? in.key(i) : 0u;
    from[r] = i < n ? in.place(i) : 0;
  }
  for (int b = lane; b < kBins; b += 64) next[wave][b] = 0;
  asm volatile("" ::: "memory");   // the wavefront's own table, in its own order
  int rank[kPlaceSteps];
#pragma unroll
  for (int r = 0; r < kPlaceSteps; ++r) rank[r] = rank_of(next[wave], key[r] >> shift & mask, base + r * 64 < n, digit_bits, below);
  // where the chunk's entries of a digit begin: behind those of lower digits, and those of the chunks before
  static_assert(kBins <= kPlaceWaves * 64, "a bin to a thread");
  int start = 0;
  if (scanned) {
    if (tid < kBins) start = counts[(int64_t)blockIdx.x * kBins + tid];
  } else {
    int total = 0;
    if (tid < kBins) {
#pragma unroll 16
      for (int c = 0; c < chunks; ++c) {
        const int count = counts[(int64_t)c * kBins + tid];
        start += c < (int)blockIdx.x ? count : 0;
        total += count;
      }
    }
    start += bins_before(total, wave_sums);
  }
  __syncthreads();
  if (tid < kBins) {
#pragma unroll
    for (int w = 0; w < kPlaceWaves; ++w) {
      const int c = next[w][tid];
      next[w][tid] = start;
      start += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kPlaceSteps; ++r) {
    if (base + r * 64 < n) {
      const int place = next[wave][key[r] >> shift & mask] + rank[r];
      keys[place] = (int32_t)key[r];
      places[place] = from[r];
    }
  }
}

// ---- sums ------------------------------------------------------------------------------------------------------------
// What a chunk left of long runs: one that begins in it and goes on; one that comes in, and whether that goes on.
enum { kBegins = 1, kGoesOn = 2 };

// parts: [chunk][2][cols], fp32: of the long run that comes in from the chunk before, and of the one that begins and goes on into
// the next.  flags: [chunk].
template <int TYPE, bool SHORT>
__global__ __launch_bounds__(kSumWaves * 64) void embedding_sum_kernel(const int32_t* __restrict__ keys,
                                                                       const int32_t* __restrict__ places, int n, int chunk,
                                                                       int slices, const void* __restrict__ dy_, int table,
                                                                       int cols, float scale, void* __restrict__ dw_,
                                                                       float* __restrict__ parts, int32_t* __restrict__ flags) {
  typedef Elements<TYPE> E;
  typedef typename E::bits bits;
  constexpr int V = E::kVec, AHEAD = kSumMinChunk;
  const int lane = threadIdx.x % 64;
  const uint32_t unit = blockIdx.x * kSumWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int c = unit / slices, slice = unit - c * slices;
  const int64_t p0 = (int64_t)c * chunk;
  if (p0 >= n) return;
  const int count = (int)min((int64_t)chunk, n - p0);
  // the chunk's entries and what follows them, 128 in all, and the 64 in front; -1: none
  const auto key_at = [&](int64_t p) { return p >= 0 && p < n ? keys[p] : -1; };
  const int32_t front = key_at(p0 - 64 + lane), key0 = key_at(p0 + lane), key1 = key_at(p0 + 64 + lane);
  const int32_t place0 = p0 + lane < n ? places[p0 + lane] : 0, place1 = p0 + 64 + lane < n ? places[p0 + 64 + lane] : 0;
  const auto held = [&](int32_t key, int32_t id) { return __popcll(__ballot(key == id)); };
  const int32_t first = __builtin_amdgcn_readlane(key0, 0), last = __builtin_amdgcn_readlane(key0, count - 1);
  const int before = held(front, first);   // equal ones are neighbours
  const bool comes = before > 0 && first != table;
  const bool comes_long = comes && before + held(key0, first) + held(key1, first) > kLongRun;
  int begin = 0, end = count;
  if (comes && !comes_long) begin = min(held(key0, first), count);   // another wavefront's
  // the chunk's last run: to its end, or as far as the chunk where it is long
  const int more = __popcll(__ballot(key0 == last && lane >= count)) + held(key1, last);
  const bool goes = more > 0 && last != table && begin < count;
  const bool goes_long = goes && (comes_long && first == last || held(key0, last) + held(key1, last) > kLongRun);
  if (goes && !goes_long) end = count + more;
  // keys of `table` take no part; they stand at the end
  end = min(end, __popcll(__ballot(key0 >= 0 && key0 < table)) + __popcll(__ballot(key1 >= 0 && key1 < table)));
  const bool all = comes_long && first == last;   // the chunk lies inside one long run, which may end with it
  if (slice == 0 && lane == 0) flags[c] = (goes_long && !all ? kBegins : 0) | (goes_long && all ? kGoesOn : 0);
  if (begin >= end) return;

  const int at = piece_at<V, SHORT>((slice * 64 + lane) * V, cols), mine = piece_size<V, SHORT>(at, cols);
  const bits* const dy = static_cast<const bits*>(dy_) + at;
  const auto key_of_entry = [&](int i) { return i < 64 ? __builtin_amdgcn_readlane(key0, i) : __builtin_amdgcn_readlane(key1, i - 64); };
  u32x4 next[AHEAD];
  const auto load = [&](int i0) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int i = min(i0 + j, end - 1);
      const int32_t place = i < 64 ? __builtin_amdgcn_readlane(place0, i) : __builtin_amdgcn_readlane(place1, i - 64);
      next[j] = E::template load<true>(dy + (int64_t)place * cols, mine);
    }
  };
  load(begin);
  float sum[V] = {};
  int32_t id = key_of_entry(begin);
  bool head = comes_long;   // the present run came in
  const auto flush = [&](bool tail) {
    if (!head && !tail) {
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] *= scale;
      E::template store<true>(static_cast<bits*>(dw_) + (int64_t)id * cols + at, mine, E::pack(sum));
    } else {
      uint32_t* const out = reinterpret_cast<uint32_t*>(parts + ((int64_t)c * 2 + (head ? 0 : 1)) * cols + at);
#pragma unroll
      for (int q = 0; q < V / 4; ++q)
        Elements<FP8GMM_TYPE_FP32>::store(out + q * 4, mine - q * 4,
                                          u32x4{__float_as_uint(sum[4 * q]), __float_as_uint(sum[4 * q + 1]),
                                                __float_as_uint(sum[4 * q + 2]), __float_as_uint(sum[4 * q + 3])});
    }
  };
#pragma unroll 1
  for (int i0 = begin; i0 < end; i0 += AHEAD) {
    u32x4 raw[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) raw[j] = next[j];
    if (i0 + AHEAD < end) load(i0 + AHEAD);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (i0 + j >= end) break;
      const int32_t k = key_of_entry(i0 + j);
      if (k != id) {
        flush(false);
        id = k;
        head = false;
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] = 0.f;
      }
      float f[V];
      E::unpack(raw[j], f);
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] += f[i];
    }
  }
  flush(goes_long);
}

// A long run: its partial sums, from the chunk that it begins in on, a share of them to a wavefront, and the shares in their
// order.  A workgroup has 256 columns of the runs that begin in its chunks.
template <int TYPE>
__global__ __launch_bounds__(kJoinWaves * 64) void embedding_join_kernel(const int32_t* __restrict__ keys, int chunks, int chunk,
                                                                        int cols, float scale, const float* __restrict__ parts,
                                                                        const int32_t* __restrict__ flags, void* __restrict__ dw_) {
  typedef Elements<TYPE> E;
  typedef Elements<FP8GMM_TYPE_FP32> F;
  typedef typename E::bits bits;
  __shared__ u32x4 shares[kJoinWaves][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int c0 = blockIdx.x * kJoinChunks;
  const int32_t flag = lane < kJoinChunks && c0 + lane < chunks ? flags[c0 + lane] : 0;
  for (uint64_t owners = __ballot(flag & kBegins); owners != 0; owners &= owners - 1) {
    const int c = c0 + __builtin_ctzll(owners);
    int more = 1;   // chunks behind this one: those that the run goes on through, and the one where it ends
    for (int at = c + 1;; at += 64) {
      const uint64_t ends = ~__ballot(at + lane < chunks && (flags[at + lane] & kGoesOn) != 0);
      more += ends != 0 ? __builtin_ctzll(ends) : 64;
      if (ends != 0) break;
    }
    const int per = (more + 1 + kJoinWaves - 1) / kJoinWaves, last = min(more + 1, (wave + 1) * per);
    const int64_t col = (int64_t)blockIdx.y * 256 + lane * 4;
    const int mine = (int)min((int64_t)4, cols - col);
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int k = wave * per; k < last; ++k) {
      const u32x4 part = F::load(reinterpret_cast<const uint32_t*>(parts) + ((int64_t)(c + k) * 2 + (k == 0 ? 1 : 0)) * cols + col, mine);
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] += __uint_as_float(part[i]);
    }
    shares[wave][lane] = __builtin_bit_cast(u32x4, sum);
    __syncthreads();
    const int64_t own = (int64_t)blockIdx.y * 256 + threadIdx.x;
    if (threadIdx.x < 256 && own < cols) {
      float total = 0.f;
#pragma unroll
      for (int w = 0; w < kJoinWaves; ++w) total += __uint_as_float(shares[w][threadIdx.x / 4][threadIdx.x % 4]);
      static_cast<bits*>(dw_)[(int64_t)keys[(int64_t)(c + 1) * chunk - 1] * cols + own] = E::pack1(total * scale);
    }
    __syncthreads();
  }
}

// ---- few tokens ------------------------------------------------------------------------------------------------------
// The whole gradient in one launch: a workgroup has some rows of the table, looks for their tokens in the list, a token to a
// thread, and writes zeros to the rows without.  The first token of a row in the workgroup's list is its sum's, for 64 pieces of
// the columns a wavefront, over the row's tokens in their order; a row of more than 64 tokens is shared out by 64 entries of the
// list to a wavefront.  Bound by latency, its own and the host's, which has three launches fewer.  Short batches, call to call, by
// this launch and by the sort: 1000 tokens of 4001 x 256, fp32, 8.6 and 18.4 us; 500 of 50000 x 65, bf16, 7.0 and 18.3; 1000 of a
// million rows of 64, bf16, 21 and 43; but all of 1024 tokens of 512 columns the same, 25 and 15.  A table of 262 MB is written
// faster beside the sort (41 us, 49).
template <int V>
struct RowSum {
  float f[V];
};
// Adds the rows of dy of the tokens of the lanes `those`, in the order of the lanes
template <int TYPE>
__device__ __forceinline__ void add_entries(uint64_t those, int token, const typename Elements<TYPE>::bits* dy, int cols, int size,
                                            RowSum<Elements<TYPE>::kVec>& sum) {
  typedef Elements<TYPE> E;
  constexpr int V = E::kVec, AHEAD = 8;
  while (those != 0) {
    u32x4 raw[AHEAD];
    const int count = min(__popcll(those), AHEAD);
    int last = 0;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {   // the last one again in the place of none
      if (j < count) {
        last = __builtin_amdgcn_readlane(token, __builtin_ctzll(those));
        those &= those - 1;
      }
      raw[j] = E::load(dy + (int64_t)last * cols, size);
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (j >= count) continue;
      float f[V];
      E::unpack(raw[j], f);
#pragma unroll
      for (int q = 0; q < V; ++q) sum.f[q] += f[q];
    }
  }
}

template <int TYPE, typename Id, bool SHORT>
__global__ __launch_bounds__(kFewTokens) void embedding_few_kernel(const Id* __restrict__ ids, int n, const void* __restrict__ dy_,
                                                                   void* __restrict__ dw_, int64_t table, int rows_each, int cols,
                                                                   float scale, int64_t padding) {
  typedef Elements<TYPE> E;
  typedef typename E::bits bits;
  constexpr int V = E::kVec, WAVES = kFewTokens / 64;
  __shared__ int row_of[kFewTokens], token_of[kFewTokens], counts[WAVES];
  __shared__ int tokens_of[kFewRows];             // a row's tokens
  __shared__ int many[kFewTokens / 64], n_many;   // rows of more than 64 tokens, in any order
  __shared__ RowSum<V> shares[WAVES][64];
  const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const int64_t r0 = (int64_t)blockIdx.x * rows_each;
  const int rows = (int)min((int64_t)rows_each, table - r0);
  for (int r = tid; r < rows; r += kFewTokens) tokens_of[r] = 0;
  if (tid == 0) n_many = 0;
  const uint32_t row = (tid < n ? key_of(ids[tid], table, padding) : (uint32_t)table) - (uint32_t)r0;
  const bool here = row < (uint32_t)rows;   // the key of none is no row of any workgroup
  const uint64_t mask = __ballot(here);
  if (lane == 0) counts[wave] = __popcll(mask);
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    before += w < wave ? counts[w] : 0;
    total += counts[w];
  }
  if (here) {
    const int at = before + __popcll(mask & ((1ull << lane) - 1ull));
    row_of[at] = (int)row;
    token_of[at] = tid;
    if (atomicAdd(&tokens_of[row], 1) == 64) many[atomicAdd(&n_many, 1)] = (int)row;
  }
  __syncthreads();
  bits* const dw = static_cast<bits*>(dw_) + r0 * cols;
  const int pieces = (cols + V - 1) / V, rows_on = kFewTokens / pieces, pieces_on = kFewTokens % pieces;
  for (int r = tid / pieces, piece = tid % pieces; r < rows;) {
    if (tokens_of[r] == 0) {
      const int at = piece_at<V, SHORT>(piece * V, cols);
      E::template store<true>(dw + (int64_t)r * cols + at, piece_size<V, SHORT>(at, cols), u32x4{0u, 0u, 0u, 0u});
    }
    r += rows_on;
    piece += pieces_on;
    if (piece >= pieces) {
      piece -= pieces;
      ++r;
    }
  }
  const int slices = (pieces + 63) / 64;
  const auto finish = [&](RowSum<V>& sum, int r, int at, int size) {
#pragma unroll
    for (int q = 0; q < V; ++q) sum.f[q] *= scale;
    E::store(dw + (int64_t)r * cols + at, size, E::pack(sum.f));
  };
  for (int unit = wave; unit < total * slices; unit += WAVES) {
    const int i = unit / slices, slice = unit - i * slices;
    const int mine = __builtin_amdgcn_readfirstlane(row_of[i]);
    if (__builtin_amdgcn_readfirstlane(tokens_of[mine]) > 64) continue;
    bool first = true;
    for (int j0 = 0; j0 < i && first; j0 += 64) first = __ballot(j0 + lane < i && row_of[j0 + lane] == mine) == 0;
    if (!first) continue;
    const int at = piece_at<V, SHORT>((slice * 64 + lane) * V, cols), size = piece_size<V, SHORT>(at, cols);
    RowSum<V> sum = {};
    for (int j0 = i & ~63; j0 < total; j0 += 64)
      add_entries<TYPE>(__ballot(j0 + lane < total && row_of[j0 + lane] == mine), token_of[j0 + lane], static_cast<const bits*>(dy_) + at,
                        cols, size, sum);
    finish(sum, mine, at, size);
  }
  // as many slices at a time as there are wavefronts for their shares
  const int groups = (total + 63) / 64, at_once = WAVES / max(groups, 1);
  for (int m = 0; m < n_many; ++m) {
    const int mine = __builtin_amdgcn_readfirstlane(many[m]);
    for (int first = 0; first < slices; first += at_once) {
      const int slice = first + wave / groups, j0 = wave % groups * 64;
      const bool busy = slice < slices && wave < at_once * groups;
      const int at = piece_at<V, SHORT>((slice * 64 + lane) * V, cols), size = piece_size<V, SHORT>(at, cols);
      RowSum<V> sum = {};
      if (busy)
        add_entries<TYPE>(__ballot(j0 + lane < total && row_of[j0 + lane] == mine), token_of[j0 + lane], static_cast<const bits*>(dy_) + at,
                          cols, size, sum);
      __syncthreads();   // the shares before have been added up
      shares[wave][lane] = sum;
      __syncthreads();
      if (!busy || j0 != 0) continue;
      for (int w = wave + 1; w < wave + groups; ++w)
#pragma unroll
        for (int q = 0; q < V; ++q) sum.f[q] += shares[w][lane].f[q];
      finish(sum, mine, at, size);
    }
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int check_embedding(int64_t n, int64_t table, int cols, int type) {
  if (!known_type(type)) return FP8GMM_ERR_BAD_FORMAT;
  // keys below 2^31, offsets of a row in 32 bits, a grid of fewer than 2^32 threads
  if (n < 0 || n > (1 << 28) || table < 0 || table >= INT32_MAX || cols < 0 || cols > (1 << 23)) return FP8GMM_ERR_BAD_SHAPE;
  return FP8GMM_OK;
}

int slices_of(int cols, int type) { return (int)ceil_div(cols, 64 * 16 / type_bytes(type)); }

// Rows of the table of a workgroup where the gradient is one launch, or 0: a workgroup for every compute unit, and more of a table
// that is large.
int few_rows(int64_t n, int64_t table, int cols, int type) {
  const int64_t row = (int64_t)cols * type_bytes(type);
  if (n > kFewTokens || n * row > kFewTokenBytes || table * row > kFewTableBytes) return 0;
  const int64_t most = std::min<int64_t>(kFewRows, std::max<int64_t>(1, kFewBytes / row));
  return (int)std::max<int64_t>(1, std::min(most, ceil_div(table, 256)));
}

// Sorted tokens of a wavefront: few where longer chunks would leave the chip short of wavefronts (2048 tokens of 1024 columns, bf16,
// by 8 tokens 21.6 us, by 32 25; 32768 tokens 51.5 and 44; 65536 of 256 columns 47 and 41.5; 65536 of 1024 75 and 62).
int chunk_of(int64_t n, int cols, int type) {
  return ceil_div(n, kSumMaxChunk) * slices_of(cols, type) >= 1024 ? kSumMaxChunk : kSumMinChunk;
}

struct Layout {   // of the workspace
  int key_bits, passes, digit_bits, chunk;
  bool one;   // the sort in one workgroup
  int64_t chunks, sort_chunks;
  size_t list, counts, flags, parts, bytes;   // bytes of a list of the sort; offsets of the counts, flags and partial sums
};
Layout layout_of(int64_t n, int64_t table, int cols, int type) {
  Layout l{};
  while (l.key_bits < 31 && (table >> l.key_bits) != 0) ++l.key_bits;   // keys of 0 .. table
  l.one = n <= kSortMax && l.key_bits + kSortPlaceBits <= 32 &&
          (n <= kSortMax / 2 || table * cols * type_bytes(type) >= kSortZeros);
  l.passes = (int)ceil_div(l.key_bits, kMaxDigit);
  l.digit_bits = (int)ceil_div(l.key_bits, std::max(l.passes, 1));
  l.chunk = chunk_of(n, cols, type);
  l.chunks = ceil_div(n, l.chunk);
  l.sort_chunks = ceil_div(n, kPlaceChunk);
  l.list = (size_t)ceil_div(n * 4, 256) * 256;
  l.counts = l.list * (l.one ? 2 : 4);   // keys and places, twice where a pass reads from memory what another wrote
  l.flags = l.counts + (l.one ? 0 : (size_t)l.sort_chunks * kBins * 4);
  l.parts = l.flags + (size_t)ceil_div(l.chunks * 4, 16) * 16;
  l.bytes = l.parts + (size_t)l.chunks * 2 * cols * 4;
  return l;
}

}  // namespace
}  // namespace fp8gmm

extern "C" {

int fp8gmm_embedding(const void* ids, int ids64_, int64_t n, const void* weight, int64_t table, int cols, float scale, int type,
                     void* y, void* stream) {
  using namespace fp8gmm;
  const int rc = check_embedding(n, table, cols, type);
  if (rc != FP8GMM_OK) return rc;
  const bool ids64 = ids64_ != 0, stream_out = n * cols * type_bytes(type) > kStreamBytes;
  if (n == 0 || cols == 0) return FP8GMM_OK;
  if (ids == nullptr || y == nullptr || (weight == nullptr && table > 0)) return FP8GMM_ERR_NULL_POINTER;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t pieces = ceil_div(cols, 16 / type_bytes(type));
  const int lanes = pieces <= 16 * kLookupPieces ? 16 : 64, each = pieces <= 16 ? 1 : pieces <= 32 ? 2 : kLookupPieces;
  const int rows = 256 / lanes * (kLookupPieces / each);   // of a workgroup
  const unsigned segments = (unsigned)ceil_div(pieces, lanes * each);
  const int64_t slab = 1 << 22;   // tokens of a launch: a grid has fewer than 2^32 threads
  for (int64_t t0 = 0; t0 < n; t0 += slab) {
    const int64_t m = std::min(slab, n - t0);
    const dim3 grid((unsigned)ceil_div(m, rows), segments);
    const void* const from = static_cast<const char*>(ids) + t0 * (ids64 ? 8 : 4);
    void* const to = static_cast<char*>(y) + t0 * cols * type_bytes(type);
#define FP8GMM_LOOKUP_AS(TYPE, ID, STREAM)                                                                                 \
  (cols < Elements<TYPE>::kVec ? &embedding_kernel<TYPE, ID, 16, 1, true, STREAM>                                          \
   : each == 1                 ? &embedding_kernel<TYPE, ID, 16, 1, false, STREAM>                                         \
   : each == 2                 ? &embedding_kernel<TYPE, ID, 16, 2, false, STREAM>                                         \
   : lanes == 16               ? &embedding_kernel<TYPE, ID, 16, kLookupPieces, false, STREAM>                             \
                               : &embedding_kernel<TYPE, ID, 64, kLookupPieces, false, STREAM>)
#define FP8GMM_LOOKUP_OF(TYPE, ID)                                                                                         \
  if (type == TYPE && ids64 == (sizeof(ID) == 8)) {                                                                        \
    auto* kernel = stream_out ? FP8GMM_LOOKUP_AS(TYPE, ID, true) : FP8GMM_LOOKUP_AS(TYPE, ID, false);                      \
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, static_cast<const ID*>(from), m, weight, table, cols, scale, to);    \
  }
    FP8GMM_LOOKUP_OF(FP8GMM_TYPE_BF16, int64_t)
    FP8GMM_LOOKUP_OF(FP8GMM_TYPE_FP16, int64_t)
    FP8GMM_LOOKUP_OF(FP8GMM_TYPE_FP32, int64_t)
    FP8GMM_LOOKUP_OF(FP8GMM_TYPE_BF16, int32_t)
    FP8GMM_LOOKUP_OF(FP8GMM_TYPE_FP16, int32_t)
    FP8GMM_LOOKUP_OF(FP8GMM_TYPE_FP32, int32_t)
#undef FP8GMM_LOOKUP_OF
#undef FP8GMM_LOOKUP_AS
  }
  return hipGetLastError() == hipSuccess ? FP8GMM_OK : FP8GMM_ERR_LAUNCH;
}

size_t fp8gmm_embedding_workspace_bytes(int64_t n, int64_t table, int cols, int type) {
  using namespace fp8gmm;
  if (check_embedding(n, table, cols, type) != FP8GMM_OK || n == 0 || cols == 0 || table == 0) return 0;
  return few_rows(n, table, cols, type) > 0 ? 0 : layout_of(n, table, cols, type).bytes;
}

int fp8gmm_embedding_backward(const void* ids, int ids64, int64_t n, const void* dy, void* dweight, int64_t table, int cols,
                              float scale, int64_t padding, int type, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace fp8gmm;
  const int rc = check_embedding(n, table, cols, type);
  if (rc != FP8GMM_OK) return rc;
  if (table == 0 || cols == 0) return FP8GMM_OK;
  const int each = few_rows(n, table, cols, type);
  if (dweight == nullptr || (n > 0 && (ids == nullptr || dy == nullptr || (each == 0 && workspace == nullptr)))) return FP8GMM_ERR_NULL_POINTER;
  if ((reinterpret_cast<uintptr_t>(dweight) & 15) || (reinterpret_cast<uintptr_t>(workspace) & 15)) return FP8GMM_ERR_ALIGNMENT;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t bytes = table * cols * type_bytes(type), pieces = bytes / 16;
  if (n == 0) {
    const Fill all = {static_cast<u32x4*>(dweight), 0, pieces, (int)(bytes % 16)};
    hipLaunchKernelGGL(embedding_fill_kernel, dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>(2048, ceil_div(pieces, 1024)))),
                       dim3(256), 0, s, all);
    return hipGetLastError() == hipSuccess ? FP8GMM_OK : FP8GMM_ERR_LAUNCH;
  }
  if (each > 0) {
    const dim3 grid((unsigned)ceil_div(table, each));
#define FP8GMM_FEW(TYPE, ID)                                                                                                   \
  if (type == TYPE && (ids64 != 0) == (sizeof(ID) == 8)) {                                                                     \
    auto* kernel = cols < Elements<TYPE>::kVec ? &embedding_few_kernel<TYPE, ID, true> : &embedding_few_kernel<TYPE, ID, false>; \
    hipLaunchKernelGGL(kernel, grid, dim3(kFewTokens), 0, s, static_cast<const ID*>(ids), (int)n, dy, dweight, table, each, cols, \
                       scale, padding);                                                                                        \
  }
    FP8GMM_FEW(FP8GMM_TYPE_BF16, int64_t)
    FP8GMM_FEW(FP8GMM_TYPE_FP16, int64_t)
    FP8GMM_FEW(FP8GMM_TYPE_FP32, int64_t)
    FP8GMM_FEW(FP8GMM_TYPE_BF16, int32_t)
    FP8GMM_FEW(FP8GMM_TYPE_FP16, int32_t)
    FP8GMM_FEW(FP8GMM_TYPE_FP32, int32_t)
#undef FP8GMM_FEW
    return hipGetLastError() == hipSuccess ? FP8GMM_OK : FP8GMM_ERR_LAUNCH;
  }
  const Layout l = layout_of(n, table, cols, type);
  if (workspace_bytes < l.bytes) return FP8GMM_ERR_WORKSPACE;
  char* const work = static_cast<char*>(workspace);
  int32_t* lists[2][2];
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2; ++j) lists[i][j] = reinterpret_cast<int32_t*>(work + l.list * (l.one ? j : 2 * i + j));
  const bool scanned = l.sort_chunks > kManyChunks;
  const int launches = l.one ? 1 : (scanned ? 3 : 2) * l.passes;
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
      if (scanned) {
        f = share(kScanThreads, &extra);
        hipLaunchKernelGGL(embedding_scan_kernel, dim3(1 + extra), dim3(kScanThreads), 0, s, counts, chunks, f);
      }
      f = share(kPlaceWaves * 64, &extra);
      hipLaunchKernelGGL(embedding_place_kernel<Id>, dim3(chunks + extra), dim3(kPlaceWaves * 64), 0, s, in, (int)n, chunks, shift,
                         l.digit_bits, counts, scanned, lists[to][0], lists[to][1], f);
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
  int32_t* const flags = reinterpret_cast<int32_t*>(work + l.flags);
  const dim3 joins((unsigned)ceil_div(l.chunks, kJoinChunks), (unsigned)ceil_div(cols, 256));
#define FP8GMM_SUMS(TYPE)                                                                                                      \
  if (type == TYPE) {                                                                                                          \
    auto* kernel = cols < Elements<TYPE>::kVec ? &embedding_sum_kernel<TYPE, true> : &embedding_sum_kernel<TYPE, false>;       \
    hipLaunchKernelGGL(kernel, dim3(sums), dim3(kSumWaves * 64), 0, s, keys, places, (int)n, l.chunk, slices, dy, (int)table,  \
                       cols, scale, dweight, parts, flags);                                                                    \
    if (n > kLongRun)                                                                                                          \
      hipLaunchKernelGGL(embedding_join_kernel<TYPE>, joins, dim3(kJoinWaves * 64), 0, s, keys, (int)l.chunks, l.chunk, cols,   \
                         scale, parts, flags, dweight);                                                                        \
  }
  FP8GMM_SUMS(FP8GMM_TYPE_BF16)
  FP8GMM_SUMS(FP8GMM_TYPE_FP16)
  FP8GMM_SUMS(FP8GMM_TYPE_FP32)
#undef FP8GMM_SUMS
  return hipGetLastError() == hipSuccess ? FP8GMM_OK : FP8GMM_ERR_LAUNCH;
}

}  // extern "C"
