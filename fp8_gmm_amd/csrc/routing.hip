// The choice of a token's experts from its scores, and the chain from their weights back to the scores, for gfx950
// (moe_ops.select_experts).
//
//   p = softmax(s) or sigmoid(s), c = p + bias
//   the experts lie in `groups` groups of neighbours; a group counts the sum of its `group_best` (1 or 2) largest c, and the
//   `top_groups` largest groups stay; of their experts the `top_k` largest c are chosen, the lower number first where two are equal
//   w = scale p[chosen], with `renormalize` scale p[chosen] / sum of p[chosen]
//
// What is compared decides where a token goes: the scores themselves where p alone would decide (it grows with them), else c and the groups'
// sums in 64 bits, p to 2^-46.  A key is such a number that holds the expert's number in its last bits, so no two keys are equal and the
// largest names its expert: 16 bits of a score and 15 of the number, or a number in 64 bits whose last 12 bits of the fraction are replaced
// (what agrees in its first 40 bits counts as equal, of groups' sums in 36).  An expert whose score or bias is minus infinity is switched
// off: it goes last, whatever the other one is.  The weights are fp32.
//
// LANES lanes have a token, 8 or 16 (of a row of the data-parallel primitives) or 64, with PER neighbouring experts in the registers of
// each: a round takes the largest key of every lane's own, exchanges them in log2(LANES) steps, and leaves it out of the next.  Bound by these
// instructions, not by the scores' bytes: 16384 tokens of 256 experts, sigmoid, bias and groups, 13.4 us, of which a unit issues vector
// instructions for 8.3 at 2.4 GHz; 131072 of 64 by softmax 12.0 and 9.0, backward 12.6 and 10.7 (the former's 6.6 and 3.0: half of it waits for memory).
#include <algorithm>
#include <type_traits>

#include "elements.h"

namespace fp8gmm {
namespace {

constexpr int kMaxChoices = FP8GMM_MAX_CHOICES;
constexpr int kThreads = 256;
constexpr int64_t kSlab = 1 << 23;   // workgroups of a launch: a grid has fewer than 2^32 threads

// exp(x) of -700 <= x <= 700, 2^-46 relative: 2^n times the series of exp to its eleventh power, on a remainder of at most ln(2) / 2, whose
// next term is below 2^-47.  n is what a large number's last bits hold, and goes into the exponent as it is.
__device__ __forceinline__ double exp64(double x) {
  constexpr double kWhole = 0x1.8p52;
  const double large = __builtin_fma(x, 1.4426950408889634, kWhole), n = large - kWhole;
  double f = __builtin_fma(n, -0.6931471805599453, x);
  f = __builtin_fma(n, -2.3190468138462996e-17, f);
  double p = 1. / 39916800.;
  p = __builtin_fma(p, f, 1. / 3628800.);
  p = __builtin_fma(p, f, 1. / 362880.);
  p = __builtin_fma(p, f, 1. / 40320.);
  p = __builtin_fma(p, f, 1. / 5040.);
  p = __builtin_fma(p, f, 1. / 720.);
  p = __builtin_fma(p, f, 1. / 120.);
  p = __builtin_fma(p, f, 1. / 24.);
  p = __builtin_fma(p, f, 1. / 6.);
  p = __builtin_fma(p, f, .5);
  p = __builtin_fma(p, f, 1.);
  p = __builtin_fma(p, f, 1.);
  return __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, p) + (__builtin_bit_cast(uint64_t, large) << 52));
}
// 1 / d for 1 <= d <= e^701: the hardware's first guess, 2^-23, and two of Newton's steps (with one, 2^-46 more on p, 131072 tokens of 64 experts
// by sigmoid and bias 18.0 us, with two 18.5)
__device__ __forceinline__ double rcp64(double d) {
  double r = __builtin_amdgcn_rcp(d);
  r = __builtin_fma(__builtin_fma(-d, r, 1.), r, r);
  return __builtin_fma(__builtin_fma(-d, r, 1.), r, r);
}
// exp(x) of x <= 0, for sums whose largest part is 1 and gradients: the hardware's power of 2 of the rounded product, and what the rounding
// left of it to the first order, 2 units in the last place.  A NaN stays one, a result below 2^-126 is zero.  (131072 tokens of 64 experts,
// softmax, us forward and backward: 10.8 and 11.9, with expf, one unit and subnormal numbers, 11.8 and 12.8.  The weights are expf's.)
__device__ __forceinline__ float exp_of(float x) {
  x = __builtin_elementwise_maximum(x, -200.f);
  const float t = x * 0x1.715476p+0f;
  const float rest = __builtin_fmaf(x, 0x1.4ae0bep-26f, __builtin_fmaf(x, 0x1.715476p+0f, -t));
  const float e = __builtin_amdgcn_exp2f(t);
  return __builtin_fmaf(e, rest * 0x1.62e43p-1f, e);
}
__device__ __forceinline__ float sigmoid(float s) { return 1.f / (1.f + expf(-s)); }

// Keys of 64 bits.  What is no number goes last, with minus infinity.
typedef double key64;
constexpr double kStruck64 = -1.7e308, kFar = 0x1p996;   // what is struck out, and what numbers and sums are cut to
constexpr double kOff = -0x1p995;   // below it, experts that are switched off and groups of none but such
// (an instruction: fmax would look for NaN in both, which keys are not)
__device__ __forceinline__ key64 larger(key64 a, key64 b) {
  key64 r;
  asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ key64 smaller(key64 a, key64 b) {
  key64 r;
  asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
// `number` < 4096; of a number between -kFar and kFar, not the zero below zero
__device__ __forceinline__ key64 key_of_plain(double v, int number) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, v);
  int32_t below = (int32_t)(bits >> 32) >> 31;
  asm("" : "+v"(below));   // (a comparison in 64 bits and a selection otherwise)
  return __builtin_bit_cast(double, (bits & ~0xfffull) | (((uint32_t)below & 0xfffu) ^ (uint32_t)(4095 - number)));
}
__device__ __forceinline__ double within(double v) { return fmin(fmax(v, -kFar), kFar) + 0.; }   // (one zero, not two)
__device__ __forceinline__ key64 key_of(double v, int number) { return key_of_plain(within(v), number); }
__device__ __forceinline__ int number_of(key64 key) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, key);
  const int low = (int)(bits & 0xfff);
  return (int64_t)bits < 0 ? low : 4095 - low;
}
// The sum of two keys' numbers, rounded to its first 36 bits: sums that are equal, as that of the sigmoids of x and -x is for every x, come
// out equal, where the keys are cut off 2^-40 below their numbers.
__device__ __forceinline__ double sum_of(key64 a, key64 b) {
  const auto plain = [](key64 k) { return __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, k) & ~0xfffull); };
  const double sum = smaller(plain(a) + plain(b), kFar);
  return __builtin_bit_cast(double, (__builtin_bit_cast(uint64_t, sum) + 0x8000) & ~0xffffull);
}
__device__ __forceinline__ void strike(key64& key, bool gone) {   // the upper half does
  const uint64_t bits = __builtin_bit_cast(uint64_t, key);
  const uint32_t hi = gone ? (uint32_t)(__builtin_bit_cast(uint64_t, kStruck64) >> 32) : (uint32_t)(bits >> 32);
  key = __builtin_bit_cast(double, (uint64_t)hi << 32 | (uint32_t)bits);
}

// Keys of 31 bits, of 16-bit scores
typedef uint32_t key32;
// Two scores as numbers without a sign in their order: 2^15 and their magnitude more or less (so there is one zero), and so much on top
// that NaN above infinity pass 2^16, to where those below minus infinity are; all of these become minus infinity.
template <int TYPE>
__device__ __forceinline__ uint32_t order_of(uint32_t two) {
  typedef uint16_t pair __attribute__((ext_vector_type(2)));
  typedef int16_t signed_pair __attribute__((ext_vector_type(2)));
  constexpr int kInf = TYPE == FP8GMM_TYPE_BF16 ? 0x7f80 : 0x7c00, kTop = 0x7fff - kInf, kLast = 0x8000 - kInf + kTop;
  const signed_pair sign = __builtin_bit_cast(signed_pair, two) >> (int16_t)15;
  const signed_pair v = (__builtin_bit_cast(signed_pair, two & 0x7fff7fffu) ^ sign) - sign;
  const pair order = __builtin_bit_cast(pair, v) + (uint16_t)(0x8000 + kTop);
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(order, pair{kLast, kLast}));
}
// of the pair's first or second
__device__ __forceinline__ key32 key_of_order(uint32_t two, bool second, int number) {
  return ((second ? two >> 1 : two << 15) & 0x7fff8000u) | (uint32_t)(0x7fff - number);
}
__device__ __forceinline__ key32 larger(key32 a, key32 b) { return max(a, b); }
__device__ __forceinline__ int number_of(key32 key) { return 0x7fff - (int)(key & 0x7fffu); }
__device__ __forceinline__ void strike(key32& key, bool gone) { key = gone ? 0u : key; }

// v of another lane of the row of 16
template <int CONTROL>
__device__ __forceinline__ uint32_t other_lane(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CONTROL, 0xf, 0xf, true);
}
template <int CONTROL>
__device__ __forceinline__ float other_lane(float v) {
  return __uint_as_float(other_lane<CONTROL>(__float_as_uint(v)));
}
template <int CONTROL>
__device__ __forceinline__ double other_lane(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)other_lane<CONTROL>((uint32_t)(b >> 32)) << 32 | other_lane<CONTROL>((uint32_t)b));
}
// v of lane i of the wavefront, for all of them
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int i) { return (uint32_t)__builtin_amdgcn_readlane((int)v, i); }
__device__ __forceinline__ float lane_of(float v, int i) { return __uint_as_float(lane_of(__float_as_uint(v), i)); }
__device__ __forceinline__ double lane_of(double v, int i) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)lane_of((uint32_t)(b >> 32), i) << 32 | lane_of((uint32_t)b, i));
}
// f joined over the lanes of a token, the same in all of them
template <int LANES, class T, class F>
__device__ __forceinline__ T over(T v, F&& f) {
  v = f(v, other_lane<0xb1>(v));    // quad_perm: the neighbour
  v = f(v, other_lane<0x4e>(v));    // quad_perm: the other pair
  v = f(v, other_lane<0x141>(v));   // row_half_mirror: the other four
  if constexpr (LANES > 8) v = f(v, other_lane<0x140>(v));   // row_mirror: the other eight
  if constexpr (LANES == 64) v = f(f(lane_of(v, 0), lane_of(v, 16)), f(lane_of(v, 32), lane_of(v, 48)));
  return v;
}
// v of lane K of a token
template <int LANES, int K, class T>
__device__ __forceinline__ T from_lane(T v) {
  if constexpr (LANES == 64) {
    return lane_of(v, K);
  } else {
    const T first = other_lane<0x150 + K>(v);   // row_newbcast
    if constexpr (LANES == 16) return first;
    else return threadIdx.x & 8 ? other_lane<0x158 + K>(v) : first;
  }
}
// calls f(k) for the choices k < top_k, as integral constants
template <int LANES, int K = 0, class F>
__device__ __forceinline__ void each_choice(int top_k, F&& f) {
  if constexpr (K < kMaxChoices && K < LANES) {
    if (K >= top_k) return;
    f(std::integral_constant<int, K>{});
    each_choice<LANES, K + 1>(top_k, f);
  }
}
struct LargerKey {
  template <class K>
  __device__ __forceinline__ K operator()(K a, K b) const { return larger(a, b); }
};
struct Largest {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Sum {
  template <class T>
  __device__ __forceinline__ T operator()(T a, T b) const { return a + b; }
};

// A lane's experts, e0 .. e0 + PER - 1 of the row: pieces of V elements, one by one where the row ends
template <int TYPE, int PER>
struct Piece {
  typedef Elements<TYPE> E;
  typedef typename E::bits bits;
  static constexpr int V = E::kVec < PER ? E::kVec : PER, kCount = PER / V, kBytes = V * E::kBytes;
  typedef uint32_t half_piece __attribute__((ext_vector_type(2), aligned(2)));
  typedef uint32_t quarter_piece __attribute__((aligned(2)));
  u32x4 raw[kCount];
  __device__ __forceinline__ void load(const void* base, int64_t first, int left) {
    const bits* const p = static_cast<const bits*>(base) + first;
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      if constexpr (kBytes == 16) {
        raw[i] = E::load(p + i * V, left - i * V);
      } else {
        raw[i] = u32x4{0u, 0u, 0u, 0u};
        if (left >= V) {
          if constexpr (kBytes == 8) {
            const u32x2 v = *reinterpret_cast<const half_piece*>(p);
            raw[i].x = v.x;
            raw[i].y = v.y;
          } else if constexpr (kBytes == 4) {
            raw[i].x = *reinterpret_cast<const quarter_piece*>(p);
          } else {
            raw[i].x = *p;
          }
        } else {
          raw[i] = E::load(p, left);
        }
      }
    }
  }
  __device__ __forceinline__ void get(float (&s)[PER], int left) const {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      float f[E::kVec];
      E::unpack(raw[i], f);
#pragma unroll
      for (int j = 0; j < V; ++j) s[i * V + j] = i * V + j < left ? f[j] : -INFINITY;
    }
  }
  __device__ __forceinline__ uint32_t two(int j) const { return raw[j / V][j % V / 2]; }   // elements j and j + 1, of 16 bits
  static __device__ __forceinline__ void store(void* base, int64_t first, int left, const float (&s)[PER]) {
    bits* const p = static_cast<bits*>(base) + first;
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      float f[E::kVec] = {};
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = s[i * V + j];
      const u32x4 v = E::pack(f);
      if constexpr (kBytes == 16) {
        E::store(p + i * V, left - i * V, v);
      } else if (left >= V) {
        if constexpr (kBytes == 8) *reinterpret_cast<half_piece*>(p) = u32x2{v.x, v.y};
        else if constexpr (kBytes == 4) *reinterpret_cast<quarter_piece*>(p) = v.x;
        else *p = (bits)v.x;
      } else {
        E::store(p, left, v);
      }
    }
  }
};
template <int TYPE>
__device__ __forceinline__ float score_of(const void* scores, int64_t token, int experts, int e) {
  typedef Elements<TYPE> E;
  float f[E::kVec];
  E::unpack(E::load(static_cast<const typename E::bits*>(scores) + token * experts + e, 1), f);
  return f[0];
}

struct Choice {
  const float* bias;
  int experts, top_k, groups, top_groups, group_best;
  bool sigmoid, renormalize;
  float scale;
};

// p[chosen] / sum of p[chosen], of the chosen score v of every lane that `has` one.  p itself may be too small for a number, of all of
// them where a bias or the groups keep the largest scores out: these are shares by the largest of the chosen ones, m.  Softmax: e^(v - m).
// Sigmoid: p, where the sum is no small number; else, with e^m left out of all, e^(v - m) / (1 + e^v).
template <int LANES>
__device__ __forceinline__ float share_of(const Choice& c, bool has, float v) {
  float part = 0.f;
  if (c.sigmoid) {
    part = has ? sigmoid(v) : 0.f;
    const float sum = over<LANES>(part, Sum{});
    if (__builtin_expect(!(sum < 0.5f), 1)) return part / sum;
  }
  const float m = over<LANES>(has ? v : -INFINITY, Largest{});
  if (has) part = c.sigmoid ? expf(v - m) / (1.f + expf(v)) : expf(v - m);
  return part / over<LANES>(part, Sum{});
}

// Which experts' groups stay: strikes the others' keys out.  A group's key is its largest expert's (BEST 1), or made of the sum of its
// two largest, of which one that is switched off adds nothing, and the group's number.
template <int LANES, int PER, int BEST, class K>
__device__ __forceinline__ void keep_groups(K (&key)[PER], const Choice& c, int lane) {
  const int size = c.experts / c.groups;
  const auto take = [](K& first, K& second, K v) {
    if constexpr (BEST == 2) second = larger(second, smaller(first, v));
    first = larger(first, v);
  };
  const auto join = [&](K& first, K& second, K a, K b) {
    take(first, second, a);
    if constexpr (BEST == 2) second = larger(second, b);
  };
  const auto made = [&](K first, K second, int g) {
    if constexpr (BEST == 2) return key_of_plain(sum_of(first, second > kOff ? second : 0.), g);
    else return first;
  };
  K none = key[0];
  strike(none, true);
  // groups of whole lanes, a power of two of them in a row: every lane looks at its own group
  const int span = size / PER;
  if (c.experts == LANES * PER && size % PER == 0 && span <= (LANES > 8 ? 16 : 8) && (span & (span - 1)) == 0) {
    K first = key[0], second = none;
    if constexpr (BEST == 2) second = -kFar;
#pragma unroll
    for (int j = 1; j < PER; ++j) take(first, second, key[j]);
    if (span > 1) join(first, second, other_lane<0xb1>(first), other_lane<0xb1>(second));
    if (span > 2) join(first, second, other_lane<0x4e>(first), other_lane<0x4e>(second));
    if (span > 4) join(first, second, other_lane<0x141>(first), other_lane<0x141>(second));
    if (LANES > 8 && span > 8) join(first, second, other_lane<0x140>(first), other_lane<0x140>(second));
    K mine = made(first, second, lane / span);
    bool kept = false;
    for (int i = 0; i < c.top_groups; ++i) {
      const K best = over<LANES>(mine, LargerKey{});
      const bool it = mine == best;
      kept = kept || it;
      strike(mine, it);
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) strike(key[j], !kept);
    return;
  }
  // any others: one after the other, lane g keeps the key of group g (there are no more groups than lanes)
  K mine = none;
  for (int g = 0; g < c.groups; ++g) {
    K first = none, second = none;
    if constexpr (BEST == 2) first = second = -kFar;
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if ((uint32_t)(lane * PER + j - g * size) < (uint32_t)size) take(first, second, key[j]);
    const auto pair = [&](auto control) {
      constexpr int CONTROL = decltype(control)::value;
      const K a = other_lane<CONTROL>(first), b = other_lane<CONTROL>(second);
      join(first, second, a, b);
    };
    pair(std::integral_constant<int, 0xb1>{});
    pair(std::integral_constant<int, 0x4e>{});
    pair(std::integral_constant<int, 0x141>{});
    if constexpr (LANES > 8) pair(std::integral_constant<int, 0x140>{});
    if constexpr (LANES == 64) {
      const K a = first, b = second;
      first = lane_of(a, 0);
      second = lane_of(b, 0);
#pragma unroll
      for (int i = 16; i < 64; i += 16) join(first, second, lane_of(a, i), lane_of(b, i));
    }
    if (g == lane) mine = made(first, second, g);
  }
  uint32_t kept = 0;
  for (int i = 0; i < c.top_groups; ++i) {
    const K best = over<LANES>(mine, LargerKey{});
    kept |= 1u << (BEST == 2 ? number_of(best) : number_of(best) / size);
    strike(mine, mine == best);
  }
  int g = lane * PER / size, rest = lane * PER - g * size;   // of a lane's first expert
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    strike(key[j], !(kept >> (g & 31) & 1));
    if (++rest == size) rest = 0, ++g;
  }
}

template <int PER>
__device__ __forceinline__ void in_order(key64 (&key)[PER], int i, int j) {
  const key64 a = key[i], b = key[j];
  key[i] = larger(a, b);
  key[j] = smaller(a, b);
}
// Sorts keys at .. at + 7, the largest first, by merges of sorted pairs and fours
template <int PER>
__device__ __forceinline__ void sort8(key64 (&key)[PER], int at) {
  constexpr int kSteps[19][2] = {{0, 1}, {2, 3}, {4, 5}, {6, 7}, {0, 2}, {1, 3}, {4, 6}, {5, 7}, {1, 2}, {5, 6},
                                 {0, 4}, {1, 5}, {2, 6}, {3, 7}, {2, 4}, {3, 5}, {1, 2}, {3, 4}, {5, 6}};
#pragma unroll
  for (int i = 0; i < 19; ++i) in_order(key, at + kSteps[i][0], at + kSteps[i][1]);
}

// The top_k largest keys' numbers, number k in lane k.  Keys of 31 bits stay as they are: less the last one taken, modulo 2^32, those
// below it are the largest, in their order.
template <int LANES, int PER, class K>
__device__ __forceinline__ int take_largest(K (&key)[PER], int top_k, int lane) {
  K mine = key[0], last = K();
  if constexpr (std::is_same_v<K, key64> && PER >= 16) {
    // A lane's 8 largest in their order: a round looks at the first ones, and the lane that has the largest moves up (us of 16384 tokens of 256
    // experts, 8 choices, 10.2, by a look at all keys in every round 11.0; 4 choices 9.0 and 9.3, but 2 choices 8.3 and 8.2; 2000 tokens of 4096
    // experts 21.2 and 28.9).
    if (top_k > 2 && top_k <= 8) {
      sort8(key, 0);
#pragma unroll
      for (int at = 8; at < PER; at += 8) {   // the larger of opposite ones are the 8 largest, and fall and rise
        sort8(key, at);
#pragma unroll
        for (int i = 0; i < 8; ++i) key[i] = larger(key[i], key[at + 7 - i]);
#pragma unroll
        for (int step = 4; step > 0; step /= 2)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if ((i & step) == 0) in_order(key, i, i + step);
      }
      for (int k = 0; k < top_k; ++k) {
        const K best = over<LANES>(key[0], LargerKey{});
        const bool it = key[0] == best;
#pragma unroll
        for (int j = 0; j < 7; ++j) key[j] = it ? key[j + 1] : key[j];
        strike(key[7], it);
        if (k == lane) mine = best;
      }
      return number_of(mine);
    }
  }
  if constexpr (std::is_same_v<K, key32>) last = 1u << 31;
  for (int k = 0; k < top_k; ++k) {
    K best;
    if constexpr (std::is_same_v<K, key32>) {
      best = key[0] - last;
#pragma unroll
      for (int j = 1; j < PER; ++j) best = larger(best, key[j] - last);
      best = last = over<LANES>(best, LargerKey{}) + last;
    } else {
      best = key[0];
#pragma unroll
      for (int j = 1; j < PER; ++j) best = larger(best, key[j]);
      best = over<LANES>(best, LargerKey{});
      const int at = number_of(best) - lane * PER;
#pragma unroll
      for (int j = 0; j < PER; ++j) strike(key[j], at == j);
    }
    if (k == lane) mine = best;
  }
  return number_of(mine);
}

// SCORES: the scores decide; else p in 64 bits does, with the bias or for the groups' sums.  WHOLE: as many experts as the lanes hold.
template <int TYPE, int LANES, int PER, bool SCORES, bool WHOLE>
__global__ __launch_bounds__(kThreads) void select_experts_kernel(const void* __restrict__ scores, int tokens, const Choice c,
                                                                  float* __restrict__ weights, int64_t* __restrict__ selected) {
  const int lane = threadIdx.x % LANES;
  const int64_t token = (int64_t)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const bool live = token < tokens;   // the others' lanes are read by nobody, but go along
  const int64_t from = live ? token : tokens - 1;
  const int e0 = lane * PER, left = WHOLE ? PER : c.experts - e0;
  Piece<TYPE, PER> piece;
  piece.load(scores, from * c.experts + e0, left);
  float s[PER];
  piece.get(s, left);
  float most = 0.f, total = 1.f;   // of the softmax
  if (!c.sigmoid) {
    float m = s[0];
#pragma unroll
    for (int j = 1; j < PER; ++j) m = fmaxf(m, s[j]);
    most = over<LANES>(m, Largest{});
  }
  const bool grouped = c.top_groups < c.groups;
  int chosen;
  if constexpr (SCORES) {
    if (!c.sigmoid) {
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < PER; ++j) sum += j < left ? exp_of(s[j] - most) : 0.f;
      total = over<LANES>(sum, Sum{});
    }
    std::conditional_t<TYPE == FP8GMM_TYPE_FP32, key64, key32> key[PER];
    uint32_t two = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if constexpr (TYPE == FP8GMM_TYPE_FP32) {
        key[j] = key_of((double)s[j], e0 + j);
      } else {
        if (j % 2 == 0) two = order_of<TYPE>(piece.two(j));
        key[j] = key_of_order(two, j % 2, e0 + j);
      }
      strike(key[j], j >= left);
    }
    if (grouped) keep_groups<LANES, PER, 1>(key, c, lane);
    chosen = take_largest<LANES>(key, c.top_k, lane);
  } else {
    double p[PER];
    float odd = 0.f;   // a NaN where one of a lane's scores or biases is one or infinite
    if (c.sigmoid) {
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        p[j] = rcp64(1. + exp64((double)__builtin_amdgcn_fmed3f(-s[j], -700.f, 700.f)));
        odd = __builtin_fmaf(s[j], 0.f, odd);
      }
    } else {
      double sum = 0.;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        p[j] = exp64(fmax((double)s[j] - (double)most, -700.));   // (a NaN comes out as one of these numbers)
        sum += j < left ? p[j] : 0.;
        odd = __builtin_fmaf(j < left ? s[j] : 0.f, 0.f, odd);
      }
      const double numbers = sum;
      if (__builtin_expect(odd != odd, 0)) {
#pragma unroll
        for (int j = 0; j < PER; ++j) sum = s[j] != s[j] ? (double)s[j] : sum;
      }
      sum = over<LANES>(sum, Sum{});
      total = (float)sum + (most - most);   // (no number where the largest score is none)
      if (__builtin_expect(sum != sum, 0)) sum = over<LANES>(numbers, Sum{});   // a NaN leaves the others' order as it is
      const double inv = most < INFINITY ? 1. / sum : 0.;
#pragma unroll
      for (int j = 0; j < PER; ++j) p[j] *= inv;
    }
    if (c.bias != nullptr) {
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const float b = j < left ? c.bias[e0 + j] : 0.f;
        p[j] += (double)b;
        odd = __builtin_fmaf(b, 0.f, odd);
      }
    }
    if (__builtin_expect(odd != odd, 0)) {
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const double first = !c.sigmoid && s[j] == INFINITY && p[j] > -kFar ? kFar : p[j];
        p[j] = within(s[j] > -INFINITY ? first : -kFar);   // switched off, or no number
      }
    }
    key64 key[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      key[j] = key_of_plain(p[j], e0 + j);
      strike(key[j], j >= left);
    }
    if (grouped) c.group_best == 2 ? keep_groups<LANES, PER, 2>(key, c, lane) : keep_groups<LANES, PER, 1>(key, c, lane);
    chosen = take_largest<LANES>(key, c.top_k, lane);
  }
  const bool has = lane < c.top_k;
  float w = has ? score_of<TYPE>(scores, from, c.experts, chosen) : 0.f;
  if (c.renormalize) w = __builtin_fmaf(total, 0.f, share_of<LANES>(c, has, w));   // (a total that is no number leaves none)
  else w = c.sigmoid ? sigmoid(w) : expf(w - most) / total;
  if (has && live) {
    weights[token * c.top_k + lane] = w * c.scale;
    selected[token * c.top_k + lane] = chosen;
  }
}

// Of the weights' gradients, with v = p[chosen] and dv = scale dw: through the sigmoid ds = dv v (1 - v) of the chosen scores, through the
// softmax ds = p (dv - sum of dv v) of all.  Of renormalized weights, u = v / sum of v: ds = u (dv - sum of dv u) of the chosen scores, by the
// sigmoid times 1 - v.
template <int TYPE, int LANES, int PER, bool WHOLE>
__global__ __launch_bounds__(kThreads) void select_experts_backward_kernel(const void* __restrict__ scores, int tokens, const Choice c,
                                                                           const int64_t* __restrict__ selected,
                                                                           const float* __restrict__ grad_weights,
                                                                           void* __restrict__ grad_scores) {
  const int lane = threadIdx.x % LANES;
  const int64_t token = (int64_t)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const bool live = token < tokens;
  const int64_t from = live ? token : tokens - 1;
  const int e0 = lane * PER, left = WHOLE ? PER : c.experts - e0;
  float s[PER], most = 0.f, total = 1.f;
  if (!c.sigmoid) {
    Piece<TYPE, PER> piece;
    piece.load(scores, from * c.experts + e0, left);
    piece.get(s, left);
    float m = s[0];
#pragma unroll
    for (int j = 1; j < PER; ++j) m = fmaxf(m, s[j]);
    most = over<LANES>(m, Largest{});
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      s[j] = j < left ? exp_of(s[j] - most) : 0.f;
      sum += s[j];
    }
    total = over<LANES>(sum, Sum{});
  }
  int chosen = -1;
  float g = 0.f, v = 0.f, back = 0.f;
  if (lane < c.top_k) {
    const int64_t e = selected[from * c.top_k + lane];
    if ((uint64_t)e < (uint64_t)c.experts) {   // not an expert: no gradient
      chosen = (int)e;
      g = grad_weights[from * c.top_k + lane] * c.scale;
      v = score_of<TYPE>(scores, from, c.experts, chosen);
    }
  }
  const bool has = chosen >= 0;
  if (c.renormalize) {
    const float share = share_of<LANES>(c, has, v);
    g = share * (g - over<LANES>(g * share, Sum{}));
  } else if (c.sigmoid) {
    g *= sigmoid(v);
  } else {
    back = over<LANES>(has ? g * (expf(v - most) / total) : 0.f, Sum{});
  }
  if (c.sigmoid) g *= 1.f / (1.f + expf(v));
  float out[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) out[j] = 0.f;
  each_choice<LANES>(c.top_k, [&](auto k) {   // (by exchanges through LDS 3 % slower, single tokens 6 %)
    const int at = (int)from_lane<LANES, decltype(k)::value>((uint32_t)chosen) - e0;
    const float v = from_lane<LANES, decltype(k)::value>(g);
#pragma unroll
    for (int j = 0; j < PER; ++j) out[j] = at == j ? v : out[j];
  });
  const float inv = 1.f / total;
  if (!c.sigmoid)
#pragma unroll
    for (int j = 0; j < PER; ++j) out[j] = c.renormalize ? __builtin_fmaf(total, 0.f, out[j]) : s[j] * inv * (out[j] - back);
  if (!live) return;
  Piece<TYPE, PER>::store(grad_scores, token * c.experts + e0, left, out);
}

// calls f(TYPE, LANES, PER).  Few tokens have a wavefront each, whose lanes hold few experts (us, forward by p in 64 bits / backward:
// 1 token, 256 experts in 8 groups, 4.2 / 2.4, by 16 lanes 4.6 / 3.0; 1024 tokens 4.8 / 2.7 and 5.3 / 3.4; 2048 5.5 / 3.0 and 5.1 / 3.5; 4096
// 7.8 / 3.6 and 5.1 / 3.7; 2048 tokens of 512 experts 6.4 / 3.3 and 7.5 / 5.0).  Many tokens of few experts have 8 lanes each, as long as
// every choice and group has a lane of its own (131072 tokens, 64 experts, 6 choices by their scores, 10.8 / 11.9, by 16 lanes 13.5 / 15.0;
// 8 experts 5.3 / 6.0 and 7.9 / 8.6; 16384 tokens, 64 experts, 3.2 / 3.7 and 3.6 / 3.8, 4096 tokens 2.7 / 3.2 and 2.6 / 2.9).
constexpr int kFewTokens = 2048, kManyTokens = 8192;
template <class F>
void with_shape(int type, int64_t tokens, const Choice& c, F&& f) {
  const bool few = tokens <= kFewTokens;
  const int experts = c.experts;
  const auto shape = [&](auto t) {
    const auto as = [&](auto lanes, auto per) { f(t, lanes, per); };
    constexpr std::integral_constant<int, 8> half{};
    constexpr std::integral_constant<int, 16> row{};
    constexpr std::integral_constant<int, 64> wave{};
    if (tokens > kManyTokens && c.top_k <= 8 && c.groups <= 8 && experts <= 64) {
      if (experts <= 16) as(half, std::integral_constant<int, 2>{});
      else if (experts <= 32) as(half, std::integral_constant<int, 4>{});
      else as(half, std::integral_constant<int, 8>{});
    } else if (experts <= 64) {
      if (experts <= 16) as(row, std::integral_constant<int, 1>{});
      else if (experts <= 32) as(row, std::integral_constant<int, 2>{});
      else as(row, std::integral_constant<int, 4>{});
    }
    else if (experts <= 128) few ? as(wave, std::integral_constant<int, 2>{}) : as(row, std::integral_constant<int, 8>{});
    else if (experts <= 256) few ? as(wave, std::integral_constant<int, 4>{}) : as(row, std::integral_constant<int, 16>{});
    else if (experts <= 512) few ? as(wave, std::integral_constant<int, 8>{}) : as(row, std::integral_constant<int, 32>{});
    else if (experts <= 1024) as(wave, std::integral_constant<int, 16>{});
    else as(wave, std::integral_constant<int, 64>{});
  };
  if (type == FP8GMM_TYPE_BF16) shape(std::integral_constant<int, FP8GMM_TYPE_BF16>{});
  else if (type == FP8GMM_TYPE_FP16) shape(std::integral_constant<int, FP8GMM_TYPE_FP16>{});
  else shape(std::integral_constant<int, FP8GMM_TYPE_FP32>{});
}

// calls f(first token, tokens, workgroups) for each launch
template <class F>
void each_slab(int64_t tokens, int per_group, F&& f) {
  for (int64_t first = 0; first < tokens; first += kSlab * per_group) {
    const int64_t some = std::min(tokens - first, kSlab * per_group);
    f(first, (int)some, (int)((some + per_group - 1) / per_group));
  }
}

int check_choice(int type, int64_t tokens, const fp8gmm_choice* c) {
  if (c == nullptr) return FP8GMM_ERR_NULL_POINTER;
  if (!known_type(type)) return FP8GMM_ERR_BAD_FORMAT;
  if (tokens < 0 || tokens > INT32_MAX || c->experts < 1 || c->experts > FP8GMM_MAX_CHOICE_EXPERTS) return FP8GMM_ERR_BAD_SHAPE;
  if ((c->scoring != FP8GMM_SCORING_SOFTMAX && c->scoring != FP8GMM_SCORING_SIGMOID) || c->groups < 1 || c->groups > FP8GMM_MAX_CHOICE_GROUPS ||
      c->experts % c->groups != 0 || c->top_groups < 1 || c->top_groups > c->groups || c->group_best < 1 || c->group_best > 2 ||
      c->top_k < 1 || c->top_k > kMaxChoices || c->top_k > c->experts / c->groups * c->top_groups)
    return FP8GMM_ERR_BAD_ARGUMENT;
  return FP8GMM_OK;
}
Choice choice_of(const fp8gmm_choice& c) {
  return {c.bias, c.experts, c.top_k, c.groups, c.top_groups, c.group_best, c.scoring == FP8GMM_SCORING_SIGMOID, c.renormalize != 0, c.scale};
}

}  // namespace
}  // namespace fp8gmm

extern "C" {

int fp8gmm_select_experts(const void* scores, int type, int64_t tokens, const fp8gmm_choice* choice, float* weights, int64_t* selected,
                          void* stream) {
  using namespace fp8gmm;
  const int rc = check_choice(type, tokens, choice);
  if (rc != FP8GMM_OK) return rc;
  if (tokens == 0) return FP8GMM_OK;
  if (scores == nullptr || weights == nullptr || selected == nullptr) return FP8GMM_ERR_NULL_POINTER;
  const Choice c = choice_of(*choice);
  with_shape(type, tokens, c, [&](auto t, auto lanes, auto per) {
    constexpr int TOKENS = kThreads / decltype(lanes)::value;
    constexpr int TYPE = decltype(t)::value, LANES = decltype(lanes)::value, PER = decltype(per)::value;
    const bool by_scores = c.bias == nullptr && (c.top_groups == c.groups || c.group_best == 1), whole = c.experts == LANES * PER;
    auto* kernel = by_scores ? whole ? &select_experts_kernel<TYPE, LANES, PER, true, true> : &select_experts_kernel<TYPE, LANES, PER, true, false>
                   : whole   ? &select_experts_kernel<TYPE, LANES, PER, false, true>
                             : &select_experts_kernel<TYPE, LANES, PER, false, false>;
    each_slab(tokens, TOKENS, [&](int64_t first, int some, int groups) {
      hipLaunchKernelGGL(kernel, dim3(groups), dim3(kThreads), 0, static_cast<hipStream_t>(stream),
                         static_cast<const char*>(scores) + first * c.experts * type_bytes(type), some, c, weights + first * c.top_k,
                         selected + first * c.top_k);
    });
  });
  return hipGetLastError() == hipSuccess ? FP8GMM_OK : FP8GMM_ERR_LAUNCH;
}

int fp8gmm_select_experts_backward(const void* scores, int type, int64_t tokens, const fp8gmm_choice* choice, const int64_t* selected,
                                   const float* grad_weights, void* grad_scores, void* stream) {
  using namespace fp8gmm;
  const int rc = check_choice(type, tokens, choice);
  if (rc != FP8GMM_OK) return rc;
  if (tokens == 0) return FP8GMM_OK;
  if (scores == nullptr || selected == nullptr || grad_weights == nullptr || grad_scores == nullptr) return FP8GMM_ERR_NULL_POINTER;
  const Choice c = choice_of(*choice);
  with_shape(type, tokens, c, [&](auto t, auto lanes, auto per) {
    constexpr int TOKENS = kThreads / decltype(lanes)::value;
    constexpr int TYPE = decltype(t)::value, LANES = decltype(lanes)::value, PER = decltype(per)::value;
    auto* kernel = c.experts == LANES * PER ? &select_experts_backward_kernel<TYPE, LANES, PER, true>
                                            : &select_experts_backward_kernel<TYPE, LANES, PER, false>;
    each_slab(tokens, TOKENS, [&](int64_t first, int some, int groups) {
      const int64_t at = first * c.experts * type_bytes(type);
      hipLaunchKernelGGL(kernel, dim3(groups), dim3(kThreads), 0, static_cast<hipStream_t>(stream), static_cast<const char*>(scores) + at,
                         some, c, selected + first * c.top_k, grad_weights + first * c.top_k, static_cast<char*>(grad_scores) + at);
    });
  });
  return hipGetLastError() == hipSuccess ? FP8GMM_OK : FP8GMM_ERR_LAUNCH;
}

}  // extern "C"
