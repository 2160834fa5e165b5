// The choice of a token's experts from its scores, and the chain from their weights back to the scores, for gfx950
// (moe_ops.select_experts).
//
//   p = softmax(s) or sigmoid(s), c = p + bias
//   the experts lie in `groups` groups of neighbours; a group counts the sum of its `group_best` (1 or 2) largest c, and the
//   `top_groups` largest groups stay; of their experts the `top_k` largest c are chosen, the lower number first where two are equal
//   w = scale p[chosen], with `renormalize` scale p[chosen] / sum of p[chosen]
//
// What is compared decides where a token goes, so it is compared exactly: the scores themselves where p alone would decide (it grows
// with them), else c and the groups' sums in 64 bits.  A key is such a number with the last 12 bits of its fraction replaced by the
// expert's number, so no two keys are equal, the largest key names its expert, and numbers that agree in their first 40 bits count as
// equal.  The weights are fp32.
//
// LANES lanes have a token, 16 (a row of the data-parallel primitives) or 64, with PER neighbouring experts in the registers of each:
// a round takes the largest key of every lane's own, exchanges them in log2(LANES) steps, and strikes it out.
#include <algorithm>
#include <type_traits>

#include "elements.h"

namespace fp8gmm {
namespace {

constexpr int kMaxChoices = FP8GMM_MAX_CHOICES;
constexpr int kThreads = 256;
constexpr double kFar = 1e300;          // nearer to zero than what is struck out; scores and sums are cut to it
constexpr double kStruck = -1.7e308;

// exp(x) for x <= 0 or moderate x, 2^-46 relative: 2^n times the series of exp to its eleventh power, on a remainder of at most
// ln(2) / 2, whose next term is below 2^-47.
__device__ __forceinline__ double exp64(double x) {
  const double cut = fmin(fmax(x, -700.), 700.), n = rint(cut * 1.4426950408889634);
  double f = __builtin_fma(n, -0.6931471805599453, cut);
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
  return x == x ? __builtin_ldexp(p, (int)n) : x;
}
__device__ __forceinline__ float sigmoid(float s) { return 1.f / (1.f + expf(-s)); }

// The key of a number: what is no number goes last.  `number` < 4096.
__device__ __forceinline__ double key_of(double v, int number) {
  v = fmin(fmax(v, -kFar), kFar) + 0.;   // (one zero, not two)
  const uint64_t bits = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (bits & ~0xfffull) | (uint64_t)(v < 0. ? number : 4095 - number));
}
__device__ __forceinline__ int number_of(double key) {
  const int low = (int)(__builtin_bit_cast(uint64_t, key) & 0xfff);
  return key < 0. ? low : 4095 - low;
}

// v of another lane of the row of 16
template <int CONTROL>
__device__ __forceinline__ double lane64(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CONTROL, 0xf, 0xf, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CONTROL, 0xf, 0xf, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int CONTROL>
__device__ __forceinline__ float lane32(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CONTROL, 0xf, 0xf, true));
}
// f joined over the lanes of a token, the same in all of them
template <int LANES, class F>
__device__ __forceinline__ double over64(double v, F&& f) {
  v = f(v, lane64<0xb1>(v));
  v = f(v, lane64<0x4e>(v));
  v = f(v, lane64<0x141>(v));
  v = f(v, lane64<0x140>(v));
  if constexpr (LANES == 64) {
    v = f(v, __shfl_xor(v, 16, 64));
    v = f(v, __shfl_xor(v, 32, 64));
  }
  return v;
}
template <int LANES, class F>
__device__ __forceinline__ float over32(float v, F&& f) {
  v = f(v, lane32<0xb1>(v));
  v = f(v, lane32<0x4e>(v));
  v = f(v, lane32<0x141>(v));
  v = f(v, lane32<0x140>(v));
  if constexpr (LANES == 64) {
    v = f(v, __shfl_xor(v, 16, 64));
    v = f(v, __shfl_xor(v, 32, 64));
  }
  return v;
}
struct Largest {
  __device__ double operator()(double a, double b) const { return fmax(a, b); }
  __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Sum {
  __device__ double operator()(double a, double b) const { return a + b; }
  __device__ float operator()(float a, float b) const { return a + b; }
};

// A lane's experts: e0 .. e0 + PER - 1 of the row, minus infinity behind its end
template <int TYPE, int PER>
__device__ __forceinline__ void load_scores(const void* scores, int64_t token, int experts, int e0, float (&s)[PER]) {
  typedef Elements<TYPE> E;
  const typename E::bits* const row = static_cast<const typename E::bits*>(scores) + token * experts;
  constexpr int V = E::kVec < PER ? E::kVec : PER;
#pragma unroll
  for (int j = 0; j < PER; j += V) {
    float f[E::kVec];
    E::unpack(E::load(row + e0 + j, V < E::kVec ? min(V, experts - e0 - j) : experts - e0 - j), f);
#pragma unroll
    for (int i = 0; i < V; ++i) s[j + i] = e0 + j + i < experts ? f[i] : -INFINITY;
  }
}
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

// The two largest of what two lanes or experts have
__device__ __forceinline__ void take_two(double& first, double& second, double v) {
  second = fmax(second, fmin(first, v));
  first = fmax(first, v);
}

template <int TYPE, int LANES, int PER>
__global__ __launch_bounds__(kThreads) void select_experts_kernel(const void* __restrict__ scores, int tokens, const Choice c,
                                                                  float* __restrict__ weights, int64_t* __restrict__ selected) {
  const int lane = threadIdx.x % LANES;
  const int64_t token = (int64_t)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const bool live = token < tokens;   // the others' lanes are read by nobody, but go along
  const int64_t from = live ? token : tokens - 1;
  const int e0 = lane * PER;
  float s[PER];
  load_scores<TYPE, PER>(scores, from, c.experts, e0, s);
  float most = 0.f, total = 1.f;   // of the softmax
  if (!c.sigmoid) {
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < PER; ++j) m = fmaxf(m, s[j]);
    most = over32<LANES>(m, Largest{});
  }
  const bool by_scores = c.bias == nullptr && (c.groups == 1 || c.group_best == 1);
  double key[PER];
  if (by_scores) {
#pragma unroll
    for (int j = 0; j < PER; ++j) key[j] = e0 + j < c.experts ? key_of((double)s[j], e0 + j) : kStruck;
    if (!c.sigmoid) {
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < PER; ++j) sum += e0 + j < c.experts ? expf(s[j] - most) : 0.f;
      total = over32<LANES>(sum, Sum{});
    }
  } else {
    double p[PER], sum = 0.;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      p[j] = c.sigmoid ? 1. / (1. + exp64(-(double)s[j])) : exp64((double)s[j] - (double)most);
      sum += e0 + j < c.experts ? p[j] : 0.;
    }
    if (!c.sigmoid) {
      sum = over64<LANES>(sum, Sum{});
      total = (float)sum;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (!c.sigmoid) p[j] /= sum;
      if (c.bias != nullptr && e0 + j < c.experts) p[j] += (double)c.bias[e0 + j];
      key[j] = e0 + j < c.experts ? key_of(p[j], e0 + j) : kStruck;
    }
  }
  if (c.groups > 1 && c.top_groups < c.groups) {
    const int size = c.experts / c.groups;
    double mine = kStruck;   // the key of the group that a lane stands for
    uint32_t kept = 0;
    for (int g = 0; g < c.groups; ++g) {
      double first = -kFar, second = -kFar;
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if ((uint32_t)(e0 + j - g * size) < (uint32_t)size) take_two(first, second, key[j]);
      const auto join = [&](double a, double b) {
        take_two(first, second, a);
        second = fmax(second, b);
      };
      join(lane64<0xb1>(first), lane64<0xb1>(second));
      join(lane64<0x4e>(first), lane64<0x4e>(second));
      join(lane64<0x141>(first), lane64<0x141>(second));
      join(lane64<0x140>(first), lane64<0x140>(second));
      if constexpr (LANES == 64) {
        join(__shfl_xor(first, 16, 64), __shfl_xor(second, 16, 64));
        join(__shfl_xor(first, 32, 64), __shfl_xor(second, 32, 64));
      }
      const double value = c.group_best == 2 && size > 1 ? first + second : first;
      if (g == lane) mine = key_of(value, g);
    }
    for (int i = 0; i < c.top_groups; ++i) {
      const double best = over64<LANES>(mine, Largest{});
      kept |= 1u << (number_of(best) & 31);
      if (mine == best) mine = kStruck;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (e0 + j < c.experts && !(kept >> ((e0 + j) / size) & 1)) key[j] = kStruck;
  }
  int chosen = 0;
  for (int k = 0; k < c.top_k; ++k) {
    double best = key[0];
#pragma unroll
    for (int j = 1; j < PER; ++j) best = fmax(best, key[j]);
    best = over64<LANES>(best, Largest{});
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (key[j] == best) key[j] = kStruck;
    if (k == lane) chosen = number_of(best);
  }
  const bool has = lane < c.top_k;
  float w = 0.f;
  if (has) {
    const float v = score_of<TYPE>(scores, from, c.experts, chosen);
    w = c.sigmoid ? sigmoid(v) : expf(v - most) / total;
  }
  if (c.renormalize) w /= over32<LANES>(w, Sum{});
  if (has && live) {
    weights[token * c.top_k + lane] = w * c.scale;
    selected[token * c.top_k + lane] = chosen;
  }
}

// Of the weights' gradients: with v = p[chosen] and renormalized weights dv = (dw - (sum of dw v) / (sum of v)) scale / (sum of v),
// otherwise dv = scale dw; through the sigmoid ds = dv p (1 - p), through the softmax ds = p (dv - sum of dv v).
template <int TYPE, int LANES, int PER>
__global__ __launch_bounds__(kThreads) void select_experts_backward_kernel(const void* __restrict__ scores, int tokens, const Choice c,
                                                                           const int64_t* __restrict__ selected,
                                                                           const float* __restrict__ grad_weights,
                                                                           void* __restrict__ grad_scores) {
  typedef Elements<TYPE> E;
  const int lane = threadIdx.x % LANES;
  const int64_t token = (int64_t)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const bool live = token < tokens;
  const int64_t from = live ? token : tokens - 1;
  const int e0 = lane * PER;
  float s[PER], most = 0.f, total = 1.f;
  if (!c.sigmoid) {
    load_scores<TYPE, PER>(scores, from, c.experts, e0, s);
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < PER; ++j) m = fmaxf(m, s[j]);
    most = over32<LANES>(m, Largest{});
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      s[j] = e0 + j < c.experts ? expf(s[j] - most) : 0.f;
      sum += s[j];
    }
    total = over32<LANES>(sum, Sum{});
  }
  const bool has = lane < c.top_k;
  int chosen = -1;
  float g = 0.f, p = 0.f, rest = 0.f;
  if (has) {
    const int64_t e = selected[from * c.top_k + lane];
    g = grad_weights[from * c.top_k + lane] * c.scale;
    if ((uint64_t)e < (uint64_t)c.experts) {   // not an expert: no gradient
      chosen = (int)e;
      const float v = score_of<TYPE>(scores, from, c.experts, chosen);
      p = c.sigmoid ? sigmoid(v) : expf(v - most) / total;
      rest = c.sigmoid ? 1.f / (1.f + expf(v)) : 0.f;
    } else {
      g = 0.f;
    }
  }
  if (c.renormalize) {
    const float sum = over32<LANES>(p, Sum{}), dot = over32<LANES>(g * p, Sum{});
    g = has ? (g - dot / sum) / sum : 0.f;
  }
  const float back = c.sigmoid ? 0.f : over32<LANES>(g * p, Sum{});
  if (c.sigmoid) g *= p * rest;
  float out[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) out[j] = 0.f;
  for (int k = 0; k < c.top_k; ++k) {
    const int at = __shfl(chosen, k, LANES) - e0;
    const float v = __shfl(g, k, LANES);
#pragma unroll
    for (int j = 0; j < PER; ++j) out[j] = at == j ? v : out[j];
  }
  if (!c.sigmoid)
#pragma unroll
    for (int j = 0; j < PER; ++j) out[j] = s[j] / total * (out[j] - back);
  if (!live) return;
  typename E::bits* const row = static_cast<typename E::bits*>(grad_scores) + token * c.experts;
  constexpr int V = E::kVec < PER ? E::kVec : PER;
#pragma unroll
  for (int j = 0; j < PER; j += V) {
    float f[E::kVec] = {};
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = out[j + i];
    E::store(row + e0 + j, V < E::kVec ? min(V, c.experts - e0 - j) : c.experts - e0 - j, E::pack(f));
  }
}

// calls f(TYPE, LANES, PER): 16 lanes up to 512 experts, as few of them to each as there are sizes for
template <class F>
void with_shape(int type, int experts, F&& f) {
  const auto shape = [&](auto t) {
    const auto as = [&](auto lanes, auto per) { f(t, lanes, per); };
    constexpr std::integral_constant<int, 16> row{};
    constexpr std::integral_constant<int, 64> wave{};
    if (experts <= 16) as(row, std::integral_constant<int, 1>{});
    else if (experts <= 32) as(row, std::integral_constant<int, 2>{});
    else if (experts <= 64) as(row, std::integral_constant<int, 4>{});
    else if (experts <= 128) as(row, std::integral_constant<int, 8>{});
    else if (experts <= 256) as(row, std::integral_constant<int, 16>{});
    else if (experts <= 512) as(row, std::integral_constant<int, 32>{});
    else if (experts <= 1024) as(wave, std::integral_constant<int, 16>{});
    else as(wave, std::integral_constant<int, 64>{});
  };
  if (type == FP8GMM_TYPE_BF16) shape(std::integral_constant<int, FP8GMM_TYPE_BF16>{});
  else if (type == FP8GMM_TYPE_FP16) shape(std::integral_constant<int, FP8GMM_TYPE_FP16>{});
  else shape(std::integral_constant<int, FP8GMM_TYPE_FP32>{});
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
  with_shape(type, c.experts, [&](auto t, auto lanes, auto per) {
    constexpr int TOKENS = kThreads / decltype(lanes)::value;
    hipLaunchKernelGGL((select_experts_kernel<decltype(t)::value, decltype(lanes)::value, decltype(per)::value>),
                       dim3((unsigned)((tokens + TOKENS - 1) / TOKENS)), dim3(kThreads), 0, static_cast<hipStream_t>(stream), scores,
                       (int)tokens, c, weights, selected);
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
  with_shape(type, c.experts, [&](auto t, auto lanes, auto per) {
    constexpr int TOKENS = kThreads / decltype(lanes)::value;
    hipLaunchKernelGGL((select_experts_backward_kernel<decltype(t)::value, decltype(lanes)::value, decltype(per)::value>),
                       dim3((unsigned)((tokens + TOKENS - 1) / TOKENS)), dim3(kThreads), 0, static_cast<hipStream_t>(stream), scores,
                       (int)tokens, c, selected, grad_weights, grad_scores);
  });
  return hipGetLastError() == hipSuccess ? FP8GMM_OK : FP8GMM_ERR_LAUNCH;
}

}  // extern "C"
