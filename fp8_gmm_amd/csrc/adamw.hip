// A step of AdamW over many tensors, for gfx950 (backend.multi_adamw, optim.AdamW).
//
//   g = grad * min(1, max_norm / (norm + 1e-6))
//   m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2
//   p = p - lr decay p - lr / (1 - beta1^t) m / (sqrt(v / (1 - beta2^t)) + eps)
//
// with p kept in fp32 (`master`) beside 16-bit weights where the caller wants that.  m and v are fp32, or in 8 bits: e4m3 codes of m
// and of sqrt(v), each 128 elements with a scale of their own in fp32, the largest magnitude over 448.  All arithmetic is fp32; what decides
// the codes is a fixed sequence of correctly rounded operations (but for the root, off in one of a million), so that who follows it gets
// the same codes.
//
// 8-bit moments are rounded by a threshold that runs evenly through [0, 1) from step to step and from element to element, the
// multiples of two irrational numbers: a moment that grows by less than half a code's distance each step would stay where it is for
// ever if it were rounded to nearest.  m is rounded so that its mean over the thresholds is m, sqrt(v) so that the mean of its square is
// v: with beta2 near 1 a bias of a thousandth of v in each step would be all there is.  A root that is not zero never becomes zero.
//
// Bound by memory: everything passes once.
#include <algorithm>
#include <cmath>
#include <vector>

#include "elements.h"

namespace fp8gmm {
namespace {

// Threads and elements of a workgroup, 4 (32 bits) or 8 to a thread at a time.  Of lists that no cache holds, us: 400 tensors of bf16 with
// fp32 moments by 512 threads and 2048 elements 596, by 256 and 1024 597, and 2048 625, and 4096 670, by 128 and 2048 669; 96 tensors of fp32
// by 512 and 2048 761, by 256 and 1024 786; 96 tensors with 8-bit moments, which take ten times the instructions, by 256 and 4096 287, and
// 6144 287, by 512 and 8192 300, by 128 and 2048 284; the same with masters 463, 478, 460 and 469, of fp32 472, 483, 475 and 482.
constexpr int threads(bool bits8) { return bits8 ? 256 : 512; }
constexpr int sweep(bool bits8) { return bits8 ? 4096 : 2048; }
// From so many bytes on everything is read and written with the streaming hint: nothing of it is found in the caches by the next step
// (470 million weights with masters 2364 us, without the hint 2470, with it on the reads or the writes alone 2454 and 2470; 16 million
// without masters 64 and 73).  Below, what the caches hold from call to call counts (8 million: 31.9 with the hint, 28.7 without).
constexpr int64_t kStreamBytes = (int64_t)256 << 20;
constexpr int kBlock = FP8GMM_ADAMW_BLOCK;
constexpr float kMost = Fp8Limits<FP8GMM_E4M3>::kMax;
constexpr float kTiny = 0x1p-100f;   // moments below it are zeros in 8 bits
// thresholds in units of 2^-32
constexpr uint32_t kStep = 0x9E3779B9u, kElement = 0x6A09E667u;   // the golden ratio and the root of 2, without their whole numbers

// LDS that nobody uses: with it two workgroups share a compute unit and not four, and the nine streams of a step with masters find their
// memory's rows open more often (470 million weights 2256 us, without it 2335; without masters it costs: 400 tensors 622 and 590).
constexpr unsigned kIdleLds = 55 * 1024;

struct Entry {
  void* param;
  const void* grad;
  void *m, *v;
  float *m_scale, *v_scale, *master;
  int64_t count;
  uint32_t begin;   // first chunk
  int type, grad_type;
};
// The tensors of a launch travel in its arguments, 48 bits of each of PTRS addresses, 40 of the count, and the types: nothing is uploaded,
// and a captured call holds its table.
template <int PTRS>
struct Part {
  static constexpr int kWords = 3 * PTRS + 3, kTensors = 3600 / (4 + 2 * kWords);
  uint32_t begin[kTensors];
  uint16_t word[kTensors][kWords];
};
constexpr int pointers(bool master, bool bits8) { return 4 + (bits8 ? 2 : 0) + (master ? 1 : 0); }
template <bool MASTER, bool BITS8>
using PartOf = Part<pointers(MASTER, BITS8)>;

template <bool MASTER, bool BITS8>
void pack(PartOf<MASTER, BITS8>& part, int at, const Entry& e) {
  part.begin[at] = e.begin;
  uint16_t* w = part.word[at];
  const auto put = [&](uint64_t v) {
    for (int k = 0; k < 3; ++k) *w++ = (uint16_t)(v >> 16 * k);
  };
  const auto address = [&](const void* p) { put(reinterpret_cast<uintptr_t>(p)); };
  address(e.param);
  address(e.grad);
  address(e.m);
  address(e.v);
  if (BITS8) {
    address(e.m_scale);
    address(e.v_scale);
  }
  if (MASTER) address(e.master);
  put((uint64_t)e.count | (uint64_t)e.type << 40 | (uint64_t)e.grad_type << 44);
}
template <bool MASTER, bool BITS8>
__device__ __forceinline__ Entry unpack(const PartOf<MASTER, BITS8>& part, int at) {
  Entry e = {};
  e.begin = part.begin[at];
  const uint16_t* w = part.word[at];
  const auto get = [&] {
    const uint64_t v = (uint64_t)w[0] | (uint64_t)w[1] << 16 | (uint64_t)w[2] << 32;
    w += 3;
    return v;
  };
  // global memory: an address without a space would be accessed as if it might be LDS
  const auto address = [&] { return (void*)reinterpret_cast<__attribute__((address_space(1))) void*>(get()); };
  e.param = address();
  e.grad = address();
  e.m = address();
  e.v = address();
  if constexpr (BITS8) {
    e.m_scale = static_cast<float*>(address());
    e.v_scale = static_cast<float*>(address());
  }
  if constexpr (MASTER) e.master = static_cast<float*>(address());
  const uint64_t last = get();
  e.count = (int64_t)(last & 0xffffffffffull);
  e.type = (int)(last >> 40 & 0xf);
  e.grad_type = (int)(last >> 44);
  return e;
}

struct Hyper {
  float b1, b2, c1, c2;   // the betas, and 1 - beta
  float eps, decay;       // decay: lr * weight_decay, or weight_decay where lr is the device's
  float rate, root;       // lr / (1 - beta1^t) and 1 / sqrt(1 - beta2^t)
  float max_norm;
  uint32_t dither;        // t * kStep
  const float* norm;
  // of a step whose number and learning rate the device has (a captured one): the logarithms of the betas, to the base 2
  const int64_t* step;
  const float* lr;
  double log1, log2, lr_host;
};

// VEC elements of a type, of which the first n are there
template <int TYPE, int VEC, bool STREAM>
struct Values {
  typedef Elements<TYPE> E;
  typedef typename E::bits bits;
  static constexpr int kBytes = VEC * E::kBytes;
  typedef uint32_t half_piece __attribute__((ext_vector_type(2), aligned(2)));
  u32x4 raw[kBytes < 16 ? 1 : kBytes / 16];
  template <bool FULL>
  __device__ __forceinline__ void load(const void* base, int64_t at, int n) {
    const bits* const p = static_cast<const bits*>(base) + at;
    if constexpr (kBytes < 16) {
      if constexpr (FULL) {
        const half_piece* const from = reinterpret_cast<const half_piece*>(p);
        const u32x2 v = STREAM ? __builtin_nontemporal_load(from) : *from;
        raw[0] = u32x4{v.x, v.y, 0u, 0u};
      } else {
        raw[0] = E::load(p, min(n, VEC));
      }
    } else {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) raw[i] = E::template load<STREAM>(p + i * E::kVec, FULL ? E::kVec : n - i * E::kVec);
    }
  }
  __device__ __forceinline__ void get(float (&f)[VEC]) const {
    constexpr int N = VEC < E::kVec ? VEC : E::kVec;
#pragma unroll
    for (int i = 0; i < VEC; i += N) {
      float part[E::kVec];
      E::unpack(raw[i / N], part);
#pragma unroll
      for (int j = 0; j < N; ++j) f[i + j] = part[j];
    }
  }
  template <bool FULL>
  static __device__ __forceinline__ void store(void* base, int64_t at, int n, const float (&f)[VEC]) {
    bits* const p = static_cast<bits*>(base) + at;
    constexpr int N = VEC < E::kVec ? VEC : E::kVec;
#pragma unroll
    for (int i = 0; i < VEC; i += N) {
      float part[E::kVec] = {};
#pragma unroll
      for (int j = 0; j < N; ++j) part[j] = f[i + j];
      const u32x4 v = E::pack(part);
      if constexpr (N < E::kVec) {
        if constexpr (FULL && STREAM) __builtin_nontemporal_store((half_piece)u32x2{v.x, v.y}, reinterpret_cast<half_piece*>(p));
        else if constexpr (FULL) *reinterpret_cast<half_piece*>(p) = u32x2{v.x, v.y};
        else E::store(p, min(n, N), v);
      } else {
        E::template store<STREAM>(p + i, FULL ? E::kVec : n - i, v);
      }
    }
  }
};

// Eight codes
template <bool STREAM>
struct Codes {
  u32x2 raw;
  template <bool FULL>
  __device__ __forceinline__ void load(const void* base, int64_t at, int n) {
    const uint8_t* const p = static_cast<const uint8_t*>(base) + at;
    if constexpr (FULL) {
      const u32x2* const from = reinterpret_cast<const u32x2*>(p);
      raw = STREAM ? __builtin_nontemporal_load(from) : *from;
    } else {
      raw = u32x2{0u, 0u};
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) raw[i / 4] |= (uint32_t)p[i] << i % 4 * 8;
    }
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)raw[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)raw[i], true);
      f[4 * i] = lo.x;
      f[4 * i + 1] = lo.y;
      f[4 * i + 2] = hi.x;
      f[4 * i + 3] = hi.y;
    }
  }
  template <bool FULL>
  static __device__ __forceinline__ void store(void* base, int64_t at, int n, u32x2 w) {
    uint8_t* const p = static_cast<uint8_t*>(base) + at;
    if constexpr (FULL && STREAM) {
      __builtin_nontemporal_store(w, reinterpret_cast<u32x2*>(p));
    } else if constexpr (FULL) {
      *reinterpret_cast<u32x2*>(p) = w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) p[i] = (uint8_t)(w[i / 4] >> i % 4 * 8);
    }
  }
};

// y to a code, up with the probability of its way to the next one: the hardware's rounding by a random number, of which it adds the upper
// 20 bits to what lies between two codes.  Byte I of `old`.  (Behind 448 there is no code: the largest's product may round to more.)
template <int I>
__device__ __forceinline__ uint32_t round_linear(float y, uint32_t h, uint32_t old) {
  return (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(__builtin_amdgcn_fmed3f(y, -kMost, kMost), (int)h, (int)old, I);
}
// 0 <= y <= 448 to a code, up with the probability of its square's way to the next one's.  The codes lie 2^(e-3) apart from 2^e on, from
// 2^-6 down 2^-9: adding 2^-6 there makes the distance that of all numbers with its exponent, and the last 20 bits of the fraction what
// lies between two codes.
__device__ __forceinline__ float threshold_of(uint32_t h) { return (float)((h ^ 0x80000000u) >> 8); }   // in units of 2^-24
__device__ __forceinline__ float round_root(float y, uint32_t h) {
  const float off = y < 0x1p-6f ? 0x1p-6f : 0.f;
  const uint32_t bits = __float_as_uint(y + off);
  const float lo = __uint_as_float(bits & 0xfff00000u) - off, eight = __uint_as_float(bits & 0x7f800000u), gap = eight * 0.125f;
  const float ways = eight * 0x1p-27f * __builtin_fmaf(2.f, lo, gap);   // the squares' distance, in units of the threshold
  const bool up = (y - lo) * (y + lo) > threshold_of(h) * ways;
  const float code = up ? lo + gap : lo;
  return y > 0.f ? fmaxf(code, 0x1p-9f) : code;
}
// The same of 2^-6 <= y, with the fraction alone, as a number between 8 and 16, where the codes lie 1 apart; the hardware's rounding by a
// random number of ones or zeros goes up (from what is no code) or down.  Byte I of `old`.
template <int I>
__device__ __forceinline__ uint32_t round_normal_root(float y, uint32_t h, uint32_t old) {
  const uint32_t bits = (__float_as_uint(y) & 0x007fffffu) | 0x41000000u;
  const float v = __uint_as_float(bits), lo = __uint_as_float(bits & 0xfff00000u);
  const bool up = (v - lo) * (v + lo) > threshold_of(h) * __builtin_fmaf(0x1p-23f, lo, 0x1p-24f);
  return (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(y, up ? -1 : 0, (int)old, I);
}

// The root of a number that is zero, normal or a NaN: the hardware's guess of its inverse and a step of Newton's, correctly rounded but in
// one of a million (8 instructions' time, sqrtf takes 17).
__device__ __forceinline__ float root_of(float v) {
  const float y = __builtin_amdgcn_rsqf(fmaxf(v, 0x1p-126f)), s = v * y;
  return __builtin_fmaf(__builtin_fmaf(-s, s, v), 0.5f * y, s);
}
// The largest magnitude of a block, 8 elements in each of 16 lanes; a NaN where one of them is
__device__ __forceinline__ float block_max(float v) {
  const auto step = [&](auto control) {
    const float other = __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), decltype(control)::value, 0xf, 0xf, true));
    v = amax_or_nan(v, other, other);
  };
  step(std::integral_constant<int, 0xb1>{});
  step(std::integral_constant<int, 0x4e>{});
  step(std::integral_constant<int, 0x141>{});
  step(std::integral_constant<int, 0x140>{});
  return v;
}

// 448 times the inverse of `most`, a guess and a step of Newton's, which is correctly rounded as the guess is off by one at most (a division
// takes three times as long); and its share of a code
__device__ __forceinline__ float codes_per(float most) {
  if (__builtin_expect(!(most >= kTiny && most < 0x1p120f), 0)) return most >= kTiny ? kMost * (1.f / most) : 0.f;
  const float r = __builtin_amdgcn_rcpf(most);
  return kMost * __builtin_fmaf(__builtin_fmaf(-most, r, 1.f), r, r);
}
__device__ __forceinline__ float per_code(float most) { return most < kTiny ? 0.f : most * (1.f / kMost); }

// What a step multiplies by, the same for all elements
struct Factors {
  float grad, rate, root, decay;
  uint32_t dither;
};
__device__ __forceinline__ Factors factors_of(const Hyper& h) {
  Factors f = {1.f, h.rate, h.root, h.decay, h.dither};
  if (h.step != nullptr || h.lr != nullptr) {
    const double lr = h.lr != nullptr ? (double)*h.lr : h.lr_host;
    f.decay = (float)(lr * (double)h.decay);
    if (h.step != nullptr) {
      const double t = (double)*h.step;
      f.rate = (float)(lr / (1. - exp2(t * h.log1)));
      f.root = (float)(1. / sqrt(1. - exp2(t * h.log2)));
      f.dither = (uint32_t)*h.step * kStep;
    } else {
      f.rate = (float)(lr * (double)h.rate);
    }
  }
  if (h.norm != nullptr) {
    const float ratio = h.max_norm / (*h.norm + 1e-6f);
    f.grad = ratio > 1.f ? 1.f : ratio;   // a NaN stays one
  }
  return f;
}

// What a thread takes of a tensor at a time
template <int TYPE, int GRAD, bool MASTER, bool BITS8, bool STREAM>
struct Share {
  static constexpr int VEC = BITS8 ? 8 : 4;
  typedef Values<FP8GMM_TYPE_FP32, VEC, STREAM> F32;
  typedef Values<TYPE, VEC, STREAM> Weights;
  std::conditional_t<MASTER, F32, Weights> param;
  Values<GRAD, VEC, STREAM> grad;
  std::conditional_t<BITS8, Codes<STREAM>, F32> m, v;
  float m_scale, v_scale;
  template <bool FULL>
  __device__ __forceinline__ void load(const Entry& e, int64_t at, int n) {
    grad.template load<FULL>(e.grad, at, n);
    param.template load<FULL>(MASTER ? static_cast<const void*>(e.master) : e.param, at, n);
    m.template load<FULL>(e.m, at, n);
    v.template load<FULL>(e.v, at, n);
    if constexpr (BITS8) {
      m_scale = FULL || n > 0 ? e.m_scale[at / kBlock] : 0.f;
      v_scale = FULL || n > 0 ? e.v_scale[at / kBlock] : 0.f;
    }
  }
};

template <bool FULL, int TYPE, int GRAD, bool MASTER, bool BITS8, bool STREAM>
__device__ __forceinline__ void step_values(const Share<TYPE, GRAD, MASTER, BITS8, STREAM>& from, const Entry& e, int64_t at, int n,
                                            const Hyper& h, const Factors& by) {
  typedef Share<TYPE, GRAD, MASTER, BITS8, STREAM> S;
  constexpr int VEC = S::VEC;
  float p[VEC], g[VEC], m[VEC], v[VEC];
  from.param.get(p);
  from.grad.get(g);
  from.m.get(m);
  from.v.get(v);
  float root[VEC], ratio[VEC], v_most = 0.f;
  bool rare = !(h.eps >= (BITS8 ? 0x1p-30f : 0x1p-120f) && h.eps < 0x1p120f);
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    g[i] *= by.grad;
    if constexpr (BITS8) {
      m[i] *= from.m_scale;
      v[i] *= from.v_scale;
      v[i] *= v[i];
    }
    m[i] = h.b1 * m[i] + h.c1 * g[i];
    v[i] = h.b2 * v[i] + h.c2 * g[i] * g[i];
    root[i] = root_of(v[i]);
    if constexpr (!BITS8) rare = rare || __builtin_isfpclass(v[i], 0x290);   // subnormal, or infinite
    const float d = __builtin_fmaf(root[i], by.root, h.eps);
    const float r = __builtin_amdgcn_rcpf(d);   // and a step of Newton's: 4 instructions for a division's 10
    ratio[i] = m[i] * __builtin_fmaf(__builtin_fmaf(-d, r, 1.f), r, r);
  }
  const auto most_of = [](const float (&f)[VEC]) {
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < VEC; i += 2) most = amax_or_nan(most, f[i], f[i + 1]);
    return block_max(most);
  };
  if constexpr (BITS8) {
    // A block at a time: an infinite v leaves a NaN in its root.  A subnormal one's root is wrong, but not zero and so far below the others'
    // that its code is the smallest one, and 2^-33 of eps in the quotient (below an eps of 2^-30 all take the longer way, 356 us and not 287).
    v_most = most_of(root);
    rare = rare || !(v_most < 0x1p62f) || (v_most < 0x1p-40f && v_most != 0.f);
  }
  if (__builtin_expect(rare, 0)) {   // what the guesses do not reach
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      root[i] = sqrtf(v[i]);
      ratio[i] = m[i] / __builtin_fmaf(root[i], by.root, h.eps);
    }
    if constexpr (BITS8) v_most = most_of(root);
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    p[i] = __builtin_fmaf(-by.rate, ratio[i], __builtin_fmaf(-by.decay, p[i], p[i]));
    if constexpr (MASTER) asm("" : "+v"(p[i]));   // fp32 first, then 16 bits: the weight is the master's rounded copy
  }
  if constexpr (MASTER) S::F32::template store<FULL>(e.master, at, n, p);
  S::Weights::template store<FULL>(e.param, at, n, p);
  if constexpr (BITS8) {
    const float m_most = most_of(m);
    // The square of a finite gradient may be infinite: its root is the largest that fp32 has, since an infinite scale would take the block along.
    constexpr float kRoot = 0x1.fffffep63f;
    if (__builtin_expect(v_most > kRoot, 0) && m_most < INFINITY) v_most = kRoot;
    const float m_inv = codes_per(m_most), v_inv = codes_per(v_most);
    const uint32_t first = (uint32_t)at * kElement + by.dither;
    u32x2 mw = {0u, 0u}, vw = {0u, 0u};
    float least = kMost;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      root[i] = fminf(root[i] * v_inv, kMost);   // (the largest's product may round to more)
      least = fminf(least, root[i]);
    }
    if (__any(least < 0x1p-6f)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float c[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) c[k] = round_root(root[4 * i + k], first + (4 * i + k) * kElement);
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
        vw[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], lo, true);
      }
    } else {   // a fifth fewer instructions (96 tensors of bf16 287 us, by the longer form alone 298)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int j = 4 * i;
        vw[i] = round_normal_root<0>(root[j], first + j * kElement, vw[i]);
        vw[i] = round_normal_root<1>(root[j + 1], first + (j + 1) * kElement, vw[i]);
        vw[i] = round_normal_root<2>(root[j + 2], first + (j + 2) * kElement, vw[i]);
        vw[i] = round_normal_root<3>(root[j + 3], first + (j + 3) * kElement, vw[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int j = 4 * i;
      mw[i] = round_linear<0>(m[j] * m_inv, first + j * kElement, mw[i]);
      mw[i] = round_linear<1>(m[j + 1] * m_inv, first + (j + 1) * kElement, mw[i]);
      mw[i] = round_linear<2>(m[j + 2] * m_inv, first + (j + 2) * kElement, mw[i]);
      mw[i] = round_linear<3>(m[j + 3] * m_inv, first + (j + 3) * kElement, mw[i]);
    }
    if (threadIdx.x % 16 == 0 && (FULL || n > 0)) {
      e.m_scale[at / kBlock] = per_code(m_most);
      e.v_scale[at / kBlock] = per_code(v_most);
    }
    Codes<STREAM>::template store<FULL>(e.m, at, n, mw);
    Codes<STREAM>::template store<FULL>(e.v, at, n, vw);
  } else {
    S::F32::template store<FULL>(e.m, at, n, m);
    S::F32::template store<FULL>(e.v, at, n, v);
  }
}

template <bool MASTER, bool BITS8, bool STREAM>
__global__ __launch_bounds__(threads(BITS8)) void adamw_kernel(const PartOf<MASTER, BITS8> part, int n, const Hyper h) {
  constexpr int VEC = BITS8 ? 8 : 4, THREADS = threads(BITS8), STEP = THREADS * VEC, SWEEP = sweep(BITS8);
  __shared__ int found;
  for (int i = threadIdx.x; i < n; i += THREADS)
    if (part.begin[i] <= blockIdx.x && (i + 1 == n || blockIdx.x < part.begin[i + 1])) found = i;
  __syncthreads();
  Entry e = unpack<MASTER, BITS8>(part, __builtin_amdgcn_readfirstlane(found));
  Factors by = factors_of(h);
  const int64_t first = (int64_t)(blockIdx.x - e.begin) * SWEEP, end = first + SWEEP < e.count ? first + SWEEP : e.count;
  const auto as = [&](auto type, auto grad) {
    constexpr int TYPE = decltype(type)::value, GRAD = decltype(grad)::value;
    Share<TYPE, GRAD, MASTER, BITS8, STREAM> share;
    int left = (int)(end - first);
    int64_t at = threadIdx.x * VEC;
    if constexpr (SWEEP == STEP) {
      at += first;
      if (left >= STEP) {
        share.template load<true>(e, at, VEC);
        step_values<true>(share, e, at, VEC, h, by);
        return;
      }
    } else {
      // Where the workgroup is stays in scalar registers: without the threads' places there is room for 6 wavefronts where there are no masters
      // (96 tensors 287 us, with 5 of them 302; with masters 83 registers leave 5, 463 and 468).
      const auto go_on = [&](int64_t elements) {
        const auto go = [&](auto*& p, int64_t bytes) {
          typedef std::remove_pointer_t<std::remove_reference_t<decltype(p)>> T;
          p = reinterpret_cast<T*>(reinterpret_cast<std::conditional_t<std::is_const_v<T>, const char*, char*>>(p) + bytes);
        };
        go(e.param, elements * Elements<TYPE>::kBytes);
        go(e.grad, elements * Elements<GRAD>::kBytes);
        go(e.m, elements);
        go(e.v, elements);
        go(e.m_scale, elements / kBlock * 4);
        go(e.v_scale, elements / kBlock * 4);
        if constexpr (MASTER) go(e.master, elements * 4);
        by.dither += (uint32_t)elements * kElement;
      };
      go_on(first);
#pragma unroll 1
      for (; left >= STEP; left -= STEP) {
        share.template load<true>(e, at, VEC);
        step_values<true>(share, e, at, VEC, h, by);
        go_on(STEP);
      }
      if (left == 0) return;
    }
    const int mine = min(left - (int)threadIdx.x * VEC, VEC);
    share.template load<false>(e, at, mine);
    step_values<false>(share, e, at, mine, h, by);
  };
  constexpr std::integral_constant<int, FP8GMM_TYPE_BF16> bf16{};
  constexpr std::integral_constant<int, FP8GMM_TYPE_FP16> fp16{};
  constexpr std::integral_constant<int, FP8GMM_TYPE_FP32> fp32{};
  if (e.type == FP8GMM_TYPE_BF16) {
    e.grad_type == FP8GMM_TYPE_FP32 ? as(bf16, fp32) : as(bf16, bf16);
  } else if (e.type == FP8GMM_TYPE_FP16) {
    e.grad_type == FP8GMM_TYPE_FP32 ? as(fp16, fp32) : as(fp16, fp16);
  } else {
    if constexpr (!MASTER) as(fp32, fp32);
  }
}

// A launch for as many tensors as its arguments hold
template <bool MASTER, bool BITS8>
void launch(const fp8gmm_adamw_tensor* tensors, int n, const Hyper& h, hipStream_t s) {
  int64_t bytes = 0;
  for (int i = 0; i < n; ++i)
    bytes += tensors[i].count * (2 * type_bytes(tensors[i].type) + type_bytes(tensors[i].grad_type) + (BITS8 ? 4 : 16) + (MASTER ? 8 : 0));
  const bool stream = bytes > kStreamBytes;
  const unsigned lds = stream && MASTER && !BITS8 ? kIdleLds : 0;
  auto* kernel = stream ? &adamw_kernel<MASTER, BITS8, true> : &adamw_kernel<MASTER, BITS8, false>;
  constexpr int64_t kMostChunks = 1 << 22;   // of a launch, which holds the largest tensor: a grid has fewer than 2^32 threads
  PartOf<MASTER, BITS8> part = {};
  int used = 0;
  int64_t chunks = 0;
  const auto flush = [&] {
    if (used > 0) hipLaunchKernelGGL(kernel, dim3((unsigned)chunks), dim3(threads(BITS8)), lds, s, part, used, h);
    used = 0;
    chunks = 0;
  };
  for (int i = 0; i < n; ++i) {
    const fp8gmm_adamw_tensor& t = tensors[i];
    const int64_t all = (t.count + sweep(BITS8) - 1) / sweep(BITS8);
    if (all == 0) continue;
    if (used == part.kTensors || chunks + all > kMostChunks) flush();
    pack<MASTER, BITS8>(part, used++, {t.param, t.grad, t.exp_avg, t.exp_avg_sq, t.exp_avg_scale, t.exp_avg_sq_scale, t.master, t.count,
                                       (uint32_t)chunks, t.type, t.grad_type});
    chunks += all;
  }
  flush();
}

int check_tensors(const fp8gmm_adamw_tensor* tensors, int n, const fp8gmm_adamw_step& step) {
  int masters = 0;
  const auto off = [](const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; };
  if (off(step.norm, 4) || off(step.step_dev, 8) || off(step.lr_dev, 4)) return FP8GMM_ERR_ALIGNMENT;
  for (int i = 0; i < n; ++i) {
    const fp8gmm_adamw_tensor& t = tensors[i];
    if (!known_type(t.type) || (t.grad_type != t.type && t.grad_type != FP8GMM_TYPE_FP32)) return FP8GMM_ERR_BAD_FORMAT;
    if (t.count < 0 || t.count > (int64_t)1 << 32) return FP8GMM_ERR_BAD_SHAPE;
    if (t.count == 0) continue;
    if (t.param == nullptr || t.grad == nullptr || t.exp_avg == nullptr || t.exp_avg_sq == nullptr ||
        (step.bits == 8 && (t.exp_avg_scale == nullptr || t.exp_avg_sq_scale == nullptr)))
      return FP8GMM_ERR_NULL_POINTER;
    if (t.master != nullptr && t.type == FP8GMM_TYPE_FP32) return FP8GMM_ERR_BAD_ARGUMENT;
    masters |= t.master != nullptr ? 1 : 2;
    if (off(t.param, type_bytes(t.type)) || off(t.grad, type_bytes(t.grad_type)) || off(t.master, 4) ||
        off(t.exp_avg, step.bits == 8 ? 8 : 4) || off(t.exp_avg_sq, step.bits == 8 ? 8 : 4) || off(t.exp_avg_scale, 4) || off(t.exp_avg_sq_scale, 4))
      return FP8GMM_ERR_ALIGNMENT;
    for (const void* p : {(const void*)t.param, t.grad, (const void*)t.exp_avg, (const void*)t.exp_avg_sq, (const void*)t.exp_avg_scale,
                          (const void*)t.exp_avg_sq_scale, (const void*)t.master})
      if (reinterpret_cast<uintptr_t>(p) >> 48) return FP8GMM_ERR_BAD_ARGUMENT;
  }
  return masters == 3 ? FP8GMM_ERR_BAD_ARGUMENT : FP8GMM_OK;
}

// Nothing is written that something else of the call reads or writes.  The ranges are sorted list by list and merged: the tensors of a list
// mostly come in the order of their addresses.
int check_apart(const fp8gmm_adamw_tensor* tensors, int n, const fp8gmm_adamw_step& step) {
  struct Range {
    uintptr_t begin, end;
    bool writes;
  };
  std::vector<Range> ranges;
  ranges.reserve(7 * (size_t)n + 3);
  const auto before = [](const Range& a, const Range& b) { return a.begin < b.begin; };
  const auto add = [&](const void* p, int64_t bytes, bool writes) {
    const uintptr_t begin = reinterpret_cast<uintptr_t>(p);
    if (p != nullptr && bytes > 0) ranges.push_back({begin, begin + (uintptr_t)bytes, writes});
  };
  const auto merge = [&](size_t from) {
    const auto middle = ranges.begin() + (ptrdiff_t)from;
    if (!std::is_sorted(middle, ranges.end(), before)) std::sort(middle, ranges.end(), before);
    std::inplace_merge(ranges.begin(), middle, ranges.end(), before);
  };
  const auto list = [&](auto address, auto bytes, bool writes) {
    const size_t from = ranges.size();
    for (int i = 0; i < n; ++i) add(tensors[i].*address, bytes(tensors[i]), writes);
    merge(from);
  };
  typedef fp8gmm_adamw_tensor T;
  const auto moments = [&](const T& t) { return t.count * (step.bits / 8); };
  const auto scales = [&](const T& t) { return step.bits == 8 ? (t.count + kBlock - 1) / kBlock * 4 : 0; };
  list(&T::param, [](const T& t) { return t.count * type_bytes(t.type); }, true);
  list(&T::grad, [](const T& t) { return t.count * type_bytes(t.grad_type); }, false);
  list(&T::exp_avg, moments, true);
  list(&T::exp_avg_sq, moments, true);
  list(&T::exp_avg_scale, scales, true);
  list(&T::exp_avg_sq_scale, scales, true);
  list(&T::master, [](const T& t) { return t.count * 4; }, true);
  const size_t from = ranges.size();
  add(step.norm, 4, false);
  add(step.step_dev, 8, false);
  add(step.lr_dev, 4, false);
  merge(from);
  uintptr_t written = 0, read = 0;   // ends of what the ranges so far write and read
  for (const Range& r : ranges) {
    if (r.begin < written || (r.writes && r.begin < read)) return FP8GMM_ERR_BAD_ARGUMENT;
    (r.writes ? written : read) = std::max(r.writes ? written : read, r.end);
  }
  return FP8GMM_OK;
}

int multi_adamw(const fp8gmm_adamw_tensor* tensors, int n, const fp8gmm_adamw_step* step, hipStream_t s) {
  if (n < 0) return FP8GMM_ERR_BAD_ARGUMENT;
  if (step == nullptr || (n > 0 && tensors == nullptr)) return FP8GMM_ERR_NULL_POINTER;
  const fp8gmm_adamw_step& a = *step;
  if ((a.bits != 32 && a.bits != 8) || !(a.beta1 >= 0. && a.beta1 < 1.) || !(a.beta2 >= 0. && a.beta2 < 1.) || !(a.eps >= 0.) ||
      !(a.weight_decay >= 0.) || (a.step_dev == nullptr && a.step < 1) || (a.norm != nullptr && !(a.max_norm >= 0.)) ||
      (a.lr_dev == nullptr && !(a.lr >= 0.)))
    return FP8GMM_ERR_BAD_ARGUMENT;
  int rc = check_tensors(tensors, n, a);
  if (rc == FP8GMM_OK) rc = check_apart(tensors, n, a);
  if (rc != FP8GMM_OK) return rc;
  Hyper h = {};
  h.b1 = (float)a.beta1;
  h.b2 = (float)a.beta2;
  h.c1 = (float)(1. - a.beta1);
  h.c2 = (float)(1. - a.beta2);
  h.eps = (float)a.eps;
  h.max_norm = (float)a.max_norm;
  h.norm = a.norm;
  h.step = a.step_dev;
  h.lr = a.lr_dev;
  const bool device = h.step != nullptr || h.lr != nullptr;
  const double t = (double)a.step, lr = h.lr != nullptr ? 1. : a.lr;
  h.decay = (float)(device ? a.weight_decay : lr * a.weight_decay);
  if (h.step == nullptr) {
    h.rate = (float)((device ? 1. : lr) / (1. - std::pow(a.beta1, t)));
    h.root = (float)(1. / std::sqrt(1. - std::pow(a.beta2, t)));
    h.dither = (uint32_t)a.step * kStep;
  }
  h.log1 = std::log2(a.beta1);   // (of a beta of 0 minus infinity, whose power is 0)
  h.log2 = std::log2(a.beta2);
  h.lr_host = a.lr;
  bool master = false, any = false;
  for (int i = 0; i < n; ++i) {
    master = master || (tensors[i].count > 0 && tensors[i].master != nullptr);
    any = any || tensors[i].count > 0;
  }
  if (!any) return FP8GMM_OK;
  if (a.bits == 8) master ? launch<true, true>(tensors, n, h, s) : launch<false, true>(tensors, n, h, s);
  else master ? launch<true, false>(tensors, n, h, s) : launch<false, false>(tensors, n, h, s);
  return hipGetLastError() == hipSuccess ? FP8GMM_OK : FP8GMM_ERR_LAUNCH;
}

}  // namespace
}  // namespace fp8gmm

extern "C" {

int fp8gmm_multi_adamw(const fp8gmm_adamw_tensor* tensors, int n, const fp8gmm_adamw_step* step, void* stream) {
  try {   // the host's list of ranges is the only thing here that can fail by an exception, which ends at this border
    return fp8gmm::multi_adamw(tensors, n, step, static_cast<hipStream_t>(stream));
  } catch (...) {
    return FP8GMM_ERR_BAD_ARGUMENT;
  }
}

}  // extern "C"
