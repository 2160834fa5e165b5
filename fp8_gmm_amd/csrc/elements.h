// Rows of bf16, fp16 or fp32 in pieces of 16 bytes, for the kernels that take all three (layer_norm.hip, rms_norm.hip,
// embedding.hip, multi_norm.hip, routing.hip, adamw.hip).  A row may begin at any element: its pieces are loaded with the alignment of one, which the hardware
// takes as it takes aligned ones where a piece stays inside a line.
#pragma once

#include <type_traits>

#include "device_utils.h"

namespace fp8gmm {

typedef uint32_t u32x4_any2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_any4 __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

inline int type_bytes(int type) { return type == FP8GMM_TYPE_FP32 ? 4 : 2; }
inline bool known_type(int type) { return type >= FP8GMM_TYPE_BF16 && type <= FP8GMM_TYPE_FP32; }

template <int TYPE>
struct Elements {
  static constexpr bool kWide = TYPE == FP8GMM_TYPE_FP32;
  static constexpr int kVec = kWide ? 4 : 8;   // elements of a piece
  static constexpr int kBytes = kWide ? 4 : 2;
  typedef std::conditional_t<kWide, uint32_t, uint16_t> bits;
  typedef std::conditional_t<kWide, u32x4_any4, u32x4_any2> piece;

  static __device__ __forceinline__ void unpack(u32x4 raw, float (&f)[kVec]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (TYPE == FP8GMM_TYPE_BF16) {
        f[2 * i] = bf16_lo_to_f32(raw[i]);
        f[2 * i + 1] = bf16_hi_to_f32(raw[i]);
      } else if constexpr (TYPE == FP8GMM_TYPE_FP16) {
        const f16x2 h = __builtin_bit_cast(f16x2, (uint32_t)raw[i]);
        f[2 * i] = (float)h.x;
        f[2 * i + 1] = (float)h.y;
      } else {
        f[i] = __uint_as_float(raw[i]);
      }
    }
  }
  // to nearest, ties to even: the one rounding of a result
  static __device__ __forceinline__ u32x4 pack(const float (&f)[kVec]) {
    u32x4 raw;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (TYPE == FP8GMM_TYPE_BF16) {
        raw[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
      } else if constexpr (TYPE == FP8GMM_TYPE_FP16) {
        const f16x2 h = {(_Float16)f[2 * i], (_Float16)f[2 * i + 1]};
        raw[i] = __builtin_bit_cast(uint32_t, h);
      } else {
        raw[i] = __float_as_uint(f[i]);
      }
    }
    return raw;
  }
  static __device__ __forceinline__ bits pack1(float v) {
    if constexpr (TYPE == FP8GMM_TYPE_BF16) return (uint16_t)f32_to_bf16_bits(v);
    else if constexpr (TYPE == FP8GMM_TYPE_FP16) return __builtin_bit_cast(uint16_t, (_Float16)v);
    else return __float_as_uint(v);
  }
  // the piece at `p`, of which the first `n` elements are the row's: zeros behind them.  STREAM: with the streaming hint.
  template <bool STREAM = false>
  static __device__ __forceinline__ u32x4 load(const bits* p, int n) {
    if (n >= kVec) {
      const piece* const at = reinterpret_cast<const piece*>(p);
      if constexpr (STREAM) return __builtin_nontemporal_load(at);
      return *at;
    }
    u32x4 raw = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < kVec - 1; ++i)
      if (i < n) raw[i * kBytes / 4] |= (uint32_t)p[i] << (i * kBytes % 4 * 8);
    return raw;
  }
  template <bool STREAM = false>   // (chosen at run time, the two stores are made one by the compiler, without the hint)
  static __device__ __forceinline__ void store(bits* p, int n, u32x4 raw) {
    if (n >= kVec) {
      if constexpr (STREAM) __builtin_nontemporal_store((piece)raw, reinterpret_cast<piece*>(p));
      else *reinterpret_cast<piece*>(p) = raw;
      return;
    }
#pragma unroll
    for (int i = 0; i < kVec - 1; ++i)
      if (i < n) p[i] = (bits)(raw[i * kBytes / 4] >> (i * kBytes % 4 * 8));
  }
};

// kVec parameters of a row's piece, of the rows' type or in fp32
template <int TYPE, int PTYPE>
struct Parameters {
  typedef Elements<TYPE> E;
  typedef Elements<PTYPE> P;
  static constexpr int kPieces = E::kVec / P::kVec;
  u32x4 raw[kPieces];
  __device__ __forceinline__ void load(const void* p, int at, int n) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
      raw[i] = P::load(static_cast<const typename P::bits*>(p) + at + i * P::kVec, n - i * P::kVec);
  }
  __device__ __forceinline__ void get(float (&f)[E::kVec]) const {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      float part[P::kVec];
      P::unpack(raw[i], part);
#pragma unroll
      for (int j = 0; j < P::kVec; ++j) f[i * P::kVec + j] = part[j];
    }
  }
};

// The sum over groups of 16 lanes, or over all 64, the same bits in every lane of a group: lanes exchange their values inside the
// vector unit (data-parallel primitives), which takes a tenth of the time of an exchange through LDS.
template <int CONTROL>
__device__ __forceinline__ float lanes_step(float v) {
  return v + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CONTROL, 0xf, 0xf, true));
}
template <int WIDTH>
__device__ __forceinline__ float lanes_sum(float v) {
  static_assert(WIDTH == 16 || WIDTH == 64, "a row of the data-parallel primitives, or a wavefront");
  v = lanes_step<0xb1>(v);    // quad_perm: the neighbour
  v = lanes_step<0x4e>(v);    // quad_perm: the other pair
  v = lanes_step<0x141>(v);   // row_half_mirror: the other four
  v = lanes_step<0x140>(v);   // row_mirror: the other eight
  if constexpr (WIDTH == 64) {
    const int bits = __float_as_int(v);
    v = (__int_as_float(__builtin_amdgcn_readlane(bits, 0)) + __int_as_float(__builtin_amdgcn_readlane(bits, 16))) +
        (__int_as_float(__builtin_amdgcn_readlane(bits, 32)) + __int_as_float(__builtin_amdgcn_readlane(bits, 48)));
  }
  return v;
}

// The largest of numbers that are not negative, in the same way
template <int WIDTH>
__device__ __forceinline__ float lanes_max(float v) {
  static_assert(WIDTH == 16 || WIDTH == 64, "a row of the data-parallel primitives, or a wavefront");
  const auto step = [&](auto control) {
    v = fmaxf(v, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), decltype(control)::value, 0xf, 0xf, true)));
  };
  step(std::integral_constant<int, 0xb1>{});
  step(std::integral_constant<int, 0x4e>{});
  step(std::integral_constant<int, 0x141>{});
  step(std::integral_constant<int, 0x140>{});
  if constexpr (WIDTH == 64) {
    const int bits = __float_as_int(v);
    v = fmaxf(fmaxf(__int_as_float(__builtin_amdgcn_readlane(bits, 0)), __int_as_float(__builtin_amdgcn_readlane(bits, 16))),
              fmaxf(__int_as_float(__builtin_amdgcn_readlane(bits, 32)), __int_as_float(__builtin_amdgcn_readlane(bits, 48))));
  }
  return v;
}

}  // namespace fp8gmm
