// Device helpers shared by the attention kernels (gfx950).
#pragma once

#include <type_traits>

#include "w8a8_internal.h"

namespace w8a8 {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;

// C layout (lane l, register i): row 4(l/16) + i, column l%16; a and b give
// lane l elements 8(l/16) .. +7 of row (column) l%16.
template <typename T>
__device__ inline f32x4 mfma_16x16x32(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (std::is_same<T, __half>::value) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a),
                                                  __builtin_bit_cast(h8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a),
                                                   __builtin_bit_cast(b8, b), c, 0, 0, 0);
  }
}

// 2^x by the hardware's instruction (one ulp; results below the smallest
// normal value are 0).
__device__ inline float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// The reference that scores are taken against (in powers of two) follows the
// running maximum lazily: set kBelow below a maximum, raised once a score is
// kSlack above it.  Binary16 probabilities: up to 2^15, so that one of 2^-31 of
// the largest still counts, and the running sums are rarely rescaled; bfloat16
// ones, whose range is binary32's: up to 1, so that no product with a value
// near the type's largest overflows.
template <typename T> struct Reference {
  static constexpr bool kHalf = std::is_same<T, __half>::value;
  static constexpr float kBelow = kHalf ? 7.0f : -8.0f;
  static constexpr float kSlack = kHalf ? 15.0f : 0.0f;
};

// p0 and p1 as the sum of two 16-bit values each, packed: p = hi + lo to 22
// bits (binary16) or 16 (bfloat16), both parts cut off, not rounded.
template <typename T>
__device__ inline void split2(float p0, float p1, uint32_t& hi, uint32_t& lo) {
  if constexpr (std::is_same<T, __half>::value) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(p0, p1);
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t,
                            __builtin_amdgcn_cvt_pkrtz(p0 - static_cast<float>(h[0]),
                                                       p1 - static_cast<float>(h[1])));
  } else {
    const uint32_t u0 = __float_as_uint(p0), u1 = __float_as_uint(p1);
    hi = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
    const float r0 = p0 - __uint_as_float(u0 & 0xffff0000u);
    const float r1 = p1 - __uint_as_float(u1 & 0xffff0000u);
    lo = __builtin_amdgcn_perm(__float_as_uint(r1), __float_as_uint(r0), 0x07060302u);
  }
}

// Inclusive sum over the wavefront's lanes (each step a DPP move: shifts by 1,
// 2, 4 and 8 in rows of 16 lanes, then the rows' last lanes to the next ones).
__device__ inline uint32_t scan64(uint32_t v) {
  auto moved = [](uint32_t x, auto ctrl, auto rows) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
        0, static_cast<int>(x), decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
  };
  using std::integral_constant;
  const integral_constant<int, 0xf> all;
  v += moved(v, integral_constant<int, 0x111>{}, all);
  v += moved(v, integral_constant<int, 0x112>{}, all);
  v += moved(v, integral_constant<int, 0x114>{}, all);
  v += moved(v, integral_constant<int, 0x118>{}, all);
  v += moved(v, integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});
  v += moved(v, integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
  return v;
}
__device__ inline int lane_value(uint32_t v, int lane) {
  return __builtin_amdgcn_readlane(static_cast<int>(v), lane);
}

}  // namespace w8a8
