// ark_act.hpp -- element types and the 8-bit form of activations
// (include/ark_act.h), shared by the kernels that write and read it.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ark_act.h"
#include "ark_device.hpp"

namespace ark {

inline uint32_t act_elem_size(uint32_t dtype) { return dtype == ARK_ACT_F32 ? 4u : 2u; }

// Where the exponents of an 8-bit form start, in bytes from its values.
inline uint64_t act_groups(uint64_t tokens) {
  return tokens / ARK_ACT_GROUP + (tokens % ARK_ACT_GROUP != 0);
}

namespace dev {

// One element of type DT, widened and narrowed (round to nearest even).
template <uint32_t DT>
struct Elem;
template <>
struct Elem<ARK_ACT_F16> {
  typedef _Float16 T;
};
template <>
struct Elem<ARK_ACT_BF16> {
  typedef __bf16 T;
};
template <>
struct Elem<ARK_ACT_F32> {
  typedef float T;
};
template <uint32_t DT>
using elem_t = typename Elem<DT>::T;

// Two fp32 values to 16 bits each, to nearest even, the first in the low half.
typedef float f32x2 __attribute__((ext_vector_type(2)));
template <uint32_t DT>
__device__ __forceinline__ uint32_t narrow2(float a, float b) {
  typedef elem_t<DT> T2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), T2));
}

// The magnitudes of two 16-bit values, the larger of each pair of halves: ordered
// as whole numbers, inf and NaN above all others.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a),
                                                                __builtin_bit_cast(u16x2, b)));
}

// The exponent byte of a group whose largest magnitude has the fp32 bits
// `most` (sign clear): e + 133 for the smallest e with most <= 127 * 2^e, 255
// when it is inf or NaN.  most = 1.f * 2^(E - 127) asks for e = E - 133 while
// f <= 0x7E0000 (1.984375 = 127 / 64) and one more above it, which is what the
// carry of adding 0x1FFFF to the bits does.  fp16's largest number gives 143, so
// only there what is not finite needs no test of its own.
template <uint32_t DT>
__device__ __forceinline__ uint32_t act_exponent(uint32_t most) {
  if constexpr (DT == ARK_ACT_F16) return min(max((most + 0x1FFFFu) >> 23, 133u - 24u), 255u);
  const uint32_t s = max((min(most, 0x7F7E0000u) + 0x1FFFFu) >> 23, 133u - 126u);
  return most >= 0x7F800000u ? 255u : s;
}

// 2^e of an exponent byte; NaN for 255.
__device__ __forceinline__ float act_up(uint32_t s) {
  return __uint_as_float(s == 255u ? 0x7FC00000u : (s - 6u) << 23);
}

// The largest exponent of a type, where |x| can pass the largest value there
// (127 * 2^121, or 63 * 2^10 in fp16) and is held to it.
template <uint32_t DT>
constexpr uint32_t kActTop = DT == ARK_ACT_F16 ? 143u : 254u;
template <uint32_t DT>
__device__ __forceinline__ float act_hold(uint32_t s, float x) {
  const float most = DT != ARK_ACT_F16 ? 0x1.FCp127f : s >= kActTop<DT> ? 64512.0f : 65536.0f;
  return __builtin_amdgcn_fmed3f(x, -most, most);
}

// Four values' bytes under exponent byte s, the first lowest: x 2^-e rounds to a
// whole number in the last place of 1.5 * 2^23 + 128, whose low byte then is
// q + 128.  A group that is NaN gets bytes that mean nothing.
__device__ __forceinline__ uint32_t act_bytes4(uint32_t s, float x0, float x1, float x2, float x3) {
  const float down = __uint_as_float((260u - s) << 23);
  const auto one = [&](float x) {
    return __float_as_uint(__builtin_fmaf(x, down, 12583040.0f));
  };
  const uint32_t lo = __builtin_amdgcn_perm(one(x1), one(x0), 0x0C0C0400u);
  const uint32_t hi = __builtin_amdgcn_perm(one(x3), one(x2), 0x04000C0Cu);
  return lo | hi;
}

// Value i of a word of bytes: q 2^e.
__device__ __forceinline__ float act_value(uint32_t word, uint32_t i, float up) {
  return (float)(int8_t)((word ^ 0x80808080u) >> (8 * i)) * up;
}

}  // namespace dev
}  // namespace ark
