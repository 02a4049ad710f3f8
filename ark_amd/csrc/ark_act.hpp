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
// carry of adding 0x1FFFF to the bits does.
template <uint32_t DT>
__device__ __forceinline__ uint32_t act_exponent(uint32_t most) {
  const uint32_t e = (most + 0x1FFFFu) >> 23;
  constexpr uint32_t lo = DT == ARK_ACT_F16 ? 133u - 24u : 133u - 126u;
  const uint32_t s = e < lo ? lo : e > 254u ? 254u : e;
  return most >= 0x7F800000u ? 255u : s;
}

// 2^-e and 2^e of an exponent byte; NaN for 255.
__device__ __forceinline__ float act_down(uint32_t s) {
  return __uint_as_float(s == 255u ? 0x7FC00000u : (260u - s) << 23);
}
__device__ __forceinline__ float act_up(uint32_t s) {
  return __uint_as_float(s == 255u ? 0x7FC00000u : (s - 6u) << 23);
}

// What quantises a group: x 2^-e rounds to a whole number in the last place of
// 1.5 * 2^23 + 128, whose low byte then is q + 128.  |x| is held to 127 * 2^e
// first (63 * 2^10 at fp16's top exponent), which binds only where e is the
// largest there is.  A group that is NaN gets bytes that mean nothing.
struct ActScale {
  uint32_t s;
  float down, most;
};
template <uint32_t DT>
__device__ __forceinline__ ActScale act_scale(uint32_t most) {
  const uint32_t s = act_exponent<DT>(most);
  return {s, act_down(s), act_up(s) * (DT == ARK_ACT_F16 && s >= 143u ? 63.0f : 127.0f)};
}
// Four values' bytes, the first lowest.
__device__ __forceinline__ uint32_t act_bytes4(const ActScale& a, float x0, float x1, float x2,
                                               float x3) {
  const auto one = [&](float x) {
    return __float_as_uint(__builtin_fmaf(__builtin_amdgcn_fmed3f(x, -a.most, a.most), a.down,
                                          12583040.0f));
  };
  const uint32_t lo = __builtin_amdgcn_perm(one(x1), one(x0), 0x0C0C0400u);
  const uint32_t hi = __builtin_amdgcn_perm(one(x3), one(x2), 0x04000C0Cu);
  return lo | hi;
}
__device__ __forceinline__ float act_value(uint32_t byte, float up) {
  return (float)((int)byte - 128) * up;
}

}  // namespace dev
}  // namespace ark
