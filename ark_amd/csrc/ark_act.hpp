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

// fp32 -> T with the fp32 value formed first: fp16's conversion must not merge
// with the multiply before it (see f2h).
template <typename T>
__device__ __forceinline__ T narrow(float f) {
  asm("" : "+v"(f));
  return (T)f;
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

// The byte of x in a group of exponent byte s: q + 128, with |q| held to 127,
// or to 63 at fp16's top exponent.  A group that is NaN stores q = 0.
template <uint32_t DT>
__device__ __forceinline__ uint32_t act_byte(float x, uint32_t s, float down) {
  float q = __builtin_rintf(x * down);
  const float most = DT == ARK_ACT_F16 && s >= 143u ? 63.0f : 127.0f;
  q = __builtin_fminf(__builtin_fmaxf(q, -most), most);
  return s == 255u ? 128u : (uint32_t)((int)q + 128);
}
__device__ __forceinline__ float act_value(uint32_t byte, float up) {
  return (float)((int)byte - 128) * up;
}

}  // namespace dev
}  // namespace ark
