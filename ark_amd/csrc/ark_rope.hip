// ark_rope.hip -- rotary positions and the norms of queries and keys
// (include/ark_rope.h).
#include <math.h>

#include <new>
#include <type_traits>
#include <vector>

#include "ark_act.hpp"
#include "ark_common.hpp"
#include "ark_rope.h"

namespace {

using namespace ark::dev;

// A [batch][tokens][heads][head_dim] array; strides in elements.
struct Array {
  const void* p;
  uint64_t sb, st, sh;
};

// One of a call's two tensors, q or k; of the two, those that have heads, the
// first of them first.  Kernels are launched for no others.
struct Part {
  Array x;           // the input; for the backward pass the norm's input
  Array dy;          // backward: the gradient of the output
  Array y;           // the output
  const void* gain;  // head_dim values
  uint8_t* act;      // 8-bit form written or read, or NULL
  uint32_t heads;
};

struct Args {
  Part part[2];
  const uint64_t* turns;  // 2^64 inv_freq / (2 pi) of every pair
  const void* positions;
  float* partial;         // backward: [part][block][head_dim] of the gains' gradients
  uint64_t start, tokens, all;  // all: batch * tokens
  float magnitude, eps, one_over_head;
  uint32_t position_bytes, head, rotary, layout, inverse, gain_dtype;
  uint32_t lanes;         // of a row: a power of two
  uint32_t tile;          // tokens a block takes at once
  uint32_t slices;        // tiles_kernel: blocks that share a group's heads
};

// sin and cos of an angle given in turns / 2^32, by eighths: |r| <= pi / 4
// after the nearest quarter turn is taken off, then the Taylor series (what
// is left out is below 2^-28 of the result).
__device__ __forceinline__ void sincos_turns(uint32_t phase, float* s, float* c) {
  const uint32_t h = phase + 0x20000000u;
  const int r = (int)(h & 0x3FFFFFFFu) - 0x20000000;
  const float a = (float)r * 1.46291807926715968e-9f;  // 2 pi / 2^32
  const float z = a * a;
  float p = __builtin_fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
  p = __builtin_fmaf(z, p, 8.3333333e-3f);
  p = __builtin_fmaf(z, p, -1.6666667e-1f);
  const float sn = __builtin_fmaf(a * z, p, a);
  float w = __builtin_fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
  w = __builtin_fmaf(z, w, -1.3888889e-3f);
  w = __builtin_fmaf(z, w, 4.1666667e-2f);
  w = __builtin_fmaf(z, w, -0.5f);
  const float cs = __builtin_fmaf(z, w, 1.0f);
  const uint32_t k = h >> 30;
  const float u = k & 1u ? cs : sn, v = k & 1u ? sn : cs;
  *s = __uint_as_float(__float_as_uint(u) ^ ((k & 2u) << 30));
  *c = __uint_as_float(__float_as_uint(v) ^ (((k + 1u) & 2u) << 30));
}

__device__ __forceinline__ int64_t position_at(const Args& a, uint64_t bt) {
  if (!a.positions) return (int64_t)(a.start + (bt < a.tokens ? bt : bt % a.tokens));
  return a.position_bytes == 8 ? ((const int64_t*)a.positions)[bt]
                               : ((const int32_t*)a.positions)[bt];
}

// Top 32 bits of position * turns, modulo a whole turn.
__device__ __forceinline__ uint32_t phase_of(int64_t position, uint64_t turns) {
  return (uint32_t)(((uint64_t)position * turns) >> 32);
}

__device__ __forceinline__ float gain_at(const Args& a, const void* gain, uint32_t j) {
  if (a.gain_dtype == ARK_ACT_F16) return (float)((const _Float16*)gain)[j];
  if (a.gain_dtype == ARK_ACT_BF16) return (float)((const __bf16*)gain)[j];
  return ((const float*)gain)[j];
}

// op of a lane's value and that of the lane that differs in one bit, 1 to 32, in
// both lanes; no bit needs LDS.  Bit 4 mirrors eight lanes, so it is for values
// that already are the same in lanes that differ in bits 1 and 2.
template <uint32_t BIT, typename F>
__device__ __forceinline__ uint32_t fold(uint32_t v, F op) {
  if constexpr (BIT >= 16) {
    // two rows of 16 lanes (or of 32) change places: both rows then hold both values
    const auto r = BIT == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false)
                             : __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return op(r[0], r[1]);
  } else {
    constexpr int kHow = BIT == 1 ? 0xB1     // quad 1 0 3 2
                         : BIT == 2 ? 0x4E   // quad 2 3 0 1
                         : BIT == 4 ? 0x141  // half row mirrored
                                    : 0x128; // row turned by 8
    return op(v, __builtin_amdgcn_mov_dpp(v, kHow, 0xF, 0xF, false));
  }
}
template <uint32_t BIT>
__device__ __forceinline__ float fold_sum(float v) {
  return __uint_as_float(fold<BIT>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}

// The sum over the lanes of a row, 8 to 64 of them, in every lane.
__device__ __forceinline__ float row_sum(float v, uint32_t lanes) {
  v = fold_sum<1>(v);
  v = fold_sum<2>(v);
  v = fold_sum<4>(v);
  if (lanes >= 16) v = fold_sum<8>(v);
  if (lanes >= 32) v = fold_sum<16>(v);
  if (lanes == 64) v = fold_sum<32>(v);
  return v;
}

// 1 / sqrt(a): the instruction's, within an ulp; it takes no subnormals.
__device__ __forceinline__ float inverse_root(float a) {
  const bool small = a < 0x1p-100f;
  return __builtin_amdgcn_rsqf(small ? a * 0x1p100f : a) * (small ? 0x1p50f : 1.0f);
}

enum Op { kRope, kNorm, kBack };

constexpr uint32_t kBlock = 256, kWaves = 4;

// N neighbouring elements as they lie in memory, at any element's alignment
// (gfx950 takes unaligned global accesses).
template <uint32_t DT, uint32_t N>
struct Raw {
  static constexpr uint32_t kWords = DT == ARK_ACT_F32 ? N : (N + 1) / 2;
  uint32_t w[kWords];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (uint32_t i = 0; i < kWords; ++i) w[i] = 0;
  }
  __device__ __forceinline__ void load(const elem_t<DT>* p) {
    if constexpr (DT != ARK_ACT_F32 && N == 1) {
      w[0] = ld_g<uint16_t>(p);
    } else {
      typedef uint32_t T __attribute__((ext_vector_type(kWords), aligned(DT == ARK_ACT_F32 ? 4 : 2)));
      const T v = *(const ARK_GLOBAL T*)p;
#pragma unroll
      for (uint32_t i = 0; i < kWords; ++i) w[i] = v[i];
    }
  }
  __device__ __forceinline__ void store(elem_t<DT>* p) const {
    if constexpr (DT != ARK_ACT_F32 && N == 1) {
      st_g<uint16_t>(p, (uint16_t)w[0]);
    } else {
      typedef uint32_t T __attribute__((ext_vector_type(kWords), aligned(DT == ARK_ACT_F32 ? 4 : 2)));
      T v;
#pragma unroll
      for (uint32_t i = 0; i < kWords; ++i) v[i] = w[i];
      *(ARK_GLOBAL T*)p = v;
    }
  }
  __device__ __forceinline__ float get(uint32_t i) const {
    if constexpr (DT == ARK_ACT_F32)
      return __uint_as_float(w[i]);
    else if constexpr (DT == ARK_ACT_F16)
      return h2f(w[i / 2] >> (i % 2 * 16) & 0xFFFFu);
    else
      return __uint_as_float(i % 2 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
  }
  __device__ __forceinline__ void set(const float* f) {
#pragma unroll
    for (uint32_t i = 0; i < kWords; ++i) {
      if constexpr (DT == ARK_ACT_F32)
        w[i] = __float_as_uint(f[i]);
      else
        w[i] = narrow2<DT>(f[2 * i], N > 1 ? f[2 * i + 1] : 0.0f);
    }
  }
};

// N elements of a and N after them, in order, to every other one and those
// between; and back.
template <uint32_t DT, uint32_t N>
__device__ __forceinline__ void unmix(Raw<DT, N>& a, Raw<DT, N>& b) {
  uint32_t t[2 * N], *const aw = a.w, *const bw = b.w;
  if constexpr (DT == ARK_ACT_F32) {
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) t[i] = aw[i], t[N + i] = bw[i];
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) aw[i] = t[2 * i], bw[i] = t[2 * i + 1];
  } else if constexpr (N > 1) {
#pragma unroll
    for (uint32_t i = 0; i < N / 2; ++i) t[i] = aw[i], t[N / 2 + i] = bw[i];
#pragma unroll
    for (uint32_t i = 0; i < N / 2; ++i) {
      aw[i] = __builtin_amdgcn_perm(t[2 * i + 1], t[2 * i], 0x05040100u);
      bw[i] = __builtin_amdgcn_perm(t[2 * i + 1], t[2 * i], 0x07060302u);
    }
  }
}
template <uint32_t DT, uint32_t N>
__device__ __forceinline__ void mix(Raw<DT, N>& a, Raw<DT, N>& b) {
  uint32_t t[2 * N], *const aw = a.w, *const bw = b.w;
  if constexpr (DT == ARK_ACT_F32) {
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) t[2 * i] = aw[i], t[2 * i + 1] = bw[i];
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) aw[i] = t[i], bw[i] = t[N + i];
  } else if constexpr (N > 1) {
#pragma unroll
    for (uint32_t i = 0; i < N / 2; ++i) {
      t[2 * i] = __builtin_amdgcn_perm(bw[i], aw[i], 0x05040100u);
      t[2 * i + 1] = __builtin_amdgcn_perm(bw[i], aw[i], 0x07060302u);
    }
#pragma unroll
    for (uint32_t i = 0; i < N / 2; ++i) aw[i] = t[i], bw[i] = t[N / 2 + i];
  }
}

// A row (a head of a token) over its lanes: a lane takes V neighbouring pairs,
// and of long rows with V = 1 the pairs 64 on too, K in all.  Pairs past the
// rotary ones are made of what is left of the head the same way, and turn by
// nothing.  A lane's pairs are two stretches of V elements, u and v, in the half
// layout; in the interleaved one they are one of 2V, sorted once loaded.  Lanes
// past the row's end load its first pairs, add nothing to its sums and store
// nothing; the last pair of an odd head has no second element.
template <uint32_t DT, uint32_t V, uint32_t K>
struct Row {
  static constexpr uint32_t kE = V * K;
  typedef elem_t<DT> T;
  uint32_t pair[K], eu[K], ev[K];
  bool on[K], pairs_v[K];
  uint32_t half;
  bool mixed;  // interleaved
  __device__ __forceinline__ Row(const Args& a, uint32_t lane) {
    half = a.rotary / 2;
    mixed = a.layout == ARK_ROPE_INTERLEAVED;
    const uint32_t rest = (a.head - a.rotary + 1) / 2;
#pragma unroll
    for (uint32_t k = 0; k < K; ++k) {
      pair[k] = (lane + 64 * k) * V;
      const uint32_t p = pair[k];
      on[k] = p < half + rest;
      if (mixed) {
        eu[k] = 2 * p;
        ev[k] = 2 * p + (V == 1 ? 1 : V);  // as loaded
      } else {
        eu[k] = p < half ? p : a.rotary + p - half;
        ev[k] = p < half ? half + p : a.rotary + rest + p - half;
      }
      pairs_v[k] = on[k] && ev[k] < a.head;
      if (!on[k]) eu[k] = 0;
      if (!pairs_v[k]) ev[k] = eu[k];
    }
  }
  // Places in the row are formed where they are used: kept through a loop they
  // cost a register an element.
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (uint32_t k = 0; k < K; ++k) asm volatile("" : "+v"(eu[k]), "+v"(ev[k]));
  }
  struct Data {
    Raw<DT, V> u[K], v[K];
    __device__ __forceinline__ void load(const Row& r, const T* p) {
#pragma unroll
      for (uint32_t k = 0; k < K; ++k) {
        u[k].load(p + r.eu[k]);
        v[k].load(p + r.ev[k]);
        if (V == 1 && !r.pairs_v[k]) v[k].clear();
      }
    }
    // what the interleaved layout loaded, e0 e1 ..., to e0 e2 ... and e1 e3 ...
    __device__ __forceinline__ void sort(const Row& r) {
      if (V > 1 && r.mixed)
#pragma unroll
        for (uint32_t k = 0; k < K; ++k) unmix(u[k], v[k]);
    }
    __device__ __forceinline__ void store(const Row& r, T* p) {
      if (V > 1 && r.mixed)
#pragma unroll
        for (uint32_t k = 0; k < K; ++k) mix(u[k], v[k]);
#pragma unroll
      for (uint32_t k = 0; k < K; ++k) {
        if (r.on[k]) u[k].store(p + r.eu[k]);
        if (r.pairs_v[k]) v[k].store(p + r.ev[k]);
      }
    }
    __device__ __forceinline__ void opaque() {
#pragma unroll
      for (uint32_t k = 0; k < K; ++k)
#pragma unroll
        for (uint32_t i = 0; i < Raw<DT, V>::kWords; ++i)
          asm volatile("" : "+v"(u[k].w[i]), "+v"(v[k].w[i]));
    }
    // element by element the larger magnitude, inf and NaN above all others
    __device__ __forceinline__ void larger(const Data& d) {
#pragma unroll
      for (uint32_t k = 0; k < K; ++k)
#pragma unroll
        for (uint32_t i = 0; i < Raw<DT, V>::kWords; ++i) {
          u[k].w[i] = larger2(u[k].w[i], d.u[k].w[i]);
          v[k].w[i] = larger2(v[k].w[i], d.v[k].w[i]);
        }
    }
    template <uint32_t BIT>
    __device__ __forceinline__ void larger_across() {
#pragma unroll
      for (uint32_t k = 0; k < K; ++k)
#pragma unroll
        for (uint32_t i = 0; i < Raw<DT, V>::kWords; ++i) {
          u[k].w[i] = fold<BIT>(u[k].w[i], larger2);
          v[k].w[i] = fold<BIT>(v[k].w[i], larger2);
        }
    }
    static __device__ __forceinline__ uint32_t larger2(uint32_t a, uint32_t b) {
      return DT == ARK_ACT_F32 ? max(a, b & 0x7FFFFFFFu) : max_u16x2(a, b & 0x7FFF7FFFu);
    }
    // element `second` of the lane's pair e
    __device__ __forceinline__ float get(uint32_t e, bool second) const {
      return second ? v[e / V].get(e % V) : u[e / V].get(e % V);
    }
    __device__ __forceinline__ void set(const float* fu, const float* fv) {
#pragma unroll
      for (uint32_t k = 0; k < K; ++k) u[k].set(fu + k * V), v[k].set(fv + k * V);
    }
  };
  // where element `second` of pair e lies in the row
  __device__ __forceinline__ uint32_t at(uint32_t e, bool second) const {
    const uint32_t k = e / V, i = e % V;
    return mixed ? eu[k] + 2 * i + second : (second ? ev[k] : eu[k]) + i;
  }
  __device__ __forceinline__ bool has(uint32_t e, bool second) const {
    return second ? pairs_v[e / V] : on[e / V];
  }
  __device__ __forceinline__ void gains(const Args& a, const void* g, float* gu, float* gv) const {
#pragma unroll
    for (uint32_t e = 0; e < kE; ++e) {
      gu[e] = gain_at(a, g, at(e, false));
      gv[e] = gain_at(a, g, has(e, true) ? at(e, true) : 0);
    }
  }
  // the pairs' cosines and sines from a token's line of the block's table; for pairs
  // past the rotary ones numbers that are not used
  __device__ __forceinline__ void turn(const float2* line, float* c, float* s) const {
#pragma unroll
    for (uint32_t e = 0; e < kE; ++e) c[e] = 1.0f, s[e] = 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < K; ++k)
      if (pair[k] < half)
#pragma unroll
        for (uint32_t i = 0; i < V; ++i) {
          const float2 t = line[pair[k] + i];
          c[k * V + i] = t.x, s[k * V + i] = t.y;
        }
  }
  // y = the rotation of x, or of x r gain.  Pairs past the rotary ones are two values
  // that have nothing to do with each other: a product with their sine of 0 would
  // bring an inf or NaN of the one, and the sign of its zero, into the other, so
  // they are kept (chosen under a condition of the whole call: without it the
  // backward pass's registers spill, 32768 tokens of 16 + 16 heads of 128, bf16,
  // both ways 601 us for 283)
  template <Op OP>
  __device__ __forceinline__ void forward(const Args& a, uint32_t lanes, const Data& x, const float* gu,
                                          const float* gv, const float* c, const float* s,
                                          Data* y) const {
    float u[kE], v[kE], r = 1.0f, q = 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < K; ++k) {
      float p = 0.0f;
#pragma unroll
      for (uint32_t e = k * V; e < k * V + V; ++e) {
        u[e] = x.get(e, false), v[e] = x.get(e, true);
        p = __builtin_fmaf(u[e], u[e], p);
        p = __builtin_fmaf(v[e], v[e], p);
      }
      q += on[k] ? p : 0.0f;
    }
    if constexpr (OP == kNorm) r = inverse_root(row_sum(q, lanes) * a.one_over_head + a.eps);
#pragma unroll
    for (uint32_t e = 0; e < kE; ++e) {
      const float nu = OP == kNorm ? u[e] * (r * gu[e]) : u[e];
      const float nv = OP == kNorm ? v[e] * (r * gv[e]) : v[e];
      u[e] = __builtin_fmaf(nu, c[e], -(nv * s[e]));
      v[e] = __builtin_fmaf(nu, s[e], nv * c[e]);
      if (a.rotary < a.head && pair[e / V] >= half) u[e] = nu, v[e] = nv;
    }
    y->set(u, v);
  }
  // dx from dy and x, and dy rotated back times x r into the gain's sums.  A row that
  // is not `there` comes as zeros and adds nothing: without eps its 1 / rms is
  // infinite, and is taken as 0
  __device__ __forceinline__ void backward(const Args& a, uint32_t lanes, bool there,
                                           const Data& dy, const float* xu,
                                           const float* xv, const float* gu, const float* gv,
                                           const float* c, const float* s, float* su, float* sv,
                                           Data* dx) const {
    float du[kE], dv[kE], q = 0.0f, along = 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < K; ++k) {
      float p = 0.0f, l = 0.0f;
#pragma unroll
      for (uint32_t e = k * V; e < k * V + V; ++e) {
        const float u = dy.get(e, false), v = dy.get(e, true);
        du[e] = __builtin_fmaf(u, c[e], v * s[e]);
        dv[e] = __builtin_fmaf(v, c[e], -(u * s[e]));
        if (a.rotary < a.head && pair[k] >= half) du[e] = u, dv[e] = v;
        p = __builtin_fmaf(xu[e], xu[e], p);
        p = __builtin_fmaf(xv[e], xv[e], p);
        l = __builtin_fmaf(du[e] * gu[e], xu[e], l);
        l = __builtin_fmaf(dv[e] * gv[e], xv[e], l);
      }
      q += on[k] ? p : 0.0f;
      along += on[k] ? l : 0.0f;
    }
    const float root = inverse_root(row_sum(q, lanes) * a.one_over_head + a.eps);
    const float r = there ? root : 0.0f;
    along = row_sum(along, lanes) * a.one_over_head * r * r;
#pragma unroll
    for (uint32_t e = 0; e < kE; ++e) {
      su[e] = __builtin_fmaf(du[e], xu[e] * r, su[e]);
      sv[e] = __builtin_fmaf(dv[e], xv[e] * r, sv[e]);
      du[e] = r * __builtin_fmaf(-xu[e], along, du[e] * gu[e]);
      dv[e] = r * __builtin_fmaf(-xv[e], along, dv[e] * gv[e]);
    }
    dx->set(du, dv);
  }
  // a wave's sums of the gain's gradient, its rows' lanes together, into LDS
  __device__ __forceinline__ void gather(const Args& a, uint32_t lanes, float* su, float* sv, float* out) const {
#pragma unroll
    for (uint32_t e = 0; e < kE; ++e) {
      if (lanes <= 8) su[e] = fold_sum<8>(su[e]), sv[e] = fold_sum<8>(sv[e]);
      if (lanes <= 16) su[e] = fold_sum<16>(su[e]), sv[e] = fold_sum<16>(sv[e]);
      if (lanes <= 32) su[e] = fold_sum<32>(su[e]), sv[e] = fold_sum<32>(sv[e]);
      if (threadIdx.x % 64 < lanes) {
        if (has(e, false)) out[at(e, false)] = su[e];
        if (has(e, true)) out[at(e, true)] = sv[e];
      }
    }
  }
};

// What a block keeps of its tokens in LDS: their cosines and sines, one line of
// rotary / 2 a token, and where each token starts in the part's x, dy and y.
struct Tokens {
  float2* turns;
  uint64_t* at;  // [token][x, dy, y]
  __device__ __forceinline__ Tokens(const Args& a, uint8_t* lds) {
    at = (uint64_t*)lds;
    turns = (float2*)(lds + a.tile * 24);
  }
  __device__ __forceinline__ void starts(const Args& a, const Part& p, uint64_t first,
                                         uint32_t n) const {
    for (uint32_t i = threadIdx.x; i < n * 3; i += kBlock) {
      const uint64_t bt = first + i / 3;
      const Array& r = i % 3 == 0 ? p.x : i % 3 == 1 ? p.dy : p.y;
      uint64_t b = 0, t = bt;
      if (a.all != a.tokens) b = bt / a.tokens, t = bt % a.tokens;
      at[i] = b * r.sb + t * r.st;
    }
  }
  // N of a lane's angles at a time, whose positions and frequencies are then on
  // their way together: two for blocks of 32 tokens (237M training pass, backward
  // 38.0 us, 41.2 by ones), one for those of a few, which have no more
  template <uint32_t N>
  __device__ __forceinline__ void angles(const Args& a, uint64_t first, uint32_t n,
                                         bool back) const {
    const uint32_t half = a.rotary / 2, all = n * half;
    for (uint32_t i = threadIdx.x; i < all; i += N * kBlock) {
      uint64_t turn[N];
      int64_t position[N];
#pragma unroll
      for (uint32_t k = 0; k < N; ++k) {
        const uint32_t e = N == 1 ? i : min(i + k * kBlock, all - 1), t = e / half;
        turn[k] = a.turns[e - t * half];
        position[k] = position_at(a, first + t);
      }
#pragma unroll
      for (uint32_t k = 0; k < N; ++k) {
        float s, c;
        sincos_turns(phase_of(position[k], turn[k]), &s, &c);
        if (N == 1 || i + k * kBlock < all)
          turns[i + k * kBlock] =
              make_float2(c * a.magnitude, s * (back ? -a.magnitude : a.magnitude));
      }
    }
  }
};

// Rows of tokens taken `tile` at a time by every block in turn: a wave takes 64
// / lanes rows at once, neighbouring heads of a token, kUnroll times over before
// it works on the first.  A token's angles are formed once, in LDS, for all its
// heads; a row's sum of squares stays in its lanes.  One pass over the data,
// bound by HBM when long: 16384 tokens of 16 + 16 heads of 128, bf16, rotated, 268
// MB in 46 us, 5.8 TB/s; 5003 tokens of 12 + 12 heads of 64, fp32, 61 MB in 11 us,
// 5.6 TB/s.  4099 tokens of 12 + 12 of 64 normed and rotated, fp16, 25 MB, take
// 10 us, mostly the way through one round of blocks: angles, loads, sums, stores.
// Backward from tensors, 32768 tokens of 16 + 16 heads of 128, bf16, 805 MB take 176
// us, 4.6 TB/s; in fp32, four pairs a lane, its registers spill 72 bytes a lane.
template <uint32_t DT, Op OP, uint32_t V, uint32_t K>
__global__ __launch_bounds__(kBlock, 4) void rows_kernel(Args a) {
  typedef Row<DT, V, K> R;
  typedef elem_t<DT> T;
  constexpr uint32_t kUnroll = V == 4 ? 2 : 1;
  extern __shared__ __align__(16) uint8_t lds[];
  const Tokens tok(a, lds);
  const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const R row(a, lane % a.lanes);
  const uint32_t at_once = 64 / a.lanes;
  const Part& P = a.part[blockIdx.y];
  const uint64_t columns = (uint64_t)P.heads * a.head;
  float su[R::kE] = {}, sv[R::kE] = {}, gu[R::kE], gv[R::kE];
  // the condition always holds, and leaves the gains a block of their own: backward,
  // 32768 tokens of 16 + 16 heads of 128, bf16, with it 285 us of both passes, 289
  // without (fences for the scheduler or the values do not do the same)
  if (OP != kRope && P.heads) row.gains(a, P.gain, gu, gv);
  for (uint64_t first = (uint64_t)blockIdx.x * a.tile; first < a.all;
       first += (uint64_t)gridDim.x * a.tile) {
    const uint32_t n = (uint32_t)(a.all - first < a.tile ? a.all - first : a.tile);
    __syncthreads();
    tok.starts(a, P, first, n);
    __syncthreads();
    {
      const uint8_t* exps = P.act + (a.all + ARK_ACT_GROUP - 1) / ARK_ACT_GROUP * columns * ARK_ACT_GROUP;
      typename R::Data x[kUnroll], dy[kUnroll];
      uint32_t t[kUnroll], h[kUnroll];
      bool in[kUnroll];
      const auto load = [&](uint32_t r0) {
#pragma unroll
        for (uint32_t i = 0; i < kUnroll; ++i) {
          const uint32_t r = r0 + i * kWaves * at_once + lane / a.lanes;
          in[i] = r < n * P.heads;
          t[i] = in[i] ? r / P.heads : 0;
          h[i] = in[i] ? r - t[i] * P.heads : 0;
          if (OP != kBack || !P.act)
            x[i].load(row, (const T*)P.x.p + tok.at[t[i] * 3] + h[i] * P.x.sh);
          if (OP == kBack)
            dy[i].load(row, (const T*)P.dy.p + tok.at[t[i] * 3 + 1] + h[i] * P.dy.sh);
        }
      };
      // the first rows are on their way while the angles are formed
      load(wave * at_once);
      tok.angles<1>(a, first, n, OP != kBack && a.inverse);
      __syncthreads();
      for (uint32_t r0 = wave * at_once; r0 < n * P.heads; r0 += kWaves * at_once * kUnroll) {
        if (r0 != wave * at_once) load(r0);
#pragma unroll
        for (uint32_t i = 0; i < kUnroll; ++i) {
          float c[R::kE], s[R::kE];
          row.turn(tok.turns + t[i] * (a.rotary / 2), c, s);
          if (OP != kBack || !P.act) x[i].sort(row);
          if (OP == kBack) dy[i].sort(row);
          typename R::Data y;
          if constexpr (OP == kBack) {
            float xu[R::kE], xv[R::kE];
            const uint64_t bt = first + t[i], g = bt / ARK_ACT_GROUP;
            const auto kept = [&](uint32_t e, bool second) {
              if (second && !row.has(e, second)) return 0.0f;
              const uint64_t col = g * columns + h[i] * a.head + row.at(e, second);
              return act_value(P.act[col * ARK_ACT_GROUP + bt % ARK_ACT_GROUP], 0, act_up(exps[col]));
            };
#pragma unroll
            for (uint32_t e = 0; e < R::kE; ++e) {
              xu[e] = P.act ? kept(e, false) : x[i].get(e, false);
              xv[e] = P.act ? kept(e, true) : x[i].get(e, true);
            }
            if (!in[i])  // a row that is not there adds nothing to the gain
#pragma unroll
              for (uint32_t e = 0; e < R::kE; ++e) xu[e] = xv[e] = 0.0f;
            if (!in[i]) dy[i] = typename R::Data();
            row.backward(a, a.lanes, in[i], dy[i], xu, xv, gu, gv, c, s, su, sv, &y);
          } else {
            row.template forward<OP>(a, a.lanes, x[i], gu, gv, c, s, &y);
          }
          if (in[i]) y.store(row, (T*)P.y.p + tok.at[t[i] * 3 + 2] + h[i] * P.y.sh);
          if (OP == kBack) __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }
  if constexpr (OP == kBack) {
    float* sum = (float*)lds;
    __syncthreads();
    row.gather(a, a.lanes, su, sv, sum + wave * a.head);
    __syncthreads();
    for (uint32_t j = threadIdx.x; j < a.head; j += kBlock)
      a.partial[((uint64_t)blockIdx.y * gridDim.x + blockIdx.x) * a.head + j] =
          (sum[j] + sum[a.head + j]) + (sum[2 * a.head + j] + sum[3 * a.head + j]);
  }
}

// The exponent bytes of a lane's 2V columns: V bytes at u's place, V at v's.
template <uint32_t V>
struct Exps {
  uint32_t u = 0, v = 0;
  template <typename R>
  __device__ __forceinline__ void load(const R& row, const uint8_t* p) {
    uint32_t a = row.eu[0], b = row.ev[0];
    asm volatile("" : "+v"(a), "+v"(b));
    u = bytes(p + a);
    v = bytes(p + b);
  }
  // in order to every other one and those between
  template <typename R>
  __device__ __forceinline__ void sort(const R& row) {
    if (V > 1 && row.mixed) {
      const uint64_t t = (uint64_t)v << (8 * V) | u;
      u = v = 0;
#pragma unroll
      for (uint32_t i = 0; i < V; ++i) {
        u |= (uint32_t)(t >> (16 * i) & 255u) << (8 * i);
        v |= (uint32_t)(t >> (16 * i + 8) & 255u) << (8 * i);
      }
    }
  }
  template <typename R>
  __device__ __forceinline__ void store(const R& row, uint8_t* p) const {
    uint32_t a = u, b = v;
    if (V > 1 && row.mixed) {
      uint64_t t = 0;
#pragma unroll
      for (uint32_t i = 0; i < V; ++i)
        t |= (uint64_t)(u >> (8 * i) & 255u) << (16 * i) |
             (uint64_t)(v >> (8 * i) & 255u) << (16 * i + 8);
      a = (uint32_t)t;
      b = (uint32_t)(t >> (8 * V));
    }
    if (row.on[0]) put(p + row.eu[0], a);
    if (row.pairs_v[0]) put(p + row.ev[0], b);
  }
  __device__ __forceinline__ uint32_t get(uint32_t i, bool second) const {
    return (second ? v : u) >> (8 * i) & 255u;
  }
  __device__ __forceinline__ void set(uint32_t i, bool second, uint32_t s) {
    (second ? v : u) |= s << (8 * i);
  }

 private:
  typedef uint32_t u32_a1 __attribute__((aligned(1)));
  typedef uint16_t u16_a1 __attribute__((aligned(1)));
  static __device__ __forceinline__ uint32_t bytes(const uint8_t* p) {
    return V == 4 ? *(const ARK_GLOBAL u32_a1*)p : V == 2 ? *(const ARK_GLOBAL u16_a1*)p
                                                          : *(const ARK_GLOBAL uint8_t*)p;
  }
  static __device__ __forceinline__ void put(uint8_t* p, uint32_t x) {
    if (V == 4)
      *(ARK_GLOBAL u32_a1*)p = x;
    else if (V == 2)
      *(ARK_GLOBAL u16_a1*)p = (uint16_t)x;
    else
      *(ARK_GLOBAL uint8_t*)p = (uint8_t)x;
  }
};

// The norm with the 8-bit form of its input, 32 tokens of a head at a time:
// written by the forward pass, read by the backward pass.  A lane holds kIt
// neighbouring tokens of its columns, so that its bytes of a column are
// neighbours.  In the forward pass a wave holds all 32 tokens, and a column's
// largest magnitude is its lanes'; the backward pass has no need of that and
// takes what kIt = 4 leaves of the head.  The next head is loaded while this one
// is worked on.  Writing and reading the 8-bit form in the norm's own pass saves
// a pass over x each way.
//
// 16384 tokens of 12 + 12 heads of 64, fp16, 127 MB each way: forward 35.5 us,
// backward 34.7, 3.6 TB/s; 32768 of 16 + 16 of 128, bf16, 678 MB: 152 and 180 us,
// 4.5 and 3.8 TB/s.  Neither more waves nor fewer change the forward pass, nor do
// fewer vector instructions: memory's share (23 us of the first at a copy's rate)
// and the vector units' (17) overlap only in part.
//
// Waves of a SIMD the registers are cut for, by the words a head's share takes of a
// lane twice over: the most without spills (but for 28 bytes at V = 1 forward, of 16-bit types).
// Backward at four waves instead of three spills 88 bytes and takes 50 us for 38
// (237M training pass).
constexpr int tile_waves(bool back, uint32_t words) {
  return back ? (words <= 16 ? 3 : 2) : words <= 16 ? 4 : words <= 32 ? 3 : words <= 64 ? 2 : 1;
}
template <uint32_t DT, bool BACK, uint32_t V, uint32_t kIt, uint32_t kLanes>
__global__ __launch_bounds__(kBlock, tile_waves(BACK, V * kIt * (DT == ARK_ACT_F32 ? 2 : 1)))
void tiles_kernel(Args a) {
  typedef Row<DT, V, 1> R;
  typedef elem_t<DT> T;
  constexpr uint32_t kTokens = 64 / kLanes * kIt;           // a wave's of a head
  constexpr uint32_t kSubs = ARK_ACT_GROUP / kTokens;       // waves' shares of a group
  static_assert(BACK || kSubs == 1, "the forward pass needs whole columns");
  typedef uint32_t Bytes __attribute__((ext_vector_type(kIt / 4), aligned(4)));
  extern __shared__ __align__(16) uint8_t lds[];
  const Tokens tok(a, lds);
  const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  R row(a, lane % kLanes);
  const uint64_t groups = (a.all + ARK_ACT_GROUP - 1) / ARK_ACT_GROUP;
  const Part& P = a.part[blockIdx.y];
  const uint64_t columns = (uint64_t)P.heads * a.head;
  float su[R::kE] = {}, sv[R::kE] = {}, gu[R::kE], gv[R::kE];
  row.gains(a, P.gain, gu, gv);
  const uint32_t units = P.heads * kSubs, slice = blockIdx.x % a.slices;
  const uint32_t first_unit = slice * kWaves + wave, stride = a.slices * kWaves;
  for (uint64_t g = blockIdx.x / a.slices; g < groups; g += gridDim.x / a.slices) {
    const uint64_t first = g * ARK_ACT_GROUP;
    const uint32_t n = (uint32_t)(a.all - first < ARK_ACT_GROUP ? a.all - first : ARK_ACT_GROUP);
    uint8_t* const values = P.act + g * columns * ARK_ACT_GROUP;
    uint8_t* const exps = P.act + groups * columns * ARK_ACT_GROUP + g * columns;
    // a unit as it is loaded
    struct Held {
      typename R::Data in[kIt];
      Bytes b[R::kE][2];
      Exps<V> e;
    };
    const auto mine_of = [&](uint32_t unit) {
      return unit % kSubs * kTokens + lane / kLanes * kIt;
    };
    const auto load = [&](uint32_t unit, Held* held) {
      const Array& from = BACK ? P.dy : P.x;
      const uint32_t h = unit / kSubs, mine = mine_of(unit);
      row.forget();
#pragma unroll
      for (uint32_t i = 0; i < kIt; ++i) {
        uint32_t t = min(mine + i, n - 1);
        asm volatile("" : "+v"(t));
        held->in[i].load(row, (const T*)from.p + tok.at[t * 3 + BACK] + h * from.sh);
      }
      if constexpr (BACK) {
        held->e.load(row, exps + h * a.head);
#pragma unroll
        for (uint32_t k = 0; k < 2 * R::kE; ++k) {
          const bool second = k & 1;
          uint32_t c = V == 1 && second && !row.pairs_v[0] ? row.eu[0] : row.at(k / 2, second);
          c = c * ARK_ACT_GROUP + mine;
          asm volatile("" : "+v"(c));  // an offset from a scalar base, not an address kept
          held->b[k / 2][second] =
              *(const ARK_GLOBAL Bytes*)(values + (uint64_t)h * a.head * ARK_ACT_GROUP + c);
        }
      }
    };
    Held now, next;
    __syncthreads();
    tok.starts(a, P, first, n);
    __syncthreads();
    // the first head is on its way while the angles are formed
    if (first_unit < units) load(first_unit, &now);
    tok.angles<2>(a, first, n, false);
    __syncthreads();
    for (uint32_t unit = first_unit; unit < units; unit += stride) {
      if (unit + stride < units) load(unit + stride, &next);
      const uint32_t h = unit / kSubs, mine = mine_of(unit);
      row.forget();
      if (n < ARK_ACT_GROUP)  // tokens past the last: zeros in the 8-bit form and the sums
#pragma unroll
        for (uint32_t i = 0; i < kIt; ++i)
          if (mine + i >= n) now.in[i] = typename R::Data();
      if (row.mixed)
#pragma unroll
        for (uint32_t i = 0; i < kIt; ++i) now.in[i].sort(row);
      float up[R::kE][2];
      if constexpr (BACK) {
        now.e.sort(row);
#pragma unroll
        for (uint32_t k = 0; k < R::kE; ++k) {
          up[k][0] = act_up(now.e.get(k, false));
          up[k][1] = V == 1 && !row.pairs_v[0] ? 0.0f : act_up(now.e.get(k, true));
        }
      } else {
        Exps<V> e;
        // the largest magnitudes of a lane's columns, as the types' bits order them
        typename R::Data most = typename R::Data();
#pragma unroll
        for (uint32_t i = 0; i < kIt; ++i) most.larger(now.in[i]);
        if (kLanes <= 8) most.template larger_across<8>();
        if (kLanes <= 16) most.template larger_across<16>();
        if (kLanes <= 32) most.template larger_across<32>();
        bool at_top = false;
#pragma unroll
        for (uint32_t k = 0; k < 2 * R::kE; ++k) {
          const uint32_t s = act_exponent<DT>(__float_as_uint(most.get(k / 2, k & 1)));
          e.set(k / 2, k & 1, s);
          at_top |= s >= kActTop<DT>;
        }
        const auto quantise = [&](auto hold) {
#pragma unroll
          for (uint32_t k = 0; k < 2 * R::kE; ++k) {
            const uint32_t p = k / 2;
            const bool second = k & 1;
            const auto at = [&](uint32_t i) {
              const float f = now.in[i].get(p, second);
              return decltype(hold)::value ? act_hold<DT>(e.get(p, second), f) : f;
            };
            Bytes w;
#pragma unroll
            for (uint32_t i = 0; i < kIt; i += 4)
              w[i / 4] = act_bytes4(e.get(p, second), at(i), at(i + 1), at(i + 2), at(i + 3));
            uint32_t c = row.at(p, second) * ARK_ACT_GROUP + mine;
            asm volatile("" : "+v"(c));  // an offset from a scalar base, not an address kept
            if (V > 1 ? row.on[0] : row.has(p, second))
              *(ARK_GLOBAL Bytes*)(values + (uint64_t)h * a.head * ARK_ACT_GROUP + c) = w;
          }
        };
        if (__builtin_amdgcn_ballot_w64(at_top))
          quantise(std::true_type());
        else
          quantise(std::false_type());
        if (mine == 0) e.store(row, exps + h * a.head);
      }
#pragma unroll
      for (uint32_t i = 0; i < kIt; ++i) {
        uint32_t t = mine + i;
        // read from LDS for every head again: kept in registers over all heads the
        // lines would cost most of them
        asm volatile("" : "+v"(t));
        float c[R::kE], s[R::kE];
        row.turn(tok.turns + min(t, n - 1) * (a.rotary / 2), c, s);
        typename R::Data y;
        now.in[i].opaque();  // widened here, not with all the others
        if constexpr (BACK) {
          float xu[R::kE], xv[R::kE];
#pragma unroll
          for (uint32_t e = 0; e < R::kE; ++e) {
            asm volatile("" : "+v"(now.b[e][0][i / 4]), "+v"(now.b[e][1][i / 4]));
            xu[e] = act_value(now.b[e][0][i / 4], i % 4, up[e][0]);
            xv[e] = act_value(now.b[e][1][i / 4], i % 4, up[e][1]);
          }
          row.backward(a, kLanes, t < n, now.in[i], xu, xv, gu, gv, c, s, su, sv, &y);
        } else {
          row.template forward<kNorm>(a, kLanes, now.in[i], gu, gv, c, s, &y);
        }
        if (t < n) y.store(row, (T*)P.y.p + tok.at[t * 3 + 2] + h * P.y.sh);
        __builtin_amdgcn_sched_barrier(0);  // one row at a time: registers for more waves
      }
      now = next;
    }
  }
  if constexpr (BACK) {
    float* sum = (float*)lds;
    __syncthreads();
    row.gather(a, kLanes, su, sv, sum + wave * a.head);
    __syncthreads();
    for (uint32_t j = threadIdx.x; j < a.head; j += kBlock)
      a.partial[((uint64_t)blockIdx.y * gridDim.x + blockIdx.x) * a.head + j] =
          (sum[j] + sum[a.head + j]) + (sum[2 * a.head + j] + sum[3 * a.head + j]);
  }
}

// The 8-bit form of a part's input where tiles_kernel does not write it (one part's
// alone, or heads of which a wave cannot hold 32 tokens): a lane a column of a
// group, heads and batches wherever their strides put them.  A second pass over x.
template <uint32_t DT>
__global__ __launch_bounds__(kBlock) void keep_kernel(Args a) {
  const Part& P = a.part[blockIdx.z];
  if (!P.act) return;
  const uint64_t columns = (uint64_t)P.heads * a.head, n = a.all;
  const uint64_t groups = (n + ARK_ACT_GROUP - 1) / ARK_ACT_GROUP;
  const uint64_t i = (uint64_t)blockIdx.x * kBlock + threadIdx.x;
  if (i >= groups * columns) return;
  const uint64_t g = i / columns, col = i % columns;
  const elem_t<DT>* x = (const elem_t<DT>*)P.x.p + col / a.head * P.x.sh + col % a.head;
  float v[ARK_ACT_GROUP];
  uint32_t most = 0;
#pragma unroll
  for (uint32_t r = 0; r < ARK_ACT_GROUP; ++r) {
    const uint64_t bt = g * ARK_ACT_GROUP + r;
    v[r] = bt < n ? (float)x[bt / a.tokens * P.x.sb + bt % a.tokens * P.x.st] : 0.0f;
    const uint32_t m = __float_as_uint(v[r]) & 0x7FFFFFFFu;
    most = m > most ? m : most;
  }
  const uint32_t s = act_exponent<DT>(most);
#pragma unroll
  for (uint32_t r = 0; r < ARK_ACT_GROUP; r += 4)
    st_g<uint32_t>(P.act + i * ARK_ACT_GROUP + r,
                   act_bytes4(s, act_hold<DT>(s, v[r]), act_hold<DT>(s, v[r + 1]), act_hold<DT>(s, v[r + 2]),
                              act_hold<DT>(s, v[r + 3])));
  P.act[groups * columns * ARK_ACT_GROUP + i] = (uint8_t)s;
}

// The gains' gradients from the blocks' rows (none of a part of no heads), added in
// order: 64 rows' runs by the lanes of a column, then those.  4 us of latency for
// any number of rows met here (about 768 in all of tiles, up to 1024 a part of
// rows).
constexpr uint32_t kGainColumns = 16, kGainRuns = 64;
__global__ __launch_bounds__(kGainColumns * kGainRuns) void gain_kernel(
    const float* __restrict__ partial, uint32_t rows_q, uint32_t rows_k, uint32_t head,
    float* __restrict__ dq, float* __restrict__ dk, uint32_t accumulate) {
  __shared__ float sum[kGainRuns][kGainColumns];
  const uint32_t c = threadIdx.x % kGainColumns, run = threadIdx.x / kGainColumns;
  const uint32_t j = blockIdx.x * kGainColumns + c;
  const float* p = partial + (blockIdx.y ? (uint64_t)rows_q * head : 0) + j;
  const uint32_t rows = blockIdx.y ? rows_k : rows_q;
  float s = 0.0f;
  if (j < head)
#pragma unroll 8
    for (uint32_t i = run; i < rows; i += kGainRuns) s += p[(uint64_t)i * head];
  sum[run][c] = s;
  __syncthreads();
  for (uint32_t half = kGainRuns / 2; half; half /= 2) {
    if (run < half) sum[run][c] += sum[run + half][c];
    __syncthreads();
  }
  float* out = blockIdx.y ? dk : dq;
  if (run == 0 && j < head && out) out[j] = accumulate ? out[j] + sum[0][c] : sum[0][c];
}

// How a row goes over lanes: V pairs a lane where the head and its rotary part
// are whole chunks of 2V, and the wave's lanes for a row, at least eight.
struct Shape2 {
  uint32_t v, k, lanes;
};
Shape2 row_shape(uint32_t head, uint32_t rotary) {
  const uint32_t both = head | rotary;
  const uint32_t v = both % 8 == 0 ? 4 : both % 4 == 0 && head <= 256 ? 2 : 1;
  const uint32_t need = ((head + 1) / 2 + v - 1) / v;
  uint32_t lanes = v == 4 ? 8 : v == 2 ? 32 : 64;
  while (lanes < need && lanes < 64) lanes *= 2;
  return {v, need > 64 ? 4u : 1u, lanes};
}

template <uint32_t DT, Op OP>
void rows_of(const Shape2& w, dim3 grid, uint32_t lds, hipStream_t s, const Args& a) {
  if (w.v == 4)
    hipLaunchKernelGGL((rows_kernel<DT, OP, 4, 1>), grid, dim3(kBlock), lds, s, a);
  else if (w.v == 2)
    hipLaunchKernelGGL((rows_kernel<DT, OP, 2, 1>), grid, dim3(kBlock), lds, s, a);
  else if (w.k == 1)
    hipLaunchKernelGGL((rows_kernel<DT, OP, 1, 1>), grid, dim3(kBlock), lds, s, a);
  else
    hipLaunchKernelGGL((rows_kernel<DT, OP, 1, 4>), grid, dim3(kBlock), lds, s, a);
}
template <uint32_t DT, bool BACK>
void tiles_of(const Shape2& w, dim3 grid, uint32_t lds, hipStream_t s, const Args& a) {
#define ARK_TILES(V, L)                                                                      \
  if (w.v == V && w.lanes == L)                                                              \
    hipLaunchKernelGGL((tiles_kernel<DT, BACK, V, BACK ? 4 : L / 2, L>), grid, dim3(kBlock), lds, s, a);
  ARK_TILES(4, 8)
  ARK_TILES(4, 16)
  ARK_TILES(4, 32)
  ARK_TILES(2, 32)
  ARK_TILES(2, 64)
  ARK_TILES(1, 64)
  if constexpr (BACK) {
    ARK_TILES(4, 64)
  }
#undef ARK_TILES
}

// A block's LDS for `tile` tokens, and for the sums of the gain's gradient.
uint32_t block_lds(const Args& a, uint32_t tile) {
  const uint32_t t = tile * (24 + a.rotary / 2 * 8), sum = kWaves * a.head * 4;
  return t > sum ? t : sum;
}
// Tokens a block of rows_kernel takes: a thousand blocks before tokens share one,
// then as many as `turns` times what its waves take at once, and no more than keep
// its lines small enough for eight blocks a unit.  More blocks that end sooner
// keep reads and writes of different blocks side by side (32768 tokens of 16 + 16
// heads of 128, bf16: rotated by four turns 99 us, by fifteen 120), but the norms'
// gains and sums are set up once a block (8192 of 64 + 8 of 64: 40 us by four
// turns, 37 by eight).
uint32_t rows_tile(const Args& a, const Shape2& w, uint32_t turns) {
  uint32_t most = 16384 / (24 + a.rotary / 2 * 8);
  if (most > 32) most = 32;
  const uint32_t heads = a.part[0].heads > a.part[1].heads ? a.part[0].heads : a.part[1].heads;
  const uint32_t rows = 64 / w.lanes * kWaves * (w.v == 4 ? 2 : 1) * turns;
  const uint32_t fill = rows <= heads ? 1 : rows / (heads ? heads : 1);
  const uint64_t want = (a.all + 1023) / 1024;
  if (most > fill) most = fill;
  return want < 1 ? 1 : want < most ? (uint32_t)want : most;
}

template <Op OP>
uint32_t launch_rows(uint32_t dtype, Args* a, hipStream_t s, bool launch = true) {
  const Shape2 w = row_shape(a->head, a->rotary);
  a->lanes = w.lanes;
  a->tile = rows_tile(*a, w, OP == kRope ? 4 : 8);
  const uint64_t tiles = (a->all + a->tile - 1) / a->tile;
  // Backward, the units' fill of a part's blocks, fewer for long heads: up to 128
  // values the rows of both gains' gradients then fit a kept slot of 512 KiB.
  // Longer heads keep 512 blocks a part and take the stream's pool, whose host
  // time is 33 us.
  const uint32_t rows = 65536 / a->head;
  const uint32_t most = OP != kBack ? 1u << 20 : rows < 512 ? 512 : rows < 1024 ? rows : 1024;
  const uint32_t blocks = (uint32_t)(tiles < most ? tiles : most);
  if (!launch || !blocks) return blocks;
  const dim3 grid(blocks, a->part[1].heads ? 2 : 1);
  if (dtype == ARK_ACT_F16)
    rows_of<ARK_ACT_F16, OP>(w, grid, block_lds(*a, a->tile), s, *a);
  else if (dtype == ARK_ACT_BF16)
    rows_of<ARK_ACT_BF16, OP>(w, grid, block_lds(*a, a->tile), s, *a);
  else
    rows_of<ARK_ACT_F32, OP>(w, grid, block_lds(*a, a->tile), s, *a);
  return blocks;
}

// Whether a wave can hold 32 tokens of a head, at most 128 values a lane, or for
// the backward pass four tokens a lane.
bool tiles_fit(const Args& a, bool back) {
  const Shape2 w = row_shape(a.head, a.rotary);
  return w.k == 1 && (back || w.v * w.lanes <= 128);
}

template <bool BACK>
uint32_t launch_tiles(uint32_t dtype, Args* a, hipStream_t s, bool launch = true) {
  const Shape2 w = row_shape(a->head, a->rotary);
  a->lanes = w.lanes;
  a->tile = ARK_ACT_GROUP;
  const uint64_t groups = ark::act_groups(a->all);
  const uint32_t heads = a->part[0].heads > a->part[1].heads ? a->part[0].heads : a->part[1].heads;
  // blocks share a group's heads until there are about 500 of a part: each of them
  // forms the group's angles again (237M training pass 78.7 us with one block a
  // group, 94.4 with two)
  const uint32_t units = BACK ? heads * (w.lanes / 8) : heads;  // of a group
  uint32_t slices = (units + kWaves - 1) / kWaves;
  while (slices > 1 && groups * (slices - 1) >= 512) --slices;
  a->slices = slices;
  uint64_t by = groups;
  // Backward, as many blocks as the units hold at once, three each: every block's
  // row of the gains' gradients is one more to add up, and a last round of a few
  // blocks would have the chip to itself (237M training pass 34.7 us, 37.6 with a
  // block a group).  Their rows fit a kept slot up to heads of 170 values.
  const uint32_t parts = a->part[1].heads ? 2 : 1;
  const uint32_t held = 768 / parts / slices, most = !BACK ? 1u << 20 : held ? held : 1;
  if (by > most) by = most;
  const uint32_t blocks = (uint32_t)by * slices;
  if (!launch || !blocks) return blocks;
  const dim3 grid(blocks, a->part[1].heads ? 2 : 1);
  if (dtype == ARK_ACT_F16)
    tiles_of<ARK_ACT_F16, BACK>(w, grid, block_lds(*a, a->tile), s, *a);
  else if (dtype == ARK_ACT_BF16)
    tiles_of<ARK_ACT_BF16, BACK>(w, grid, block_lds(*a, a->tile), s, *a);
  else
    tiles_of<ARK_ACT_F32, BACK>(w, grid, block_lds(*a, a->tile), s, *a);
  return blocks;
}

}  // namespace

struct ark_rope {
  int device = 0;
  uint32_t head = 0, rotary = 0, layout = 0;
  float magnitude = 1.0f;
  uint64_t* turns = nullptr;  // on the device
};

namespace {

// An array of a call as its entry point describes it.
struct Given {
  const char* what;
  const void* p;
  const uint64_t* layout;  // heads, batch, token, head strides
  bool written;
  uint64_t bytes;          // from p to its last element's end
};

// The sizes every array of a call shares.
struct Shape {
  uint64_t batch, tokens, head;
  uint32_t es;
};

constexpr uint64_t kMaxExtent = 1ull << 46;  // elements between an array's ends

int check_given(Given* g, const Shape& s, uint64_t heads) {
  if (!g->layout) return ark::fail(ARK_OPT_EINVAL, "%s's layout is NULL", g->what);
  if (g->layout[0] != heads)
    return ark::fail(ARK_OPT_EINVAL, "%s has %llu heads, not %llu", g->what,
                     (unsigned long long)g->layout[0], (unsigned long long)heads);
  if ((uintptr_t)g->p % s.es)
    return ark::fail(ARK_OPT_EINVAL, "%s not aligned to its element", g->what);
  const uint64_t n[3] = {s.batch, s.tokens, heads};
  uint64_t last = s.head - 1;
  for (int i = 0; i < 3; ++i) {
    const uint64_t st = g->layout[i + 1];
    if (n[i] > 1 && st > kMaxExtent / (n[i] - 1))
      return ark::fail(ARK_OPT_EINVAL, "%s: stride %llu too large", g->what,
                       (unsigned long long)st);
    if (n[i] > 1) last += (n[i] - 1) * st;
  }
  g->bytes = (last + 1) * s.es;
  if (!g->written) return ARK_OPT_OK;
  // the dimensions by stride: each must step past everything inside it
  int order[3] = {0, 1, 2};
  for (int i = 0; i < 3; ++i)
    for (int j = i + 1; j < 3; ++j)
      if (g->layout[order[j] + 1] < g->layout[order[i] + 1]) {
        const int t = order[i];
        order[i] = order[j];
        order[j] = t;
      }
  uint64_t inside = s.head;
  for (int i : order) {
    if (n[i] <= 1) continue;
    if (g->layout[i + 1] < inside)
      return ark::fail(ARK_OPT_EINVAL, "%s: its rows overlap each other", g->what);
    inside += (n[i] - 1) * g->layout[i + 1];
  }
  return ARK_OPT_OK;
}

// True when two arrays of a call cannot share a byte: their ends are apart, or
// they step alike over batches (or over batches and tokens) and what lies
// inside one step of both never meets, as in views of one fused array.
bool apart(const Given& a, const Given& b, const Shape& s) {
  if (a.bytes == 0 || b.bytes == 0) return true;
  if (!ark::overlaps(a.p, a.bytes, b.p, b.bytes)) return true;
  const uint64_t n[2] = {s.batch, s.tokens};
  const uint64_t ha = (a.layout[0] - 1) * a.layout[3] + s.head;
  const uint64_t hb = (b.layout[0] - 1) * b.layout[3] + s.head;
  const int64_t off = (int64_t)((intptr_t)b.p - (intptr_t)a.p) / (int64_t)s.es;
  for (int level = 0; level < 2; ++level) {
    // the footprints inside dimension `level`, and its step
    uint64_t fa = ha, fb = hb;
    const uint64_t step = a.layout[level + 1];
    if (level == 0) {
      if (n[0] <= 1) continue;
      fa += (n[1] - 1) * a.layout[2];
      fb += (n[1] - 1) * b.layout[2];
    } else {
      if (n[1] <= 1) continue;
      if (n[0] > 1 && (a.layout[1] != b.layout[1] || a.layout[1] % (step ? step : 1))) continue;
    }
    if (step == 0 || step != b.layout[level + 1] || fa > step || fb > step) continue;
    const uint64_t r = (uint64_t)(((off % (int64_t)step) + (int64_t)step) % (int64_t)step);
    if (r >= fa && r + fb <= step) return true;
  }
  return false;
}

// In place: the same array with the same steps.
bool same(const Given& a, const Given& b, const Shape& s) {
  if (a.p != b.p) return false;
  const uint64_t n[3] = {s.batch, s.tokens, a.layout[0]};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && a.layout[i + 1] != b.layout[i + 1]) return false;
  return a.layout[0] == b.layout[0];
}

// What every entry point checks first; *empty: no rows.
int check_call(const ark_rope* r, uint32_t dtype, uint64_t batch, uint64_t tokens,
               const void* positions, uint32_t position_bytes, bool* empty) {
  *empty = batch == 0 || tokens == 0;
  if (!r) return ark::fail(ARK_OPT_EINVAL, "rope is NULL");
  if (dtype > ARK_ACT_F32) return ark::fail(ARK_OPT_EINVAL, "dtype %u unknown", dtype);
  if (batch >= (1ull << 40) || tokens >= (1ull << 40) ||
      (tokens && batch > (1ull << 40) / tokens))
    return ark::fail(ARK_OPT_EINVAL, "batch * tokens too large");
  if (positions && position_bytes != 4 && position_bytes != 8)
    return ark::fail(ARK_OPT_EINVAL, "position_bytes %u: positions are int32 or int64",
                     position_bytes);
  if (positions && (uintptr_t)positions % position_bytes)
    return ark::fail(ARK_OPT_EINVAL, "positions not aligned to their element");
  return ARK_OPT_OK;
}

int check_heads(const uint64_t* layout, const char* what, uint32_t* heads) {
  if (!layout) return ark::fail(ARK_OPT_EINVAL, "%s's layout is NULL", what);
  if (layout[0] > (1u << 20))
    return ark::fail(ARK_OPT_EINVAL, "%s has %llu heads", what, (unsigned long long)layout[0]);
  *heads = (uint32_t)layout[0];
  return ARK_OPT_OK;
}

Array array_of(const Given& g) {
  return {g.p, g.layout[1], g.layout[2], g.layout[3]};
}

// Pairwise checks of a call's arrays: each written one against every other,
// except its own input (`pair`) where it is that in place.  acts: 8-bit forms
// and other flat ranges, written or not.
struct Flat {
  const char* what;
  const void* p;
  uint64_t bytes;
  bool written;
};

int check_apart(const Given* g, int n, const int* in_place_of, const Flat* f, int nf,
                const Shape& s) {
  for (int i = 0; i < n; ++i) {
    if (g[i].bytes == 0) continue;  // not part of this call: no layout either
    for (int j = 0; j < n; ++j) {
      if (i == j || g[j].bytes == 0 || !g[i].written || (g[j].written && j < i)) continue;
      if (in_place_of[i] == j && same(g[i], g[j], s)) continue;
      if (!apart(g[i], g[j], s))
        return ark::fail(ARK_OPT_EINVAL, "%s overlaps %s (written by the call)", g[j].what,
                         g[i].what);
    }
    for (int j = 0; j < nf; ++j)
      if ((g[i].written || f[j].written) && f[j].bytes &&
          ark::overlaps(g[i].p, g[i].bytes, f[j].p, f[j].bytes))
        return ark::fail(ARK_OPT_EINVAL, "%s overlaps %s", f[j].what, g[i].what);
  }
  for (int i = 0; i < nf; ++i)
    for (int j = i + 1; j < nf; ++j)
      if ((f[i].written || f[j].written) && f[i].bytes && f[j].bytes &&
          ark::overlaps(f[i].p, f[i].bytes, f[j].p, f[j].bytes))
        return ark::fail(ARK_OPT_EINVAL, "%s overlaps %s", f[j].what, f[i].what);
  return ARK_OPT_OK;
}

int check_memory(const Given* g, int n, const Flat* f, int nf) {
  ark::BufferChecker checker;
  const void* wp[8];
  uint64_t wb[8];
  size_t w = 0;
  int rc;
  for (int i = 0; i < n; ++i) {
    if ((rc = checker.check(g[i].p, g[i].bytes, g[i].what, 0))) return rc;
    if (g[i].written) wp[w] = g[i].p, wb[w++] = g[i].bytes;
  }
  for (int i = 0; i < nf; ++i) {
    if ((rc = checker.check(f[i].p, f[i].bytes, f[i].what, 0))) return rc;
    if (f[i].written) wp[w] = f[i].p, wb[w++] = f[i].bytes;
  }
  ark::opt_units_invalidate(wp, wb, w);
  return ARK_OPT_OK;
}

Args base_args(const ark_rope* r, uint64_t batch, uint64_t tokens, const void* positions,
               uint32_t position_bytes, uint64_t start) {
  Args a = {};
  a.turns = r->turns;
  a.positions = positions;
  a.position_bytes = position_bytes;
  a.start = start;
  a.tokens = tokens;
  a.all = batch * tokens;
  a.magnitude = r->magnitude;
  a.head = r->head;
  a.one_over_head = 1.0f / (float)r->head;
  a.rotary = r->rotary;
  a.layout = r->layout;
  return a;
}

uint64_t act_size(uint64_t rows, uint64_t columns) { return 33 * ark::act_groups(rows) * columns; }

}  // namespace

extern "C" {

int ark_rope_frequencies(uint32_t rotary_dim, double base, uint32_t scaling, const double* params,
                         double* inv_freq, double* magnitude) {
  if (!inv_freq || !magnitude) return ark::fail(ARK_OPT_EINVAL, "inv_freq or magnitude is NULL");
  if (rotary_dim % 2 || rotary_dim > ARK_ROPE_MAX_HEAD)
    return ark::fail(ARK_OPT_EINVAL, "rotary_dim %u: even and at most %d are taken", rotary_dim,
                     ARK_ROPE_MAX_HEAD);
  if (!(base > 0.0) || !isfinite(base))
    return ark::fail(ARK_OPT_EINVAL, "base = %g is not a positive number", base);
  static const int kParams[] = {0, 1, 1, 4, 4};
  if (scaling > ARK_ROPE_SCALE_BANDS) return ark::fail(ARK_OPT_EINVAL, "scaling %u unknown", scaling);
  if (kParams[scaling] && !params) return ark::fail(ARK_OPT_EINVAL, "params is NULL");
  for (int i = 0; i < kParams[scaling]; ++i)
    if (!(params[i] > 0.0) || !isfinite(params[i]))
      return ark::fail(ARK_OPT_EINVAL, "scaling parameter %d = %g is not a positive number", i,
                       params[i]);
  const double pi2 = 6.283185307179586476925;
  const double R = rotary_dim, f = scaling ? params[0] : 1.0;
  if (scaling == ARK_ROPE_SCALE_YARN && (base == 1.0 || params[2] < params[3]))
    return ark::fail(ARK_OPT_EINVAL, "yarn needs a base other than 1 and fast >= slow turns");
  if (scaling == ARK_ROPE_SCALE_BANDS && !(params[2] < params[3]))
    return ark::fail(ARK_OPT_EINVAL, "bands need low < high turns");
  double b = base, lo = 0.0, hi = 0.0;
  *magnitude = 1.0;
  if (scaling == ARK_ROPE_SCALE_NTK && rotary_dim > 2) b = base * pow(f, R / (R - 2.0));
  if (scaling == ARK_ROPE_SCALE_YARN) {
    lo = floor(R * log(params[1] / (pi2 * params[2])) / (2.0 * log(base)));
    hi = ceil(R * log(params[1] / (pi2 * params[3])) / (2.0 * log(base)));
    lo = lo < 0.0 ? 0.0 : lo;
    hi = hi > R - 1.0 ? R - 1.0 : hi;
    *magnitude = f > 1.0 ? 0.1 * log(f) + 1.0 : 1.0;
  }
  for (uint32_t i = 0; i < rotary_dim / 2; ++i) {
    const double w = pow(b, -2.0 * i / R);
    double v = w;
    if (scaling == ARK_ROPE_SCALE_LINEAR) v = w / f;
    if (scaling == ARK_ROPE_SCALE_YARN) {
      const double span = hi - lo > 0.001 ? hi - lo : 0.001;
      const double x = (i - lo) / span, slow = x < 0.0 ? 0.0 : x > 1.0 ? 1.0 : x;
      v = w * (1.0 - slow) + w / f * slow;
    }
    if (scaling == ARK_ROPE_SCALE_BANDS) {
      const double n = params[1] * w / pi2, x = (n - params[2]) / (params[3] - params[2]);
      const double keep = x < 0.0 ? 0.0 : x > 1.0 ? 1.0 : x;
      v = w / f * (1.0 - keep) + w * keep;
    }
    inv_freq[i] = v;
  }
  return ARK_OPT_OK;
}

int ark_rope_create(uint32_t head_dim, uint32_t rotary_dim, uint32_t layout,
                    const double* inv_freq, double magnitude, ark_rope** out) {
  if (!out) return ark::fail(ARK_OPT_EINVAL, "out is NULL");
  *out = nullptr;
  if (head_dim == 0 || head_dim > ARK_ROPE_MAX_HEAD)
    return ark::fail(ARK_OPT_EINVAL, "head_dim %u: 1 to %d are taken", head_dim,
                     ARK_ROPE_MAX_HEAD);
  if (rotary_dim % 2 || rotary_dim > head_dim)
    return ark::fail(ARK_OPT_EINVAL, "rotary_dim %u: even and at most head_dim %u are taken",
                     rotary_dim, head_dim);
  if (layout > ARK_ROPE_INTERLEAVED) return ark::fail(ARK_OPT_EINVAL, "layout %u unknown", layout);
  if (rotary_dim && !inv_freq) return ark::fail(ARK_OPT_EINVAL, "inv_freq is NULL");
  if (!isfinite(magnitude) || fabs(magnitude) > 3.0e38)
    return ark::fail(ARK_OPT_EINVAL, "magnitude is not finite");
  // 2^64 turns a position, by whole turns' remainder; long double keeps every
  // bit of the double it is given
  std::vector<uint64_t> turns(rotary_dim / 2);
  for (uint32_t i = 0; i < rotary_dim / 2; ++i) {
    if (!isfinite(inv_freq[i]) || fabs(inv_freq[i]) > 1e9)
      return ark::fail(ARK_OPT_EINVAL, "inv_freq[%u] = %g", i, inv_freq[i]);
    long double t = (long double)inv_freq[i] / 6.283185307179586476925286766559L;
    t -= floorl(t);
    const long double scaled = t * 18446744073709551616.0L + 0.5L;
    turns[i] = scaled >= 18446744073709551616.0L ? 0 : (uint64_t)scaled;
  }
  ark_rope* r = new (std::nothrow) ark_rope();
  if (!r) return ark::fail(ARK_OPT_ENOMEM, "no memory for a rope");
  r->head = head_dim;
  r->rotary = rotary_dim;
  r->layout = layout;
  r->magnitude = (float)magnitude;
  int rc = ark::current_device_for(nullptr, &r->device);
  if (rc) {
    delete r;
    return rc;
  }
  if (!turns.empty()) {
    hipError_t e = hipMalloc(&r->turns, turns.size() * sizeof(uint64_t));
    if (e == hipSuccess)
      e = hipMemcpy(r->turns, turns.data(), turns.size() * sizeof(uint64_t),
                    hipMemcpyHostToDevice);
    if (e != hipSuccess) {
      if (r->turns) (void)hipFree(r->turns);
      delete r;
      return ark::hip_fail(e, "ark_rope_create");
    }
  }
  *out = r;
  return ARK_OPT_OK;
}

int ark_rope_destroy(ark_rope* r) {
  if (!r) return ARK_OPT_OK;
  int rc = ARK_OPT_OK;
  if (r->turns) {
    ark::DeviceGuard g(r->device);
    hipError_t e = hipFree(r->turns);
    if (e != hipSuccess) rc = ark::hip_fail(e, "hipFree");
  }
  delete r;
  return rc;
}

int ark_rope_apply(const ark_rope* r, uint32_t dtype, uint64_t batch, uint64_t tokens,
                   const void* positions, uint32_t position_bytes, uint64_t start, const void* q,
                   const uint64_t* q_layout, void* q_out, const uint64_t* q_out_layout,
                   const void* k, const uint64_t* k_layout, void* k_out,
                   const uint64_t* k_out_layout, uint32_t inverse, void* stream) {
  int rc;
  bool empty;
  if ((rc = check_call(r, dtype, batch, tokens, positions, position_bytes, &empty))) return rc;
  uint32_t heads[2] = {};
  if ((rc = check_heads(q_layout, "q", &heads[0]))) return rc;
  if (k_layout && (rc = check_heads(k_layout, "k", &heads[1]))) return rc;
  if (empty || heads[0] + heads[1] == 0) return ARK_OPT_OK;
  const Shape s = {batch, tokens, r->head, ark::act_elem_size(dtype)};
  Given g[4] = {{"q_out", q_out, q_out_layout, true, 0}, {"q", q, q_layout, false, 0},
                {"k_out", k_out, k_out_layout, true, 0}, {"k", k, k_layout, false, 0}};
  static const int in_place[4] = {1, -1, 3, -1};
  for (int i = 0; i < 4; ++i)
    if (heads[i / 2] && (rc = check_given(&g[i], s, heads[i / 2]))) return rc;
  const Flat f[1] = {{"positions", positions, positions ? batch * tokens * position_bytes : 0,
                      false}};
  if ((rc = check_apart(g, 4, in_place, f, 1, s)) || (rc = check_memory(g, 4, f, 1))) return rc;
  Args a = base_args(r, batch, tokens, positions, position_bytes, start);
  a.inverse = inverse != 0;
  Part* part = a.part;
  for (int i = 0; i < 2; ++i) {
    if (!heads[i]) continue;
    part->x = array_of(g[2 * i + 1]);
    part->y = array_of(g[2 * i]);
    part->heads = heads[i];
    ++part;
  }
  ark::DeviceGuard guard(r->device);
  if (!guard.ok) return ark::fail(ARK_OPT_EHIP, "cannot select device %d", r->device);
  launch_rows<kRope>(dtype, &a, (hipStream_t)stream);
  ARK_HIP(hipGetLastError());
  return ARK_OPT_OK;
}

int ark_rope_norm(const ark_rope* r, uint32_t dtype, uint64_t batch, uint64_t tokens,
                  const void* positions, uint32_t position_bytes, uint64_t start, float eps,
                  const void* gain_q, const void* gain_k, uint32_t gain_dtype, const void* q,
                  const uint64_t* q_layout, void* q_out, const uint64_t* q_out_layout,
                  void* q_act, const void* k, const uint64_t* k_layout, void* k_out,
                  const uint64_t* k_out_layout, void* k_act, void* stream) {
  int rc;
  bool empty;
  if ((rc = check_call(r, dtype, batch, tokens, positions, position_bytes, &empty))) return rc;
  if (gain_dtype > ARK_ACT_F32) return ark::fail(ARK_OPT_EINVAL, "gain_dtype %u unknown", gain_dtype);
  if (!(eps >= 0.0f) || !isfinite(eps)) return ark::fail(ARK_OPT_EINVAL, "eps = %g", (double)eps);
  uint32_t heads[2] = {};
  if ((rc = check_heads(q_layout, "q", &heads[0]))) return rc;
  if (k_layout && (rc = check_heads(k_layout, "k", &heads[1]))) return rc;
  if (empty || heads[0] + heads[1] == 0) return ARK_OPT_OK;
  const uint32_t ge = ark::act_elem_size(gain_dtype);
  if (((uintptr_t)gain_q | (uintptr_t)gain_k) % ge)
    return ark::fail(ARK_OPT_EINVAL, "gain_q or gain_k not aligned to its element");
  if (((uintptr_t)q_act | (uintptr_t)k_act) % 16)
    return ark::fail(ARK_OPT_EINVAL, "q_act or k_act is not 16-byte aligned");
  const Shape s = {batch, tokens, r->head, ark::act_elem_size(dtype)};
  Given g[4] = {{"q_out", q_out, q_out_layout, true, 0}, {"q", q, q_layout, false, 0},
                {"k_out", k_out, k_out_layout, true, 0}, {"k", k, k_layout, false, 0}};
  static const int in_place[4] = {1, -1, 3, -1};
  for (int i = 0; i < 4; ++i)
    if (heads[i / 2] && (rc = check_given(&g[i], s, heads[i / 2]))) return rc;
  const uint64_t n = batch * tokens;
  const Flat f[5] = {
      {"positions", positions, positions ? n * position_bytes : 0, false},
      {"gain_q", gain_q, heads[0] ? (uint64_t)r->head * ge : 0, false},
      {"gain_k", gain_k, heads[1] ? (uint64_t)r->head * ge : 0, false},
      {"q_act", q_act, q_act && heads[0] ? act_size(n, (uint64_t)heads[0] * r->head) : 0, true},
      {"k_act", k_act, k_act && heads[1] ? act_size(n, (uint64_t)heads[1] * r->head) : 0, true}};
  if ((rc = check_apart(g, 4, in_place, f, 5, s)) || (rc = check_memory(g, 4, f, 5))) return rc;
  Args a = base_args(r, batch, tokens, positions, position_bytes, start);
  a.eps = eps;
  a.gain_dtype = gain_dtype;
  const void* gains[2] = {gain_q, gain_k};
  void* acts[2] = {q_act, k_act};
  uint64_t most = 0;
  ark::DeviceGuard guard(r->device);
  if (!guard.ok) return ark::fail(ARK_OPT_EHIP, "cannot select device %d", r->device);
  bool all_kept = true;
  Part* part = a.part;
  for (int i = 0; i < 2; ++i) {
    if (!heads[i]) continue;
    part->x = array_of(g[2 * i + 1]);
    part->y = array_of(g[2 * i]);
    part->heads = heads[i];
    part->gain = gains[i];
    part->act = (uint8_t*)acts[i];
    all_kept = all_kept && acts[i];
    const uint64_t values = ark::act_groups(n) * heads[i] * r->head;
    most = acts[i] && values > most ? values : most;
    ++part;
  }
  // both parts' tiles and 8-bit forms in one pass, or each in its own
  if (all_kept && tiles_fit(a, false)) {
    launch_tiles<false>(dtype, &a, (hipStream_t)stream);
    ARK_HIP(hipGetLastError());
    return ARK_OPT_OK;
  }
  if (most) {
    const dim3 grid((uint32_t)((most + kBlock - 1) / kBlock), 1, a.part[1].heads ? 2 : 1);
    if (dtype == ARK_ACT_F16)
      hipLaunchKernelGGL(keep_kernel<ARK_ACT_F16>, grid, dim3(kBlock), 0, (hipStream_t)stream, a);
    else if (dtype == ARK_ACT_BF16)
      hipLaunchKernelGGL(keep_kernel<ARK_ACT_BF16>, grid, dim3(kBlock), 0, (hipStream_t)stream, a);
    else
      hipLaunchKernelGGL(keep_kernel<ARK_ACT_F32>, grid, dim3(kBlock), 0, (hipStream_t)stream, a);
    ARK_HIP(hipGetLastError());
  }
  launch_rows<kNorm>(dtype, &a, (hipStream_t)stream);
  ARK_HIP(hipGetLastError());
  return ARK_OPT_OK;
}

int ark_rope_norm_backward(const ark_rope* r, uint32_t dtype, uint64_t batch, uint64_t tokens,
                           const void* positions, uint32_t position_bytes, uint64_t start,
                           float eps, const void* gain_q, const void* gain_k,
                           uint32_t gain_dtype, const void* dq, const uint64_t* dq_layout,
                           const void* q, const uint64_t* q_layout, const void* q_act,
                           void* q_grad, const uint64_t* q_grad_layout, float* dgain_q,
                           const void* dk, const uint64_t* dk_layout, const void* k,
                           const uint64_t* k_layout, const void* k_act, void* k_grad,
                           const uint64_t* k_grad_layout, float* dgain_k, uint32_t accumulate,
                           void* stream) {
  int rc;
  bool empty;
  if ((rc = check_call(r, dtype, batch, tokens, positions, position_bytes, &empty))) return rc;
  if (gain_dtype > ARK_ACT_F32) return ark::fail(ARK_OPT_EINVAL, "gain_dtype %u unknown", gain_dtype);
  if (!(eps >= 0.0f) || !isfinite(eps)) return ark::fail(ARK_OPT_EINVAL, "eps = %g", (double)eps);
  uint32_t heads[2] = {};
  if ((rc = check_heads(dq_layout, "dq", &heads[0]))) return rc;
  if (dk_layout && (rc = check_heads(dk_layout, "dk", &heads[1]))) return rc;
  const uint32_t ge = ark::act_elem_size(gain_dtype);
  if (((uintptr_t)gain_q | (uintptr_t)gain_k) % ge)
    return ark::fail(ARK_OPT_EINVAL, "gain_q or gain_k not aligned to its element");
  if (((uintptr_t)dgain_q | (uintptr_t)dgain_k) % 4)
    return ark::fail(ARK_OPT_EINVAL, "dgain_q or dgain_k not aligned to its element");
  if (((uintptr_t)q_act | (uintptr_t)k_act) % 16)
    return ark::fail(ARK_OPT_EINVAL, "q_act or k_act is not 16-byte aligned");
  const Shape s = {batch, tokens, r->head, ark::act_elem_size(dtype)};
  const bool has[2] = {!empty && heads[0], !empty && heads[1]};
  // an 8-bit form's input is not an array of the call: its entry stays empty
  Given g[6] = {{"q_grad", q_grad, q_grad_layout, true, 0},
                {"dq", dq, dq_layout, false, 0},
                {"q", q_act ? nullptr : q, q_layout, false, 0},
                {"k_grad", k_grad, k_grad_layout, true, 0},
                {"dk", dk, dk_layout, false, 0},
                {"k", k_act ? nullptr : k, k_layout, false, 0}};
  static const int in_place[6] = {1, -1, -1, 4, -1, -1};
  for (int i = 0; i < 6; ++i) {
    if (!has[i / 3] || (i % 3 == 2 && (i == 2 ? q_act : k_act))) continue;
    if ((rc = check_given(&g[i], s, heads[i / 3]))) return rc;
  }
  const uint64_t n = batch * tokens;
  const uint64_t db = (uint64_t)r->head * 4;
  const Flat f[7] = {
      {"positions", positions, positions ? n * position_bytes : 0, false},
      {"gain_q", gain_q, has[0] ? (uint64_t)r->head * ge : 0, false},
      {"gain_k", gain_k, has[1] ? (uint64_t)r->head * ge : 0, false},
      {"q_act", q_act, q_act && has[0] ? act_size(n, (uint64_t)heads[0] * r->head) : 0, false},
      {"k_act", k_act, k_act && has[1] ? act_size(n, (uint64_t)heads[1] * r->head) : 0, false},
      {"dgain_q", dgain_q, db, true},
      {"dgain_k", dgain_k, dk_layout ? db : 0, true}};
  if ((rc = check_apart(g, 6, in_place, f, 7, s)) || (rc = check_memory(g, 6, f, 7))) return rc;
  Args a = base_args(r, batch, tokens, positions, position_bytes, start);
  a.eps = eps;
  a.gain_dtype = gain_dtype;
  const void* gains[2] = {gain_q, gain_k};
  const void* acts[2] = {q_act, k_act};
  bool all_kept = true;
  Part* part = a.part;
  for (int i = 0; i < 2; ++i) {
    if (!has[i]) continue;
    if (!acts[i]) part->x = array_of(g[3 * i + 2]);
    part->dy = array_of(g[3 * i + 1]);
    part->y = array_of(g[3 * i]);
    part->heads = heads[i];
    part->gain = gains[i];
    part->act = (uint8_t*)acts[i];
    all_kept = all_kept && acts[i];
    ++part;
  }
  ark::DeviceGuard guard(r->device);
  if (!guard.ok) return ark::fail(ARK_OPT_EHIP, "cannot select device %d", r->device);
  const hipStream_t st = (hipStream_t)stream;
  const bool tiled = all_kept && tiles_fit(a, true);
  const uint32_t blocks = part == a.part ? 0
                          : tiled ? launch_tiles<true>(dtype, &a, st, false)
                                  : launch_rows<kBack>(dtype, &a, st, false);
  ark::StreamBuf buf;
  if (blocks) {
    const hipError_t e = buf.alloc((uint64_t)(part - a.part) * blocks * r->head * 4, st);
    if (e != hipSuccess) return ark::hip_fail(e, "workspace of ark_rope_norm_backward");
    a.partial = (float*)buf.p;
    tiled ? launch_tiles<true>(dtype, &a, st)
          : launch_rows<kBack>(dtype, &a, st);
    ARK_HIP(hipGetLastError());
  }
  hipLaunchKernelGGL(gain_kernel, dim3((r->head + kGainColumns - 1) / kGainColumns, dk_layout ? 2 : 1),
                     dim3(kGainColumns * kGainRuns), 0, st, (const float*)buf.p,
                     has[0] ? blocks : 0, has[1] ? blocks : 0, r->head, dgain_q, dgain_k,
                     accumulate);
  ARK_HIP(hipGetLastError());
  return ARK_OPT_OK;
}

}  // extern "C"
