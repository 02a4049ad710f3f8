// ark_act.hip -- activations kept in 8 bits and the weight gradient that reads
// them (include/ark_act.h).
#include <atomic>
#include <type_traits>
#include <utility>

#include "ark_act.hpp"
#include "ark_common.hpp"

namespace {

using namespace ark::dev;

constexpr uint32_t kLanes = 256;

// N columns of a row as they lie in memory, at any element's alignment.
template <uint32_t DT, uint32_t N>
struct Columns {
  static constexpr uint32_t kWords = DT == ARK_ACT_F32 ? N : N / 2;
  typedef uint32_t V __attribute__((ext_vector_type(kWords), aligned(DT == ARK_ACT_F32 ? 4 : 2)));
  V v;
  __device__ __forceinline__ float get(uint32_t c) const {
    if constexpr (DT == ARK_ACT_F32) return __uint_as_float(v[c]);
    const uint32_t h = v[c / 2];
    if constexpr (DT == ARK_ACT_BF16) return __uint_as_float(c % 2 ? h & 0xFFFF0000u : h << 16);
    return h2f(h >> (c % 2 * 16) & 0xFFFFu);
  }
};

// A lane takes N columns of a group: 32 loads, no lane needs another's to find
// its columns' largest magnitudes, and 32 N bytes that follow one another.  The
// columns past the last whole N are the last N again, written twice alike.  The
// magnitudes are compared as the types' own bits, two fp16 or bf16 at a time, and
// a value is quantised by one fma, whose rounding is the quantisation's.  Bound
// by HBM: 16384 x 2048 fp16, 101.7 MB, 19 us, 5.3 TB/s (31 us of the round trip
// are a copy's at 6.5).
template <uint32_t DT, uint32_t N>
__global__ __launch_bounds__(kLanes) void pack_kernel(const elem_t<DT>* __restrict__ x,
                                                      uint64_t stride, uint64_t tokens,
                                                      uint32_t columns, uint8_t* __restrict__ q,
                                                      uint8_t* __restrict__ e) {
  typedef Columns<DT, N> C;
  const uint32_t c0 = (blockIdx.x * kLanes + threadIdx.x) * N;
  const uint64_t g = blockIdx.y + (uint64_t)gridDim.y * blockIdx.z;
  const uint64_t t0 = g * ARK_ACT_GROUP;
  if (c0 >= columns || t0 >= tokens) return;
  const uint32_t c = c0 + N <= columns ? c0 : columns - N;
  const uint32_t n = (uint32_t)(tokens - t0 < ARK_ACT_GROUP ? tokens - t0 : ARK_ACT_GROUP);
  const elem_t<DT>* row = x + t0 * stride + c;
  C v[ARK_ACT_GROUP];
  if (n == ARK_ACT_GROUP) {
#pragma unroll
    for (uint32_t i = 0; i < ARK_ACT_GROUP; ++i)
      v[i].v = *(const ARK_GLOBAL typename C::V*)(row + i * stride);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < ARK_ACT_GROUP; ++i) {
      v[i].v = typename C::V();
      if (i < n) v[i].v = *(const ARK_GLOBAL typename C::V*)(row + i * stride);
    }
  }
  typename C::V most = typename C::V();
#pragma unroll
  for (uint32_t i = 0; i < ARK_ACT_GROUP; ++i)
#pragma unroll
    for (uint32_t k = 0; k < C::kWords; ++k)
      most[k] = DT == ARK_ACT_F32 ? max(most[k], v[i].v[k] & 0x7FFFFFFFu)
                                  : max_u16x2(most[k], v[i].v[k] & 0x7FFF7FFFu);
  C top;
  top.v = most;
  uint8_t* out = q + (g * columns + c) * ARK_ACT_GROUP;
  uint32_t s[N];
  bool at_top = false;
#pragma unroll
  for (uint32_t k = 0; k < N; ++k) {
    s[k] = act_exponent<DT>(__float_as_uint(top.get(k)));
    at_top |= s[k] >= kActTop<DT>;
    st_g<uint8_t>(e + g * columns + c + k, (uint8_t)s[k]);
  }
  const auto quantise = [&](auto hold) {
#pragma unroll
    for (uint32_t k = 0; k < N; ++k) {
      const auto at = [&](uint32_t i) {
        return decltype(hold)::value ? act_hold<DT>(s[k], v[i].get(k)) : v[i].get(k);
      };
      u32x4 w[2];
#pragma unroll
      for (uint32_t i = 0; i < ARK_ACT_GROUP / 4; ++i)
        w[i / 4][i % 4] = act_bytes4(s[k], at(4 * i), at(4 * i + 1), at(4 * i + 2), at(4 * i + 3));
      st_g<u32x4>(out + k * ARK_ACT_GROUP, w[0]);
      st_g<u32x4>(out + k * ARK_ACT_GROUP + 16, w[1]);
    }
  };
  if (__builtin_amdgcn_ballot_w64(at_top))
    quantise(std::true_type());
  else
    quantise(std::false_type());
}

// The same lanes' 32 N bytes back to rows, q 2^e exactly but for values that fp16
// and bf16 round.  Bound by HBM: 16384 x 2048 fp16, 14.8 us, 6.9 TB/s.
template <uint32_t DT, uint32_t N>
__global__ __launch_bounds__(kLanes) void unpack_kernel(const uint8_t* __restrict__ q,
                                                        const uint8_t* __restrict__ e,
                                                        uint64_t tokens, uint32_t columns,
                                                        elem_t<DT>* __restrict__ x,
                                                        uint64_t stride) {
  typedef Columns<DT, N> C;
  const uint32_t c0 = (blockIdx.x * kLanes + threadIdx.x) * N;
  const uint64_t g = blockIdx.y + (uint64_t)gridDim.y * blockIdx.z;
  const uint64_t t0 = g * ARK_ACT_GROUP;
  if (c0 >= columns || t0 >= tokens) return;
  const uint32_t c = c0 + N <= columns ? c0 : columns - N;
  const uint32_t n = (uint32_t)(tokens - t0 < ARK_ACT_GROUP ? tokens - t0 : ARK_ACT_GROUP);
  u32x4 w[N][2];
  float up[N];
#pragma unroll
  for (uint32_t k = 0; k < N; ++k) {
    const uint8_t* in = q + (g * columns + c + k) * ARK_ACT_GROUP;
    w[k][0] = ld_g<u32x4>(in);
    w[k][1] = ld_g<u32x4>(in + 16);
    up[k] = act_up(ld_g<uint8_t>(e + g * columns + c + k));
  }
  elem_t<DT>* row = x + t0 * stride + c;
#pragma unroll
  for (uint32_t i = 0; i < ARK_ACT_GROUP; ++i) {
    float f[N];
#pragma unroll
    for (uint32_t k = 0; k < N; ++k)
      f[k] = act_value(w[k][i / 16][i / 4 % 4], i % 4, up[k]);
    typename C::V v;
#pragma unroll
    for (uint32_t k = 0; k < C::kWords; ++k) {
      if constexpr (DT == ARK_ACT_F32)
        v[k] = __float_as_uint(f[k]);
      else
        v[k] = narrow2<DT>(f[2 * k], f[2 * k + 1]);
    }
    if (i < n) *(ARK_GLOBAL typename C::V*)(row + i * stride) = v;
  }
}

// The same for a single column, a group or a token a lane, and the ones a grid on:
// a column may be longer than a launch (2^32 lanes).
template <uint32_t DT>
__global__ __launch_bounds__(kLanes) void pack1_kernel(const elem_t<DT>* __restrict__ x,
                                                       uint64_t stride, uint64_t tokens,
                                                       uint8_t* __restrict__ q,
                                                       uint8_t* __restrict__ e) {
  for (uint64_t g = (uint64_t)blockIdx.x * kLanes + threadIdx.x; g * ARK_ACT_GROUP < tokens;
       g += (uint64_t)gridDim.x * kLanes) {
    const uint64_t t0 = g * ARK_ACT_GROUP;
    uint32_t most = 0;
    const auto at = [&](uint32_t i) {
      return t0 + i < tokens ? (float)x[(t0 + i) * stride] : 0.0f;
    };
    for (uint32_t i = 0; i < ARK_ACT_GROUP; ++i)
      most = max(most, __float_as_uint(at(i)) & 0x7FFFFFFFu);
    const uint32_t s = act_exponent<DT>(most);
    const auto held = [&](uint32_t i) { return act_hold<DT>(s, at(i)); };
    for (uint32_t i = 0; i < ARK_ACT_GROUP; i += 4)
      st_g<uint32_t>(q + t0 + i, act_bytes4(s, held(i), held(i + 1), held(i + 2), held(i + 3)));
    e[g] = (uint8_t)s;
  }
}
template <uint32_t DT>
__global__ __launch_bounds__(kLanes) void unpack1_kernel(const uint8_t* __restrict__ q,
                                                         const uint8_t* __restrict__ e,
                                                         uint64_t tokens,
                                                         elem_t<DT>* __restrict__ x,
                                                         uint64_t stride) {
  for (uint64_t t = (uint64_t)blockIdx.x * kLanes + threadIdx.x; t < tokens;
       t += (uint64_t)gridDim.x * kLanes)
    x[t * stride] = (elem_t<DT>)act_value(q[t], 0, act_up(e[t / ARK_ACT_GROUP]));
}

// ---- the weight gradient -----------------------------------------------------
//
// dw = act^T dy: rows m are act's columns, columns n are dy's, and the sum runs
// over tokens, in fp32.  A block's waves, four along m and WN along n, form a
// tile of 64 MF x 16 NF WN outputs, a wave MF x NF matrix instructions of 16 x 16
// over 32 tokens.  A step is 64 tokens of both operands, which lie in LDS as
// [column or output][token], so that a lane's eight tokens are one 16-byte read.
// act's layout has a column's tokens side by side already: its bytes are widened
// exactly, once for the block, on their way into LDS.  dy's tokens are rows: a
// lane loads the same outputs of eight tokens and turns them in registers.
// What a step needs travels from memory in registers while the step before is
// multiplied, is put into the other of two LDS buffers between its instructions,
// and one barrier a step changes them over.
//
// Bound by the matrix instructions and what they wait for: 16384 x 2048 x 5504,
// bf16, 0.39 ms, 950 TFLOP/s, where a library product of 16-bit operands takes
// 0.35-0.37 and 8192^3 reaches 1.3 PFLOP/s.  The matrix units are busy 44 % of
// the cycles, the vector units and LDS 33 % each, and no access of LDS meets
// another in a bank.  The two waves a SIMD has room for (96 sums a lane) run in
// step by the barrier, so that each unit's pauses only partly fill; spreading
// the staging evenly between the instructions took 2 % off, widening act once
// and the chunks' permutation 3 %.

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
// words at any even address (gfx950 takes unaligned global accesses)
typedef uint32_t u32_a2 __attribute__((aligned(2)));
typedef uint32_t u32x2_a2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32x4_a1 __attribute__((ext_vector_type(4), aligned(1)));

#define ARK_LDS __attribute__((address_space(3)))

template <typename V>
__device__ __forceinline__ ARK_LDS V* lds_at(uint32_t byte) {
  return (ARK_LDS V*)(uintptr_t)byte;
}

constexpr uint32_t kStep = 64;                      // tokens a step
constexpr uint32_t kStepGroups = kStep / ARK_ACT_GROUP;

struct GradArgs {
  const uint8_t* q;        // act's values
  const uint8_t* e;        // and exponents
  const uint16_t* dy;
  float* dw;
  float* partial;          // [splits][tiles][tile's values in lane order], or NULL
  uint64_t tokens, dy_stride, dw_stride, groups;
  uint32_t columns, outputs;
  uint32_t m_tiles, n_tiles, splits, steps;  // steps of all splits together
  uint32_t accumulate, vec;                  // vec: dw takes 16-byte stores
};

template <typename T>
struct Mat;
template <>
struct Mat<_Float16> {
  typedef f16x8 Frag;
  static __device__ __forceinline__ f32x4 mul(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  // The instructions' products are exact, but they align a sum by the factors'
  // exponent fields: a subnormal fp16 counts as 2^-14, and the sum loses what lies 24
  // bits below that (up to 2^10 times as much as it should).  So a column is
  // multiplied by the power of two that takes its largest exponent to 9 (65024 at
  // most; 10, where |q| <= 63, stays): all its values are then normal but those more
  // than 2^23 below its largest 2^e.  The sums are scaled back at the end, exactly.
  // dy stays as it is: what a sum loses by a subnormal one is 2^-12 of half that
  // one's last place.
  static constexpr bool kShift = true;
  static __device__ __forceinline__ uint32_t shift(uint32_t top) {
    return top >= 143u ? 0u : 142u - top;
  }
  // of an exponent byte: 2^(e + shift) twice (at least 2^-24)
  static __device__ __forceinline__ uint32_t scale(uint32_t s, uint32_t shift) {
    const uint32_t h = __builtin_bit_cast(
        uint16_t, (_Float16)(s == 255u ? act_up(s) : __uint_as_float((s - 6u + shift) << 23)));
    return h | h << 16;
  }
  // Two bytes q + 128 of a word, the lower or the upper, to q 2^e: the byte becomes
  // the low mantissa of 1024 + q + 128, which fp16 holds, and both steps after it
  // are exact.
  static __device__ __forceinline__ uint32_t widen(uint32_t w, bool upper, uint32_t scale) {
    const f16x2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    const uint32_t u = __builtin_amdgcn_perm(0x64646464u, w, upper ? 0x04030402u : 0x04010400u);
    return __builtin_bit_cast(
        uint32_t, (__builtin_bit_cast(f16x2, u) + off) * __builtin_bit_cast(f16x2, scale));
  }
};
template <>
struct Mat<__bf16> {
  typedef bf16x8 Frag;
  static __device__ __forceinline__ f32x4 mul(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static constexpr bool kShift = false;  // bf16 has fp32's range
  static __device__ __forceinline__ uint32_t shift(uint32_t) { return 0; }
  static __device__ __forceinline__ uint32_t scale(uint32_t s, uint32_t) {
    return __float_as_uint(act_up(s));
  }
  // q as in fp16's case, then q 2^e in fp32, whose upper half is all of its at
  // most 7 significant bits
  static __device__ __forceinline__ uint32_t widen(uint32_t w, bool upper, uint32_t scale) {
    const float s = __uint_as_float(scale);
    const f16x2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    const uint32_t u = __builtin_amdgcn_perm(0x64646464u, w, upper ? 0x04030402u : 0x04010400u);
    const f16x2 q = __builtin_bit_cast(f16x2, u) + off;
    return __builtin_amdgcn_perm(__float_as_uint((float)q.y * s), __float_as_uint((float)q.x * s),
                                 0x07060302u);
  }
};

// N neighbouring outputs of a token of dy.
template <uint32_t N>
struct Row {
  uint32_t v[(N + 1) / 2] = {};
  __device__ __forceinline__ void load(const char* p) {
    if constexpr (N == 4) {
      const u32x2_a2 t = *(const ARK_GLOBAL u32x2_a2*)p;
      v[0] = t.x, v[1] = t.y;
    } else if constexpr (N == 2) {
      v[0] = *(const ARK_GLOBAL u32_a2*)p;
    } else {
      v[0] = ld_g<uint16_t>(p);
    }
  }
  // drops the first n
  __device__ __forceinline__ void shift(uint32_t n) {
    if constexpr (N == 4) {
      const uint64_t t = ((uint64_t)v[1] << 32 | v[0]) >> (n % 4 * 16);
      v[0] = (uint32_t)t, v[1] = (uint32_t)(t >> 32);
    } else if constexpr (N == 2) {
      v[0] >>= n % 2 * 16;
    }
  }
  // output c of this token and of the next
  __device__ __forceinline__ uint32_t pair(const Row& next, uint32_t c) const {
    return __builtin_amdgcn_perm(next.v[c / 2], v[c / 2], c % 2 ? 0x07060302u : 0x05040100u);
  }
};

// f(0), f(1), ... f(N - 1), each index a constant.
template <typename F, uint32_t... I>
__device__ __forceinline__ void each(F f, std::integer_sequence<uint32_t, I...>) {
  (f(std::integral_constant<uint32_t, I>()), ...);
}
template <uint32_t N, typename F>
__device__ __forceinline__ void each(F f) {
  each(f, std::make_integer_sequence<uint32_t, N>());
}

// A tile's shape, its LDS buffer and what a lane stages of it.
template <uint32_t MF, uint32_t NF, uint32_t WN>
struct Tile {
  static constexpr uint32_t kLanes = 256 * WN;
  static constexpr uint32_t kM = 64 * MF, kN = 16 * NF * WN;
  static constexpr uint32_t kRow = kStep * 2;                    // bytes of an output of dy
  static constexpr uint32_t kA = kN * kRow;                      // dy, then act, a column a row
  static constexpr uint32_t kBytes = kA + kM * kRow;
  static constexpr uint32_t kLds = 2 * kBytes;
  static constexpr uint32_t kWide = NF / 2;                      // outputs a lane stages of 8 tokens
  static constexpr uint32_t kAChunks = kM * (kStep / 8) / kLanes;  // of 8 tokens of act
  static_assert(kAChunks * kLanes == kM * (kStep / 8), "whole chunks");
  static constexpr uint32_t kPhases = 2 * NF;                    // of MF products a step
  static constexpr uint32_t kAhead = NF >= 4 ? 3 : 1;            // dy's reads ahead of them
  // dy and act lie in LDS as rows of one output's or column's 64 tokens, a row's
  // eight 16-byte chunks (8 tokens) permuted by its bits.  LDS takes 16-byte reads
  // sixteen lanes at a time, of each 32 lanes 0-3, 12-15 and 20-27 and then the
  // others, and writes eight neighbours at a time (measured: which pairs of lanes
  // meet).  Reads are of 16 neighbouring rows, the second half of the lanes a chunk
  // on; writes of one chunk of rows kWide apart, or of four chunks of two
  // neighbours: with this permutation none of them meet in a bank.
  static __device__ __forceinline__ uint32_t swizzle(uint32_t n) {
    return ((n >> 1 & 3u) ^ (n >> 4 & 1u)) | ((n >> 3 ^ n) & 1u) << 2;
  }
};

// One lane's four values of a 16 x 16 tile at (m, n): four neighbours of dw's
// rows, which SWAP makes n ([columns][outputs]) and otherwise m (transposed).
template <bool SWAP>
__device__ __forceinline__ void grad_out(const GradArgs& a, uint32_t m, uint32_t n, uint32_t lane,
                                         f32x4 v) {
  const uint32_t row = (SWAP ? m : n) + lane % 16, col = (SWAP ? n : m) + lane / 16 * 4;
  const uint32_t rows = SWAP ? a.columns : a.outputs, cols = SWAP ? a.outputs : a.columns;
  if (row >= rows || col >= cols) return;
  float* p = a.dw + row * a.dw_stride + col;
  if (a.vec && col + 4 <= cols) {
    if (a.accumulate) v += *(const f32x4*)p;
    *(f32x4*)p = v;
    return;
  }
#pragma unroll
  for (uint32_t k = 0; k < 4; ++k)
    if (col + k < cols) p[k] = a.accumulate ? p[k] + v[k] : v[k];
}

// ANY: any stride and number of outputs; otherwise offsets inside a step fit 32
// bits and there are four outputs at least.
template <typename T, uint32_t MF, uint32_t NF, uint32_t WN, bool SWAP, bool ANY>
__global__ __launch_bounds__(256 * WN, 2) void grad_kernel(GradArgs a) {
  typedef typename std::conditional<ANY, uint64_t, uint32_t>::type Off;
  typedef Tile<MF, NF, WN> L;
  typedef Mat<T> M;
  extern __shared__ __align__(16) uint8_t lds[];
  const uint32_t tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  const uint32_t wm = wave % 4, wn = wave / 4, li = lane % 16, lg = lane / 16;
  // blocks of one XCD (every eighth) take neighbouring tiles of one split, which
  // share their operands in its L2
  const uint32_t tiles = a.m_tiles * a.n_tiles, all = gridDim.x;
  const uint32_t per = all / 8, rest = all % 8, xcd = blockIdx.x % 8;
  const uint32_t id = xcd * per + (xcd < rest ? xcd : rest) + blockIdx.x / 8;
  const uint32_t split = id / tiles, tile = id % tiles;
  const uint32_t m0 = tile % a.m_tiles * L::kM, n0 = tile / a.m_tiles * L::kN;
  const uint32_t s0 = (uint32_t)((uint64_t)a.steps * split / a.splits);
  const uint32_t s1 = (uint32_t)((uint64_t)a.steps * (split + 1) / a.splits);

  // What this lane stages of a step: 16 bytes of dy (8 outputs of a token) or of
  // act at a time, and one exponent, at these offsets from the step's start.  No
  // load needs a bound: outputs past the last are loaded from the last eight and
  // shifted into place, columns, tokens and groups past the last repeat it, whose
  // products are never stored or meet dy's zeros.
  typedef Row<L::kWide> R;
  R rb[8];
  u32x2 ra[L::kAChunks];
  uint32_t rs[L::kAChunks], shift[L::kAChunks] = {};
  // the columns' largest exponents, in the second buffer until it is first used
  uint32_t* top = (uint32_t*)(lds + L::kBytes);
  constexpr uint32_t kAcross = L::kN / L::kWide;  // lanes of a token
  const uint32_t b_row = tid / kAcross * 8, b_n = tid % kAcross * L::kWide;
  const bool edge = n0 + L::kN > a.outputs && a.outputs % L::kWide;
  const uint32_t b_col = n0 + b_n + L::kWide <= a.outputs ? n0 + b_n : a.outputs - L::kWide;
  Off oe[L::kAChunks], ob = ((Off)b_row * (Off)a.dy_stride + b_col) * 2;  // bytes
  // chunk i: four of a column's group of 32 tokens, the step's first group first
  const auto a_group = [&](uint32_t i) { return (tid + i * L::kLanes) / (L::kM * 4); };
  const auto a_col = [&](uint32_t i) { return (tid + i * L::kLanes) / 4 % L::kM; };
  const auto place = [&](uint32_t groups) {  // of the step
#pragma unroll
    for (uint32_t i = 0; i < L::kAChunks; ++i) {
      const uint32_t m = m0 + a_col(i);
      oe[i] = (Off)min(a_group(i), groups - 1) * a.columns + min(m, a.columns - 1);
    }
  };
  const auto a_off = [&](Off column) { return column * ARK_ACT_GROUP + tid % 4 * 8; };
  uint32_t la[L::kAChunks];  // where they go in a buffer
#pragma unroll
  for (uint32_t i = 0; i < L::kAChunks; ++i)
    la[i] = L::kA + a_col(i) * L::kRow +
            (a_group(i) * 4 + tid % 4 ^ L::swizzle(a_col(i))) * 16;
  const auto load = [&](uint32_t step) {
    const char* dy = (const char*)(a.dy + (uint64_t)step * kStep * a.dy_stride);
    if (step + 1 < a.steps) {
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) rb[i].load(dy + (uint64_t)i * a.dy_stride * 2 + ob);
    } else {
      const uint32_t n = (uint32_t)(a.tokens - (uint64_t)step * kStep);
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) {
        const uint32_t t = b_row + i < n ? b_row + i : n - 1;
        rb[i].load(dy + ((Off)t * (Off)a.dy_stride + b_col) * 2);
      }
      place((uint32_t)(a.groups - (uint64_t)step * kStepGroups));
    }
    const uint64_t g0 = (uint64_t)step * kStepGroups * a.columns;
    const char *q = (const char*)a.q + g0 * ARK_ACT_GROUP, *e = (const char*)a.e + g0;
#pragma unroll
    for (uint32_t i = 0; i < L::kAChunks; ++i) {
      ra[i] = ld_g<u32x2>(q + a_off(oe[i]));
      rs[i] = ld_g<uint8_t>(e + oe[i]);
    }
  };
  // LDS is addressed in bytes.
  const uint32_t base = (uint32_t)(uintptr_t)(ARK_LDS uint8_t*)lds;
  const auto put_b = [&](uint32_t buf, uint32_t c) {  // output b_n + c
    const uint32_t n = b_n + c;
    u32x4 v;
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) v[k] = rb[2 * k].pair(rb[2 * k + 1], c);
    *lds_at<u32x4>(buf + n * L::kRow + (b_row / 8 ^ L::swizzle(n)) * 16) = v;
  };
  // a chunk of act in five parts: four words widened, then put
  u32x4 wide;
  const auto put_a = [&](uint32_t buf, uint32_t i, uint32_t part) {
    if (part < 4)
      wide[part] = M::widen(part < 2 ? ra[i].x : ra[i].y, part % 2, M::scale(rs[i], shift[i]));
    else
      *lds_at<u32x4>(buf + la[i]) = wide;
  };
  const auto store = [&](uint32_t buf, uint32_t step) {
    if (edge) {
      const uint32_t drop = n0 + b_n + L::kWide > a.outputs ? n0 + b_n + L::kWide - a.outputs : 0;
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) rb[i].shift(drop);
    }
    if (step + 1 == a.steps) {
      const uint32_t n = (uint32_t)(a.tokens - (uint64_t)step * kStep);
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i)
        if (b_row + i >= n) rb[i] = R();
    }
#pragma unroll
    for (uint32_t c = 0; c < L::kWide; ++c) put_b(buf, c);
#pragma unroll
    for (uint32_t i = 0; i < 5 * L::kAChunks; ++i) put_a(buf, i / 5, i % 5);
  };

  if (s0 < s1) {
    place(kStepGroups);
    load(s0);
  }
  uint32_t back[MF] = {};  // the shifts of this lane's sums, a byte each
  if constexpr (M::kShift) {
    for (uint32_t i = tid; i < L::kM; i += L::kLanes) top[i] = 109;
    __syncthreads();
    // the columns' exponents over the split, 16 columns of a group at a time
    const uint32_t groups = (uint32_t)((uint64_t)s1 * kStepGroups < a.groups
                                           ? (uint64_t)s1 * kStepGroups : a.groups);
    const uint32_t m = tid % (L::kM / 16) * 16;
    if (a.columns >= 16 && m0 + m < a.columns) {
      const uint32_t c = m0 + m + 16 <= a.columns ? m0 + m : a.columns - 16;
      u32x4 even = {0, 0, 0, 0}, odd = even;  // bytes 0 and 2, 1 and 3 of each word
#pragma unroll 4
      for (uint32_t g = s0 * kStepGroups + tid / (L::kM / 16); g < groups;
           g += L::kLanes / (L::kM / 16)) {
        const u32x4 v = *(const ARK_GLOBAL u32x4_a1*)(a.e + (uint64_t)g * a.columns + c);
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
          even[k] = max_u16x2(even[k], v[k] & 0x00FF00FFu);
          odd[k] = max_u16x2(odd[k], v[k] >> 8 & 0x00FF00FFu);
        }
      }
#pragma unroll
      for (uint32_t k = 0; k < 16; ++k) {
        const uint32_t v = (k % 2 ? odd : even)[k / 4] >> (k % 4 / 2 * 16) & 0xFFFFu;
        if (c + k >= m0) atomicMax(&top[c + k - m0], v);
      }
    } else if (a.columns < 16 && tid < a.columns) {  // one tile, m0 = 0
      for (uint32_t g = s0 * kStepGroups; g < groups; ++g)
        atomicMax(&top[tid], (uint32_t)a.e[(uint64_t)g * a.columns + tid]);
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < L::kAChunks; ++i) shift[i] = M::shift(top[a_col(i)]);
#pragma unroll
    for (uint32_t i = 0; i < MF; ++i)
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k)
        back[i] |= M::shift(top[(wm * MF + i) * 16 + (SWAP ? li : lg * 4 + k)]) << (8 * k);
  }

  f32x4 acc[MF][NF];
#pragma unroll
  for (uint32_t i = 0; i < MF; ++i)
#pragma unroll
    for (uint32_t j = 0; j < NF; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

  // A step's products go in phases: the MF that share dy's fragment j.
  // dy's fragments are read kAhead phases before their products, act's of the
  // next group while this one's are used.  The barrier comes when the last of
  // the step's reads is done, before its last kAhead phases, which then read
  // the next step's first fragments.
  typename M::Frag b[L::kAhead + 1], x[2][MF];
  const uint32_t b_first = wn * NF * 16 + li;
  const uint32_t b_get = b_first * L::kRow + (lg ^ L::swizzle(b_first)) * 16;
  const uint32_t a_first = wm * MF * 16 + li;
  const uint32_t a_get = L::kA + a_first * L::kRow + (lg ^ L::swizzle(a_first)) * 16;
  const auto read_b = [&](uint32_t buf, uint32_t phase) {
    const uint32_t h = phase / NF, j = phase % NF;
    // 16 rows on, bit 4 turns over, and with it the permutation's bit 0
    b[phase % (L::kAhead + 1)] = *lds_at<typename M::Frag>(
        ((buf + b_get) ^ (h * 64 + j % 2 * 16)) + j * 16 * L::kRow);
  };
  const auto read_a = [&](uint32_t buf, uint32_t h, uint32_t i) {
    x[h][i] = *lds_at<typename M::Frag>(((buf + a_get) ^ (h * 64 + i % 2 * 16)) + i * 16 * L::kRow);
  };
  static_assert(L::kPhases % (L::kAhead + 1) == 0, "a step starts at b[0]");
  if (s0 < s1) {
    store(base, s0);
    if (s0 + 1 < s1) load(s0 + 1);
    __syncthreads();
#pragma unroll
    for (uint32_t p = 0; p < L::kAhead; ++p) read_b(base, p);
#pragma unroll
    for (uint32_t i = 0; i < MF; ++i) read_a(base, 0, i);
  }
  // A plain step's staging one piece at a time: what a chunk's registers hold goes
  // to the next step's buffer, and the chunk after it is asked for.
  constexpr uint32_t kItemsB = L::kWide + 8, kItemsA = 5 * L::kAChunks;
  const auto pass_on_b = [&](auto item, uint32_t buf, uint32_t step) {
    constexpr uint32_t k = decltype(item)::value;
    if constexpr (k < L::kWide) {
      put_b(buf, k);
    } else {
      constexpr uint32_t i = k - L::kWide;
      Off o = ob;
      asm("" : "+v"(o));  // kept apart from the base, which then stays scalar
      rb[i].load((const char*)(a.dy + ((uint64_t)step * kStep + i) * a.dy_stride) + o);
    }
  };
  const auto pass_on_a = [&](auto item, uint32_t buf, uint32_t step) {
    constexpr uint32_t i = decltype(item)::value / 5, part = decltype(item)::value % 5;
    put_a(buf, i, part);
    if constexpr (part == 4) {
      const uint64_t g0 = (uint64_t)step * kStepGroups * a.columns;
      Off n = oe[i], o = a_off(n);
      asm("" : "+v"(o), "+v"(n));
      ra[i] = ld_g<u32x2>((const char*)a.q + g0 * ARK_ACT_GROUP + o);
      rs[i] = ld_g<uint8_t>((const char*)a.e + g0 + n);
    }
  };
  const auto multiply = [&](uint32_t s, auto whole) {
    constexpr bool kPlain = decltype(whole)::value;
    constexpr uint32_t kLast = L::kPhases - L::kAhead;  // first phase past the barrier
    const uint32_t odd = (s - s0) % 2;
    const uint32_t cur = base + odd * L::kBytes, nxt = base + (odd ^ 1u) * L::kBytes;
    each<L::kPhases>([&](auto phase) __attribute__((always_inline)) {
      constexpr uint32_t p = decltype(phase)::value, h = p / NF, j = p % NF;
      if constexpr (p + L::kAhead < L::kPhases)
        read_b(cur, p + L::kAhead);
      else
        read_b(nxt, p + L::kAhead - L::kPhases);
      // act's fragments of the step's second group over its first phases, of the
      // next step's first past the barrier
#pragma unroll
      for (uint32_t i = 0; i < MF; ++i) {
        if (p == i * NF / (2 * MF)) read_a(cur, 1, i);
        if (p == kLast) read_a(nxt, 0, i);
      }
      if constexpr (kPlain) {
        each<kItemsB>([&](auto k) __attribute__((always_inline)) {
          if constexpr (p == k * kLast / kItemsB) pass_on_b(k, nxt, s + 2);
        });
        each<kItemsA>([&](auto k) __attribute__((always_inline)) {
          if constexpr (p == k * kLast / kItemsA) pass_on_a(k, nxt, s + 2);
        });
      } else {
        if (p == 0 && s + 1 < s1) store(nxt, s + 1);
        if (p == 1 && s + 2 < s1) load(s + 2);
      }
#pragma unroll
      for (uint32_t i = 0; i < MF; ++i)
        acc[i][j] = SWAP ? M::mul(b[p % (L::kAhead + 1)], x[h][i], acc[i][j])
                         : M::mul(x[h][i], b[p % (L::kAhead + 1)], acc[i][j]);
      if constexpr (p + 1 == kLast) __syncthreads();
      if constexpr (kPlain) {
        // an instruction for the matrix unit, then as many as fit into its time
#pragma unroll
        for (uint32_t i = 0; i < MF; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  // steps whose loads and stores are plain, then the others
  uint32_t s = s0;
  if (!edge)
    for (; s + 2 < s1 && s + 3 < a.steps; ++s) multiply(s, std::true_type());
  for (; s < s1; ++s) multiply(s, std::false_type());
  if constexpr (M::kShift) {
#pragma unroll
    for (uint32_t i = 0; i < MF; ++i) {
      f32x4 f;
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) {
        f[k] = __uint_as_float((127u - (back[i] >> (8 * k) & 255u)) << 23);
      }
#pragma unroll
      for (uint32_t j = 0; j < NF; ++j) acc[i][j] *= f;
    }
  }

  if (a.partial) {
    f32x4* out = (f32x4*)a.partial + (uint64_t)id * MF * NF * L::kLanes + tid;
#pragma unroll
    for (uint32_t i = 0; i < MF; ++i)
#pragma unroll
      for (uint32_t j = 0; j < NF; ++j) out[(i * NF + j) * L::kLanes] = acc[i][j];
    return;
  }
#pragma unroll
  for (uint32_t i = 0; i < MF; ++i)
#pragma unroll
    for (uint32_t j = 0; j < NF; ++j)
      grad_out<SWAP>(a, m0 + (wm * MF + i) * 16, n0 + (wn * NF + j) * 16, lane, acc[i][j]);
}

// The splits' partial tiles added in order, so that equal calls give equal bits.
// Bound by memory: 16384 x 768 x 2048 in 8 splits, 50 MB read, 9.5 us.
template <uint32_t MF, uint32_t NF, uint32_t WN, bool SWAP>
__global__ __launch_bounds__(256 * WN) void grad_sum_kernel(GradArgs a) {
  typedef Tile<MF, NF, WN> L;
  const uint32_t tiles = a.m_tiles * a.n_tiles;
  const uint32_t tile = blockIdx.x / (MF * NF), f = blockIdx.x % (MF * NF);
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const f32x4* p = (const f32x4*)a.partial +
                   ((uint64_t)tile * MF * NF + f) * L::kLanes + threadIdx.x;
  const uint64_t step = (uint64_t)tiles * MF * NF * L::kLanes;
  f32x4 s = p[0];
  for (uint32_t k = 1; k < a.splits; ++k) s += p[k * step];
  grad_out<SWAP>(a, tile % a.m_tiles * L::kM + (wave % 4 * MF + f / NF) * 16,
                 tile / a.m_tiles * L::kN + (wave / 4 * NF + f % NF) * 16, lane, s);
}

int check_dtype(uint32_t dtype, const char* what) {
  if (dtype > ARK_ACT_F32) return ark::fail(ARK_OPT_EINVAL, "%s %u unknown", what, dtype);
  return ARK_OPT_OK;
}

// Sizes for which no address below wraps: fewer than 2^31 columns and 2^40 tokens,
// and 2^47 values at most, so any byte offset fits 64 bits with room to spare.
int check_sizes(uint64_t tokens, uint64_t columns) {
  if (columns >= (1ull << 31))
    return ark::fail(ARK_OPT_EINVAL, "columns = %llu too large", (unsigned long long)columns);
  if (tokens >= (1ull << 40) || (columns && tokens > (1ull << 47) / columns))
    return ark::fail(ARK_OPT_EINVAL, "tokens = %llu too large", (unsigned long long)tokens);
  return ARK_OPT_OK;
}

// Bytes that rows x row elements at a row stride span; 0 for none.  Fails when
// a written array's rows overlap or an address would wrap.
int rows_bytes(uint64_t rows, uint64_t row, uint64_t stride, uint32_t es, bool written,
               const char* what, uint64_t* bytes) {
  *bytes = 0;
  if (rows == 0 || row == 0) return ARK_OPT_OK;
  if (rows > 1 && (stride >= (1ull << 47) || (rows - 1) > (1ull << 48) / (stride ? stride : 1)))
    return ark::fail(ARK_OPT_EINVAL, "%s: stride %llu too large", what, (unsigned long long)stride);
  if (written && rows > 1 && stride < row)
    return ark::fail(ARK_OPT_EINVAL, "%s: rows of %llu elements overlap at stride %llu", what,
                     (unsigned long long)row, (unsigned long long)stride);
  *bytes = ((rows - 1) * stride + row) * es;
  return ARK_OPT_OK;
}

int check_act(const void* act, uint64_t tokens, uint64_t columns, ark::BufferChecker* checker) {
  if ((uintptr_t)act % 16)
    return ark::fail(ARK_OPT_EINVAL, "act %p is not 16-byte aligned", act);
  return checker->check(act, 33 * ark::act_groups(tokens) * columns, "act", 0);
}

// Blocks over groups in y and z, each within a launch's 65535.
constexpr uint64_t kMaxGroups = 65535ull * 32768;
dim3 group_grid(uint64_t x, uint64_t groups) {
  const uint64_t y = groups < 32768 ? groups : 32768;
  return dim3((uint32_t)x, (uint32_t)y, (uint32_t)((groups + y - 1) / y));
}

// pack and unpack's arguments.  *skip: nothing to do.
int check_copy(const void* x, uint64_t x_stride, uint32_t dtype, uint64_t tokens, uint64_t columns,
               const void* act, bool unpack, bool* skip, uint64_t* x_bytes) {
  int rc;
  *skip = tokens == 0 || columns == 0;
  if ((rc = check_dtype(dtype, "dtype"))) return rc;
  if ((rc = check_sizes(tokens, columns))) return rc;
  if (*skip) return ARK_OPT_OK;
  if (columns > 1 && ark::act_groups(tokens) > kMaxGroups)
    return ark::fail(ARK_OPT_EINVAL, "tokens = %llu too large", (unsigned long long)tokens);
  const uint32_t es = ark::act_elem_size(dtype);
  if ((uintptr_t)x % es) return ark::fail(ARK_OPT_EINVAL, "x not aligned to its element");
  if ((rc = rows_bytes(tokens, columns, x_stride, es, unpack, "x", x_bytes))) return rc;
  if (ark::overlaps(x, *x_bytes, act, 33 * ark::act_groups(tokens) * columns))
    return ark::fail(ARK_OPT_EINVAL, "x and act overlap");
  ark::BufferChecker checker;
  if ((rc = check_act(act, tokens, columns, &checker))) return rc;
  return checker.check(x, *x_bytes, "x", 0);
}

// Blocks for n lanes' work of a single column's kernels.
dim3 column_grid(uint64_t n) {
  const uint64_t blocks = (n + kLanes - 1) / kLanes;
  return dim3((uint32_t)(blocks < (1u << 20) ? blocks : 1u << 20));
}

// Columns a lane takes: two (4 bytes of 16-bit rows); four take twice the
// registers and leave half the waves (16384 x 2048 fp16, both ways: 37.5 us by
// two, 44.6 by four).
constexpr uint32_t kWide = 2;

template <uint32_t DT>
void launch_pack(const void* x, uint64_t stride, uint64_t tokens, uint64_t columns, uint8_t* act,
                 hipStream_t s) {
  const uint64_t groups = ark::act_groups(tokens);
  uint8_t* e = act + groups * columns * ARK_ACT_GROUP;
  const elem_t<DT>* p = (const elem_t<DT>*)x;
  if (columns < kWide)
    hipLaunchKernelGGL(pack1_kernel<DT>, column_grid(groups), dim3(kLanes), 0, s, p, stride,
                       tokens, act, e);
  else
    hipLaunchKernelGGL((pack_kernel<DT, kWide>),
                       group_grid((columns + kLanes * kWide - 1) / (kLanes * kWide), groups),
                       dim3(kLanes), 0, s, p, stride, tokens, (uint32_t)columns, act, e);
}

template <uint32_t DT>
void launch_unpack(const uint8_t* act, uint64_t tokens, uint64_t columns, void* x, uint64_t stride,
                   hipStream_t s) {
  const uint64_t groups = ark::act_groups(tokens);
  const uint8_t* e = act + groups * columns * ARK_ACT_GROUP;
  elem_t<DT>* p = (elem_t<DT>*)x;
  if (columns < kWide)
    hipLaunchKernelGGL(unpack1_kernel<DT>, column_grid(tokens), dim3(kLanes), 0, s, act, e,
                       tokens, p, stride);
  else
    hipLaunchKernelGGL((unpack_kernel<DT, kWide>),
                       group_grid((columns + kLanes * kWide - 1) / (kLanes * kWide), groups),
                       dim3(kLanes), 0, s, act, e, tokens, (uint32_t)columns, p, stride);
}

// How a call is cut: the tile (64 mf x 16 nf wn outputs) and the splits of the
// tokens, each summed by blocks of its own.
struct Cut {
  uint32_t mf, nf, wn, splits;
  uint64_t tiles;
  // the splits' partial tiles
  uint64_t bytes() const {
    return splits > 1 ? tiles * splits * (64 * mf) * (16 * nf * wn) * 4 : 0;
  }
};

// Microseconds a step of 64 tokens takes a tile's block: alone on its compute
// unit (256 tiles), and its share of a unit full of blocks (2048 tiles), both
// with every unit busy (MI355X, 8192 tokens, the mean of fp16 and bf16).
struct Pace {
  uint32_t mf, nf, wn;
  float alone, full;
};
constexpr Pace kPaces[] = {{3, 8, 2, 1.60f, 1.60f}, {3, 8, 1, 1.15f, 0.95f},
                           {2, 4, 1, 0.74f, 0.45f}, {1, 4, 1, 0.59f, 0.27f}};

// The cut expected to end first: the tile's pace times the blocks the fullest
// of 256 compute units gets, and for splits a launch and the partial tiles'
// way to memory and back at 4 TB/s.
Cut cut_of(uint64_t tokens, uint64_t columns, uint64_t outputs, bool any) {
  const uint64_t steps = (tokens + kStep - 1) / kStep;
  const auto tiles = [&](uint32_t mf, uint32_t n) {
    return ((columns + 64 * mf - 1) / (64 * mf)) * ((outputs + n - 1) / n);
  };
  if (any || steps == 0) return {1, 2, 2, 1, tiles(1, 64)};
  Cut best = {};
  float best_us = 0.0f;
  for (const Pace& p : kPaces) {
    const uint64_t t = tiles(p.mf, 16 * p.nf * p.wn);
    for (uint32_t k = 1; k <= 32 && k <= steps; ++k) {
      const uint64_t per_unit = (t * k + 255) / 256;
      const float pace = per_unit * p.full > p.alone ? per_unit * p.full : p.alone;
      const Cut c = {p.mf, p.nf, p.wn, k, t};
      const float us = (float)((steps + k - 1) / k) * pace +
                       (k > 1 ? 4.0f + (float)c.bytes() * 2.0f / 4e6f : 0.0f);
      if (best.mf == 0 || us < best_us) best = c, best_us = us;
    }
  }
  return best;
}

// Offsets inside a step's rows of dy and act fit 32 bits, and a lane's four
// outputs are there; other calls take the kernel that asks for neither.
bool needs_any(uint64_t columns, uint64_t dy_stride, uint64_t outputs) {
  return outputs < 4 || outputs >= (1u << 25) || dy_stride >= (1u << 25) || columns >= (1u << 25);
}

template <typename T, uint32_t MF, uint32_t NF, uint32_t WN, bool SWAP, bool ANY>
int launch_grad(const GradArgs& a, hipStream_t s) {
  typedef Tile<MF, NF, WN> L;
  const void* kernel = (const void*)grad_kernel<T, MF, NF, WN, SWAP, ANY>;
  static std::atomic<uint64_t> ready{0};  // devices that know the kernel's LDS
  int dev = 0;
  ARK_HIP(hipGetDevice(&dev));
  if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1u)) {
    ARK_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, L::kLds));
    if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  const uint64_t tiles = (uint64_t)a.m_tiles * a.n_tiles;
  hipLaunchKernelGGL((grad_kernel<T, MF, NF, WN, SWAP, ANY>), dim3((uint32_t)(tiles * a.splits)),
                     dim3(L::kLanes), L::kLds, s, a);
  ARK_HIP(hipGetLastError());
  if (a.splits > 1) {
    hipLaunchKernelGGL((grad_sum_kernel<MF, NF, WN, SWAP>), dim3((uint32_t)(tiles * MF * NF)),
                       dim3(L::kLanes), 0, s, a);
    ARK_HIP(hipGetLastError());
  }
  return ARK_OPT_OK;
}

template <typename T, uint32_t MF, uint32_t NF, uint32_t WN, bool ANY = false>
int launch_tile(const GradArgs& a, bool transposed, hipStream_t s) {
  return transposed ? launch_grad<T, MF, NF, WN, false, ANY>(a, s)
                    : launch_grad<T, MF, NF, WN, true, ANY>(a, s);
}

template <typename T>
int run_grad(const GradArgs& a, const Cut& c, bool any, bool transposed, hipStream_t s) {
  if (any) return launch_tile<T, 1, 2, 2, true>(a, transposed, s);
  if (c.mf == 3 && c.wn == 2) return launch_tile<T, 3, 8, 2>(a, transposed, s);
  if (c.mf == 3) return launch_tile<T, 3, 8, 1>(a, transposed, s);
  if (c.mf == 2) return launch_tile<T, 2, 4, 1>(a, transposed, s);
  return launch_tile<T, 1, 4, 1>(a, transposed, s);
}

// The call's checks and launches; workspace NULL: one of the library's own.
int weight_grad(const void* act, uint32_t act_dtype, uint64_t tokens, uint64_t columns,
                const void* dy, uint64_t dy_stride, uint32_t dy_dtype, uint64_t outputs,
                float* dw, uint64_t dw_stride, uint32_t flags, bool given, void* workspace,
                uint64_t workspace_bytes, void* stream) {
  int rc;
  if ((rc = check_dtype(act_dtype, "act_dtype"))) return rc;
  if (dy_dtype != ARK_ACT_F16 && dy_dtype != ARK_ACT_BF16)
    return ark::fail(ARK_OPT_EINVAL, "dy_dtype %u: dy is fp16 or bf16", dy_dtype);
  if (dy_dtype == ARK_ACT_F16 && act_dtype != ARK_ACT_F16)
    return ark::fail(ARK_OPT_EINVAL,
                     "fp16 dy needs an act packed from fp16 (others' values may not fit fp16)");
  if (flags & ~(ARK_ACT_ACCUMULATE | ARK_ACT_TRANSPOSED))
    return ark::fail(ARK_OPT_EINVAL, "flags %#x unknown", flags);
  if ((rc = check_sizes(tokens, columns)) || (rc = check_sizes(tokens, outputs))) return rc;
  if (columns == 0 || outputs == 0) return ARK_OPT_OK;
  if (((uintptr_t)dy % 2) || ((uintptr_t)dw % 4))
    return ark::fail(ARK_OPT_EINVAL, "dy or dw not aligned to its element");
  uint64_t dyb, dwb;
  const bool tr = flags & ARK_ACT_TRANSPOSED;
  if ((rc = rows_bytes(tokens, outputs, dy_stride, 2, false, "dy", &dyb))) return rc;
  if ((rc = rows_bytes(tr ? outputs : columns, tr ? columns : outputs, dw_stride, 4, true, "dw",
                       &dwb)))
    return rc;
  const uint64_t ab = 33 * ark::act_groups(tokens) * columns;
  if (ark::overlaps(dw, dwb, act, ab) || ark::overlaps(dw, dwb, dy, dyb))
    return ark::fail(ARK_OPT_EINVAL, "dw overlaps act or dy");
  if (tokens == 0 && (flags & ARK_ACT_ACCUMULATE)) return ARK_OPT_OK;
  const bool any = needs_any(columns, dy_stride, outputs);
  const Cut c = cut_of(tokens, columns, outputs, any);
  const uint64_t steps = (tokens + kStep - 1) / kStep;
  // a launch holds fewer than 2^32 lanes, 256 wn a block (the sum of splits has
  // mf * nf blocks a tile)
  const uint64_t blocks = c.splits > 1 ? c.tiles * (c.splits > c.mf * c.nf ? c.splits : c.mf * c.nf)
                                       : c.tiles;
  if (steps >= (1ull << 31) || blocks >= (1ull << 32) / (256 * c.wn))
    return ark::fail(ARK_OPT_EINVAL, "tokens, columns or outputs too large");
  ark::BufferChecker checker;
  if (given && c.bytes()) {
    if (workspace_bytes < c.bytes())
      return ark::fail(ARK_OPT_EINVAL, "workspace of %llu B, %llu B needed",
                       (unsigned long long)workspace_bytes, (unsigned long long)c.bytes());
    if ((uintptr_t)workspace % 16)
      return ark::fail(ARK_OPT_EINVAL, "workspace %p is not 16-byte aligned", workspace);
    if (ark::overlaps(workspace, c.bytes(), act, ab) || ark::overlaps(workspace, c.bytes(), dy, dyb) ||
        ark::overlaps(workspace, c.bytes(), dw, dwb))
      return ark::fail(ARK_OPT_EINVAL, "workspace overlaps act, dy or dw");
    if ((rc = checker.check(workspace, c.bytes(), "workspace", 0))) return rc;
  }
  if (tokens && (rc = check_act(act, tokens, columns, &checker))) return rc;
  if ((rc = checker.check(dy, dyb, "dy", 0))) return rc;
  if ((rc = checker.check(dw, dwb, "dw", 0))) return rc;
  {
    const void* d[2] = {dw, workspace};  // dw may be an optimizer's gradient
    const uint64_t b[2] = {dwb, given ? c.bytes() : 0};
    ark::opt_units_invalidate(d, b, given ? 2 : 1);
  }
  const hipStream_t s = (hipStream_t)stream;
  GradArgs a = {};
  a.groups = ark::act_groups(tokens);
  a.q = (const uint8_t*)act;
  a.e = a.q + a.groups * columns * ARK_ACT_GROUP;
  a.dy = (const uint16_t*)dy;
  a.dw = dw;
  a.tokens = tokens;
  a.dy_stride = dy_stride;
  a.dw_stride = dw_stride;
  a.columns = (uint32_t)columns;
  a.outputs = (uint32_t)outputs;
  a.accumulate = flags & ARK_ACT_ACCUMULATE ? 1u : 0u;
  a.vec = ((uintptr_t)dw % 16 == 0 && dw_stride % 4 == 0) ? 1u : 0u;
  a.steps = (uint32_t)steps;
  a.m_tiles = (uint32_t)((columns + 64 * c.mf - 1) / (64 * c.mf));
  a.n_tiles = (uint32_t)((outputs + 16 * c.nf * c.wn - 1) / (16 * c.nf * c.wn));
  a.splits = c.splits;
  ark::StreamBuf buf;
  if (c.splits > 1) {
    a.partial = (float*)workspace;
    if (!given) {
      const hipError_t e = buf.alloc(c.bytes(), s);
      if (e != hipSuccess) return ark::hip_fail(e, "workspace of ark_act_weight_grad");
      a.partial = (float*)buf.p;
    }
  }
  return dy_dtype == ARK_ACT_F16 ? run_grad<_Float16>(a, c, any, tr, s)
                                 : run_grad<__bf16>(a, c, any, tr, s);
}

}  // namespace

extern "C" {

int ark_act_bytes(uint64_t tokens, uint64_t columns, uint64_t* bytes) {
  if (!bytes) return ark::fail(ARK_OPT_EINVAL, "bytes is NULL");
  *bytes = 0;
  if (int rc = check_sizes(tokens, columns)) return rc;
  *bytes = 33 * ark::act_groups(tokens) * columns;
  return ARK_OPT_OK;
}

int ark_act_pack(const void* x, uint64_t x_stride, uint32_t dtype, uint64_t tokens,
                 uint64_t columns, void* act, void* stream) {
  bool skip;
  uint64_t xb;
  if (int rc = check_copy(x, x_stride, dtype, tokens, columns, act, false, &skip, &xb)) return rc;
  if (skip) return ARK_OPT_OK;
  {
    const void* d = act;
    const uint64_t b = 33 * ark::act_groups(tokens) * columns;
    ark::opt_units_invalidate(&d, &b, 1);
  }
  const hipStream_t s = (hipStream_t)stream;
  if (dtype == ARK_ACT_F16)
    launch_pack<ARK_ACT_F16>(x, x_stride, tokens, columns, (uint8_t*)act, s);
  else if (dtype == ARK_ACT_BF16)
    launch_pack<ARK_ACT_BF16>(x, x_stride, tokens, columns, (uint8_t*)act, s);
  else
    launch_pack<ARK_ACT_F32>(x, x_stride, tokens, columns, (uint8_t*)act, s);
  ARK_HIP(hipGetLastError());
  return ARK_OPT_OK;
}

int ark_act_unpack(const void* act, uint64_t tokens, uint64_t columns, uint32_t dtype, void* x,
                   uint64_t x_stride, void* stream) {
  bool skip;
  uint64_t xb;
  if (int rc = check_copy(x, x_stride, dtype, tokens, columns, act, true, &skip, &xb)) return rc;
  if (skip) return ARK_OPT_OK;
  {
    const void* d = x;
    ark::opt_units_invalidate(&d, &xb, 1);
  }
  const hipStream_t s = (hipStream_t)stream;
  const uint8_t* a = (const uint8_t*)act;
  if (dtype == ARK_ACT_F16)
    launch_unpack<ARK_ACT_F16>(a, tokens, columns, x, x_stride, s);
  else if (dtype == ARK_ACT_BF16)
    launch_unpack<ARK_ACT_BF16>(a, tokens, columns, x, x_stride, s);
  else
    launch_unpack<ARK_ACT_F32>(a, tokens, columns, x, x_stride, s);
  ARK_HIP(hipGetLastError());
  return ARK_OPT_OK;
}

int ark_act_weight_grad(const void* act, uint32_t act_dtype, uint64_t tokens, uint64_t columns,
                        const void* dy, uint64_t dy_stride, uint32_t dy_dtype, uint64_t outputs,
                        float* dw, uint64_t dw_stride, uint32_t flags, void* stream) {
  return weight_grad(act, act_dtype, tokens, columns, dy, dy_stride, dy_dtype, outputs, dw,
                     dw_stride, flags, false, nullptr, 0, stream);
}

int ark_act_weight_grad_workspace(uint64_t tokens, uint64_t columns, uint64_t dy_stride,
                                  uint64_t outputs, uint64_t* bytes) {
  if (!bytes) return ark::fail(ARK_OPT_EINVAL, "bytes is NULL");
  *bytes = 0;
  int rc;
  if ((rc = check_sizes(tokens, columns)) || (rc = check_sizes(tokens, outputs))) return rc;
  if (columns && outputs)
    *bytes = cut_of(tokens, columns, outputs, needs_any(columns, dy_stride, outputs)).bytes();
  return ARK_OPT_OK;
}

int ark_act_weight_grad_noalloc(const void* act, uint32_t act_dtype, uint64_t tokens,
                                uint64_t columns, const void* dy, uint64_t dy_stride,
                                uint32_t dy_dtype, uint64_t outputs, float* dw,
                                uint64_t dw_stride, uint32_t flags, void* workspace,
                                uint64_t workspace_bytes, void* stream) {
  return weight_grad(act, act_dtype, tokens, columns, dy, dy_stride, dy_dtype, outputs, dw,
                     dw_stride, flags, true, workspace, workspace_bytes, stream);
}

}  // extern "C"
