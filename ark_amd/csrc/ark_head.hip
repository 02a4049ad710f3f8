// ark_head.hip -- the loss over a vocabulary and its gradients, and distillation
// from a teacher's top logits (include/ark_head.h).
//
// With live rows X (the tokens that have a loss, copied together), the output
// layer W and sparse targets p, a piece of the tokens takes these steps:
//
//   rank_kernel     which tokens are live, and what follows from how many there are
//                   (for few tokens gather_kernel's)
//   gather_kernel   X, padded to whole steps of the products, and its targets; zeros
//                   for the tokens without a loss
//   logits_kernel   z = scale X W^T in tiles that stay in registers; z at targets in
//                   fp32; of every row and span of the vocabulary a power of two 2^t
//                   next to its largest exp(z) and its sum of exp(z) / 2^t, and with
//                   gradients these exponentials themselves, in 16 bits (Kept)
//   loss_kernel     the spans' sums joined: log(sum exp z), the loss
//   dz_kernel       the same, and the exponentials turned into dz where they lie
//   grad_kernel     dx = dz W and dw = dz^T X, in one launch
//   join_kernel     sums that were formed in parts
//
// The sums over spans make one pass over the vocabulary do: a span's exponentials
// are relative to its own largest, as a row's is not known yet, and take the row's
// scale when dz is formed.  Powers of two, because a largest z times log2 e would be
// rounded, the same way for all of a span, which a logit of 1000 shows in the loss.
#include <math.h>

#include <atomic>

#include "ark_act.hpp"
#include "ark_common.hpp"
#include "ark_head.h"
#include "ark_product.hpp"

namespace {

using namespace ark::dev;
using ark::fail;

constexpr uint32_t kLanes = 256;
constexpr uint32_t kRowPad = 256;   // rows of a piece are laid out for whole tiles
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr uint32_t kMaxPiece = 16384;  // tokens: what rank_kernel's block ranks
constexpr uint32_t kFew = 1024;  // tokens that gather_kernel's blocks rank themselves

// Calls of at most this many tokens form dz in two 16-bit parts, its rounded value and what
// is left of it, in rows of their own: X's rows come twice for dw, and join_kernel adds dx's
// two.  Where tokens are few a rounding of dz shows in full in dx and dw (one token's entry
// at its target is nearly all of a row of W's gradient): up to 2.2 times the error of their
// own rounding for one token, 1.55 for 56, 1.4 to 1.5 for more, and 1.0 in two parts.  It takes
// a call of up to 32 tokens 0 to 8 % longer (768 x 32000: 54 us and 57 for one token, 57 and
// 61 for 32), as its rows still fit a tile, of 64 6 to 17 % (60 and 70), of 128 28 %.
constexpr uint32_t kTwice = 64;
static_assert(kTwice <= kFew && kTwice % kProductStep == 0 && 2 * kTwice <= kRowPad,
              "ranked by gather_kernel, and room for the rows of both parts");

// What a piece's kernels leave for each other.
struct Meta {
  uint32_t live;                  // rows with a loss
  uint32_t dx_parts, dw_parts;    // that the products' sums are cut into
  uint32_t dw_first;              // dw's blocks are the longer ones
  uint32_t again;                 // rows from dz's first part to its second, or 0
  float largest, to, down;        // grad * scale = grad / largest * to * down; the products
                                  // take dz without down
};

// How both products' work is cut, decided where the number of live rows is known:
// a tile's sum whole, or in parts that join_kernel adds.  Blocks of both are in one
// launch, the longer ones first, so that the shorter ones fill what those leave.
struct Cut {
  uint32_t tiles_m, bn, units;       // tiles across, rows of a tile, blocks that run at once
  float step, part, row;             // microseconds: a step of 32 k, a block besides, a row of
                                     // partial sums out and back
  uint32_t vocab, has_dx, has_dw;
  uint32_t dx_most, dw_most;         // parts times tiles down that have room

  struct Parts {
    uint32_t dx, dw;
  };
  // Candidate i of 64.
  static __host__ __device__ Parts candidate(uint32_t i) {
    const uint64_t dx = 0x18100C0804030201ull, dw = 0x4020100804030201ull;
    return {(uint32_t)(dx >> (i % 8 * 8)) & 255u, (uint32_t)(dw >> (i / 8 * 8)) & 255u};
  }
  __host__ __device__ uint32_t tiles_of(uint32_t rows) const { return (rows + bn - 1) / bn; }
  static __host__ __device__ uint32_t steps_of(uint32_t k) {
    return (k + kProductStep - 1) / kProductStep;
  }
  __host__ __device__ float length(uint32_t k, uint32_t parts) const {
    return (float)((steps_of(k) + parts - 1) / parts) * step + part;
  }
  // When the last of n1 blocks of length l1 and then n2 of l2 <= l1 ends.
  __host__ __device__ float end(uint32_t n1, float l1, uint32_t n2, float l2) const {
    const uint32_t q = n1 / units, r = n1 % units, left = units - r;
    const float a = (float)q * l1, b = r ? a + l1 : a;
    if (!n2) return b;
    // those that start at a end turns after it, or the others turns after b
    const uint32_t later = (uint32_t)ceilf(l1 / l2), sooner = (uint32_t)(l1 / l2);
    uint32_t k = (n2 + left - 1) / left;
    if (r && k > later) k = (n2 + r * later + units - 1) / units;
    float t = a + (float)k * l2;
    if (r) {
      const uint32_t m = n2 > left * sooner ? (n2 - left * sooner + units - 1) / units : 0;
      t = fmaxf(fminf(t, b + (float)m * l2), b);
    }
    return t;
  }
  __host__ __device__ float cost(Parts p, uint32_t live) const {
    const uint32_t n = has_dx ? tiles_m * tiles_of(live) * p.dx : 0;
    const uint32_t m = has_dw ? tiles_m * tiles_of(vocab) * p.dw : 0;
    const float ln = length(vocab, p.dx), lm = length(live, p.dw);
    float t = ln >= lm ? end(n, ln, m, lm) : end(m, lm, n, ln);
    if (has_dx && p.dx > 1) t += 3.0f + (float)(p.dx * live) * row;
    if (has_dw && p.dw > 1) t += 3.0f + (float)p.dw * (float)vocab * row;
    return t;
  }
  // A part has four steps at least.
  __host__ __device__ bool may(Parts p, uint32_t live) const {
    return (p.dx == 1 || (p.dx * 4 <= steps_of(vocab) && p.dx * tiles_of(live) <= dx_most)) &&
           (p.dw == 1 || (p.dw * 4 <= steps_of(live) && p.dw * tiles_of(vocab) <= dw_most));
  }
};

template <typename T>
constexpr uint32_t kTypeOf = sizeof(T) == 4 ? ARK_HEAD_F32 : ARK_HEAD_F16;
template <>
constexpr uint32_t kTypeOf<__bf16> = ARK_HEAD_BF16;

// An exponential from 0 to under 2, relative to its span's 2^t, in 16 bits without a sign:
// an exponent's low bits and what is left of them for the fraction, so that only dz's own
// rounding counts.  fp16 4 and 12 bits (2^-13 of itself, below 2^-14 2^-27: dz in fp16 has
// 2^-11 and, of the largest gradient, 2^-38), bf16 7 and 9 (2^-10, for 2^-8; its dz has
// small numbers too).  The bits are those of an fp32 times kDown, cut off at kCut.
template <typename T>
struct Kept {
  static constexpr uint32_t kCut = 11;
  static constexpr float kDown = 0x1p-112f, kUp = 0x1p112f;
};
template <>
struct Kept<__bf16> {
  static constexpr uint32_t kCut = 14;
  static constexpr float kDown = 1.0f, kUp = 1.0f;
};
// Two of them, to nearest; and back, times kDown.
template <typename T>
__device__ __forceinline__ uint32_t keep2(float a, float b) {
  typedef Kept<T> K;
  constexpr uint32_t kLeft = 16 - K::kCut, kHalf = 1u << 15;
  const uint32_t x = (__float_as_uint(a * K::kDown) << kLeft) + kHalf;
  const uint32_t y = (__float_as_uint(b * K::kDown) << kLeft) + kHalf;
  return __builtin_amdgcn_perm(y, x, 0x07060302u);
}
template <typename T>
__device__ __forceinline__ void kept2(uint32_t v, float& a, float& b) {
  typedef Kept<T> K;
  constexpr uint32_t kMask = 0xFFFFu << K::kCut;
  a = __uint_as_float((v << K::kCut) & kMask);
  b = __uint_as_float((v >> (16 - K::kCut)) & kMask);
}

// What two values' rounded ones leave, rounded.
template <typename T>
__device__ __forceinline__ uint32_t left2(float a, float b, uint32_t rounded) {
  typedef T V __attribute__((ext_vector_type(2)));
  const V r = __builtin_bit_cast(V, rounded);
  return narrow2<kTypeOf<T>>(a - (float)r[0], b - (float)r[1]);
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

__device__ __forceinline__ int64_t ld_int(const void* p, uint32_t bytes, uint64_t i) {
  return bytes == 8 ? ld_g<int64_t>((const int64_t*)p + i) : ld_g<int32_t>((const int32_t*)p + i);
}
__device__ __forceinline__ float ld_float(const void* p, uint32_t dtype, uint64_t i) {
  if (dtype == ARK_HEAD_F32) return ld_g<float>((const float*)p + i);
  const uint32_t h = ld_g<uint16_t>((const uint16_t*)p + i);
  return dtype == ARK_HEAD_BF16 ? __uint_as_float(h << 16) : h2f(h);
}

// Where a token's targets are: one each (cross entropy), or what teacher_kernel
// left of a teacher's entries.
struct Targets {
  const void* targets;  // NULL: a teacher's
  uint32_t bytes;
  int64_t ignore;
  const uint32_t* index;  // [tokens][top], ~0: left out
  const float* p;         // [tokens][top]
  const float* self;      // [tokens] sum of p log p
  const uint32_t* there;  // [tokens]
  uint32_t top, vocab;

  __device__ __forceinline__ bool is_target(int64_t y) const {
    return y != ignore && y >= 0 && y < (int64_t)vocab;
  }
  // Which of tokens t, t + step, ... (N of them, below n) have a loss; their loads all
  // together.
  template <uint32_t N>
  __device__ __forceinline__ void live(uint32_t t, uint32_t step, uint32_t n, bool (&out)[N]) const {
    if (!targets) {
      uint32_t v[N];
#pragma unroll
      for (uint32_t k = 0; k < N; ++k) v[k] = t + k * step < n ? ld_g<uint32_t>(there + t + k * step) : 0u;
#pragma unroll
      for (uint32_t k = 0; k < N; ++k) out[k] = v[k] != 0;
    } else if (bytes == 8) {
      int64_t v[N];
#pragma unroll
      for (uint32_t k = 0; k < N; ++k)
        v[k] = t + k * step < n ? ld_g<int64_t>((const int64_t*)targets + t + k * step) : -1;
#pragma unroll
      for (uint32_t k = 0; k < N; ++k) out[k] = is_target(v[k]);
    } else {
      int32_t v[N];
#pragma unroll
      for (uint32_t k = 0; k < N; ++k)
        v[k] = t + k * step < n ? ld_g<int32_t>((const int32_t*)targets + t + k * step) : -1;
#pragma unroll
      for (uint32_t k = 0; k < N; ++k) out[k] = is_target(v[k]);
    }
  }
  __device__ __forceinline__ uint32_t at(uint32_t t, uint32_t k) const {
    return targets ? (uint32_t)ld_int(targets, bytes, t) : ld_g<uint32_t>(index + (uint64_t)t * top + k);
  }
  __device__ __forceinline__ float weight(uint32_t t, uint32_t k) const {
    return targets ? 1.0f : ld_g<float>(p + (uint64_t)t * top + k);
  }
};

// Targets of live rows lie in rows of whole 16 bytes, ~0 where there is none, or one
// behind the other where a row has one.
__host__ __device__ inline uint32_t entries_width(uint32_t top) {
  return top == 1 ? 1 : (top + 3) / 4 * 4;
}

// A teacher's distribution, a wave a token.  Latency: 4096 tokens of 64 entries 5 us.
__global__ __launch_bounds__(kLanes) void teacher_kernel(
    const void* __restrict__ index, uint32_t index_bytes, uint64_t index_stride,
    const void* __restrict__ logits, uint32_t dtype, uint64_t logits_stride, uint32_t tokens,
    uint32_t top, uint32_t vocab, float scale, uint32_t* __restrict__ out, float* __restrict__ p,
    float* __restrict__ self, uint32_t* __restrict__ there) {
  const uint32_t t = blockIdx.x * (kLanes / 64) + threadIdx.x / 64, lane = threadIdx.x % 64;
  if (t >= tokens) return;
  constexpr uint32_t kEach = ARK_HEAD_MAX_TOP / 64;
  float a[kEach], most = -INFINITY;
  uint32_t id[kEach];
#pragma unroll
  for (uint32_t i = 0; i < kEach; ++i) {
    const uint32_t k = i * 64 + lane;
    id[i] = ~0u, a[i] = -INFINITY;
    if (k < top) {
      const int64_t v = ld_int(index, index_bytes, t * index_stride + k);
      const float l = ld_float(logits, dtype, t * logits_stride + k);
      if (v >= 0 && v < (int64_t)vocab && l != -INFINITY) id[i] = (uint32_t)v, a[i] = l;
    }
    most = fmaxf(most, a[i]);
  }
  most = wave_max(most);
  float sum = 0.0f;
  bool any = false;
#pragma unroll
  for (uint32_t i = 0; i < kEach; ++i)
    // the difference before the scale, with which a logit alone may pass fp32
    if (id[i] != ~0u) a[i] = (a[i] - most) * scale, sum += expf(a[i]), any = true;
  sum = wave_sum(sum);
  const float log_sum = logf(sum);
  float own = 0.0f;
#pragma unroll
  for (uint32_t i = 0; i < kEach; ++i) {
    const uint32_t k = i * 64 + lane;
    float q = 0.0f;
    if (id[i] != ~0u) {
      q = expf(a[i]) / sum;
      if (q != 0.0f) own += q * (a[i] - log_sum);
    }
    if (k < top) {
      out[(uint64_t)t * top + k] = id[i];
      p[(uint64_t)t * top + k] = q;
    }
  }
  own = wave_sum(own);
  const bool live = __ballot(any) != 0;
  if (lane == 0) self[t] = own, there[t] = live ? 1u : 0u;
}

struct RankArgs {
  Targets targets;
  uint32_t tokens;
  uint32_t* rank;      // [tokens]: a live token's row of X, ~0
  uint32_t* rows;      // and back
  Meta* meta;
  const float* grads;  // or NULL: grad
  float grad, scale;
  uint32_t with_grad;
  uint32_t twice;  // dz has two parts
  Cut cut;

  // Rows of X and dz up to a whole step.
  static __device__ __forceinline__ uint32_t whole(uint32_t rows) {
    return (rows + kProductStep - 1) / kProductStep * kProductStep;
  }
};

// By one wave, with the number of live tokens and the largest |grad| over them.
__device__ __forceinline__ void write_meta(const RankArgs& a, uint32_t live, float largest) {
  Meta m = {live, 1, 1, 0, 0, 1.0f, 1.0f, 1.0f};
  if (a.with_grad) {
    if (a.twice) m.again = live;
    const uint32_t rows = m.again + live;
    // grad * scale = f down, f = grad / largest * to: the largest f is 2^14, a power of two
    // so that the one number of all tokens has no rounding (which they would share), unless
    // down is then below fp32.  (By parts, as the product may lie below fp32 itself.)
    if (largest > 0.0f && largest * a.scale < INFINITY) {
      int eg, es;
      const float part = frexpf(largest, &eg) * frexpf(a.scale, &es);  // 1/4 to 1
      const int e = eg + es;
      m.largest = largest;
      m.to = e >= 14 - 124 ? 0x1p14f : ldexpf(part, e + 126);
      m.down = e >= 14 - 124 ? ldexpf(part, e - 14) : 0x1p-126f;
    }
    // the cheapest of the 64 candidates, a lane each
    const Cut::Parts mine = Cut::candidate(threadIdx.x % 64);
    const float cost = a.cut.may(mine, rows) ? a.cut.cost(mine, rows) : INFINITY;
    float best = cost;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) best = fminf(best, __shfl_xor(best, o));
    const Cut::Parts p =
        Cut::candidate((uint32_t)__ffsll((unsigned long long)__ballot(cost == best)) - 1u);
    m.dx_parts = p.dx, m.dw_parts = p.dw;
    m.dw_first = a.cut.length(rows, p.dw) > a.cut.length(a.cut.vocab, p.dx) ? 1 : 0;
  }
  if (threadIdx.x % 64 == 0) *a.meta = m;
}

// |grad| as a whole number; 0 where it or its product with scale is not finite: its own
// token's gradients are not finite at any scale, and the others keep theirs.
__device__ __forceinline__ uint32_t grad_size(const RankArgs& a, uint32_t t) {
  const float g = fabsf(a.grads[t]);
  return g * a.scale < INFINITY ? __float_as_uint(g) : 0u;
}
__device__ __forceinline__ uint32_t wave_max_bits(uint32_t g) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) g = max(g, (uint32_t)__shfl_xor(g, o));
  return g;
}

// The live tokens' order, by one block: 1024 tokens at a time side by side, their
// numbers of live ones summed in the tokens' order.  Latency of one block: 16384 tokens
// 10 us.
constexpr uint32_t kRankLanes = 1024, kRankWaves = kRankLanes / 64;
constexpr uint32_t kRankEach = kMaxPiece / kRankLanes;
__global__ __launch_bounds__(kRankLanes) void rank_kernel(RankArgs a) {
  __shared__ uint32_t s_count[kRankEach * kRankWaves + 1], s_most[kRankWaves];
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  uint64_t mask[kRankEach];
  uint32_t most = 0;
  bool live[kRankEach];
  a.targets.live<kRankEach>(threadIdx.x, kRankLanes, a.tokens, live);
#pragma unroll
  for (uint32_t k = 0; k < kRankEach; ++k) mask[k] = __ballot(live[k]);
  if (a.grads) {
#pragma unroll
    for (uint32_t k = 0; k < kRankEach; ++k) {
      const uint32_t t = k * kRankLanes + threadIdx.x;
      const uint32_t g = t < a.tokens ? grad_size(a, t) : 0u;
      most = max(most, live[k] ? g : 0u);
    }
  }
  most = wave_max_bits(most);
  if (lane == 0) {
#pragma unroll
    for (uint32_t k = 0; k < kRankEach; ++k) s_count[k * kRankWaves + wave] = __popcll(mask[k]);
    s_most[wave] = most;
  }
  __syncthreads();
  static_assert(kRankEach * kRankWaves == 256, "four counts a lane");
  uint32_t live_all = 0;
  if (wave == 0) {
    uint32_t c[4], sum = 0;
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) c[k] = s_count[4 * lane + k], sum += c[k];
    uint32_t incl = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t y = __shfl_up(incl, o);
      if (lane >= (uint32_t)o) incl += y;
    }
    uint32_t from = incl - sum;
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) s_count[4 * lane + k] = from, from += c[k];
    live_all = (uint32_t)__builtin_amdgcn_readlane(incl, 63);
  }
  __syncthreads();
#pragma unroll
  for (uint32_t k = 0; k < kRankEach; ++k) {
    const uint32_t t = k * kRankLanes + threadIdx.x;
    if (t >= a.tokens) break;
    const uint32_t row = s_count[k * kRankWaves + wave] + __popcll(mask[k] & ((1ull << lane) - 1));
    a.rank[t] = live[k] ? row : ~0u;
    if (live[k]) a.rows[row] = t;
  }
  if (wave == 0)
    write_meta(a, live_all, a.grads ? __uint_as_float(wave_max_bits(s_most[lane % kRankWaves]))
                                    : fabsf(a.grad));
}

struct GatherArgs {
  RankArgs rank;
  const uint16_t* x;
  uint64_t x_stride;
  uint32_t columns, padded;  // padded: columns of out
  uint16_t* out;
  float* loss;
  uint16_t* dx;  // or NULL
  uint64_t dx_stride;
  const uint16_t* w;  // as given
  uint64_t w_stride;
  uint32_t* entries;  // targets by rows
  uint16_t* w_out;    // w padded, or NULL
  uint32_t blocks;    // those after them pad w
};

// Eight neighbouring 16-bit values at any element's alignment (gfx950 takes
// unaligned global accesses), those past n as zeros.
__device__ __forceinline__ u32x4 load8(const uint16_t* p, uint32_t n) {
  typedef uint32_t V __attribute__((ext_vector_type(4), aligned(2)));
  if (n >= 8) return *(const ARK_GLOBAL V*)p;
  uint32_t v[8];
#pragma unroll
  for (uint32_t k = 0; k < 8; ++k) v[k] = k < n ? p[k] : 0u;
  return u32x4{v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16};
}

__device__ __forceinline__ void zero8(uint16_t* p, uint32_t n) {
  typedef uint32_t V __attribute__((ext_vector_type(4), aligned(2)));
  if (n >= 8) {
    *(ARK_GLOBAL V*)p = V{0, 0, 0, 0};
    return;
  }
#pragma unroll
  for (uint32_t k = 0; k < 8; ++k)
    if (k < n) p[k] = 0;
}

// W's rows padded to whole steps, where its own cannot be read 16 bytes at a time, a
// wave a row.
__device__ __forceinline__ void pad_rows(const GatherArgs& a) {
  const uint32_t lane = threadIdx.x % 64, step = (gridDim.x - a.blocks) * (kLanes / 64);
  for (uint32_t row = (blockIdx.x - a.blocks) * (kLanes / 64) + threadIdx.x / 64;
       row < a.rank.targets.vocab; row += step)
    for (uint32_t c = lane * 8; c < a.padded; c += 512)
      *(u32x4*)(a.w_out + (uint64_t)row * a.padded + c) =
          load8(a.w + row * a.w_stride + c, c < a.columns ? a.columns - c : 0u);
}

// A wave a token: its row of x, and its targets.  The waves past the last token fill X
// up to a whole step of the products, the blocks past those pad W.  Bound by HBM:
// 16384 rows of 2048, 134 MB out and back, 26 us; where W is padded by that too (333
// tokens, 5003 rows of 901, 18 MB: 7 us).
// FEW: at most 1024 tokens, which every block ranks for itself, without rank_kernel
// before (4096 that way: 19 us, with rank_kernel 16).
template <bool FEW>
__global__ __launch_bounds__(kLanes) void gather_kernel(GatherArgs a) {
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  if (blockIdx.x >= a.blocks) {
    pad_rows(a);
    return;
  }
  const uint32_t t = __builtin_amdgcn_readfirstlane(blockIdx.x * (kLanes / 64) + wave);
  const RankArgs& r = a.rank;
  uint32_t row = ~0u, live = 0;
  if constexpr (FEW) {
    constexpr uint32_t kEach = kFew / kLanes, kMasks = kFew / 64;
    __shared__ uint64_t s_mask[kMasks];
    __shared__ uint32_t s_most[kLanes / 64];
    bool mine[kEach];
    r.targets.live<kEach>(threadIdx.x, kLanes, r.tokens, mine);
#pragma unroll
    for (uint32_t k = 0; k < kEach; ++k) {
      const uint64_t m = __ballot(mine[k]);
      if (lane == 0) s_mask[k * (kLanes / 64) + wave] = m;
    }
    if (blockIdx.x == 0 && r.grads) {
      uint32_t most = 0;
#pragma unroll
      for (uint32_t k = 0; k < kEach; ++k)
        if (mine[k]) most = max(most, grad_size(r, k * kLanes + threadIdx.x));
      most = wave_max_bits(most);
      if (lane == 0) s_most[wave] = most;
    }
    __syncthreads();
    // the live tokens before each 64, a lane each
    const uint64_t m = s_mask[lane % kMasks];
    const uint32_t count = lane < kMasks ? __popcll(m) : 0u;
    uint32_t incl = count;
#pragma unroll
    for (int o = 1; o < (int)kMasks; o <<= 1) {
      const uint32_t y = __shfl_up(incl, o);
      if (lane >= (uint32_t)o) incl += y;
    }
    live = (uint32_t)__builtin_amdgcn_readlane(incl, kMasks - 1);
    if (t < r.tokens) {
      const uint64_t own = s_mask[t / 64];
      const uint32_t before = (uint32_t)__builtin_amdgcn_readlane(incl - count, t / 64);
      if (own >> (t % 64) & 1) row = before + __popcll(own & ((1ull << (t % 64)) - 1));
    }
    if (row != ~0u && lane == 0) r.rows[row] = t;
    if (t == 0)
      write_meta(r, live,
                 r.grads ? __uint_as_float(wave_max_bits(s_most[lane % (kLanes / 64)]))
                         : fabsf(r.grad));
  } else {
    row = t < r.tokens ? r.rank[t] : ~0u;
    live = r.meta->live;
  }
  const uint32_t again = r.twice ? live : 0;  // rows to X's second copy, or 0
  if (t >= r.tokens) {
    row = again + live + (t - r.tokens);
    if (row < RankArgs::whole(again + live))
      for (uint32_t c = lane * 8; c < a.padded; c += 512)
        *(u32x4*)(a.out + (uint64_t)row * a.padded + c) = u32x4{0, 0, 0, 0};
    return;
  }
  if (row == ~0u) {
    if (lane == 0) a.loss[t] = 0.0f;
    if (a.dx)
      for (uint32_t c = lane * 8; c < a.columns; c += 512)
        zero8(a.dx + t * a.dx_stride + c, a.columns - c);
    return;
  }
  const uint16_t* src = a.x + t * a.x_stride;
  uint16_t* dst = a.out + (uint64_t)row * a.padded;
  for (uint32_t c = lane * 8; c < a.padded; c += 512) {
    const u32x4 v = load8(src + c, c < a.columns ? a.columns - c : 0u);
    *(u32x4*)(dst + c) = v;
    if (again) *(u32x4*)(dst + (uint64_t)again * a.padded + c) = v;
  }
  const uint32_t top = r.targets.top, width = entries_width(top);
  for (uint32_t k = lane; k < width; k += 64)
    a.entries[(uint64_t)row * width + k] = k < top ? r.targets.at(t, k) : ~0u;
}

// The tile of a block: blocks of one XCD (every eighth) take neighbouring tiles,
// and these go through eight tiles of rows for every tile of columns, so that the
// operands of those that run together are few.  Only tiles that have live rows
// count (tiles left out in the middle would leave whole XCDs idle).
struct Tiles {
  uint32_t m, n;
  __device__ __forceinline__ void find(uint32_t block, uint32_t blocks, uint32_t* tm,
                                       uint32_t* tn, uint32_t* split) const {
    const uint32_t per = blocks / 8, rest = blocks % 8, xcd = block % 8;
    const uint32_t id = xcd * per + min(xcd, rest) + block / 8, tiles = m * n;
    *split = id / tiles;
    const uint32_t tile = id % tiles, group = tile / (8 * m);
    const uint32_t wide = min(n - group * 8, 8u), in = tile - group * 8 * m;
    *tm = in / wide;
    *tn = group * 8 + in % wide;
  }
};

struct LogitsArgs {
  const uint16_t *x, *w;
  uint64_t w_stride;
  uint32_t padded, vocab, spans;
  uint64_t e_stride;
  float scale;
  uint32_t tiles_m;
  const Meta* meta;
  float* stats;  // [row][span] of (t, sum of 2^(z log2 e - t)), t whole, next to the largest
  uint16_t* e;   // [row][e_stride], or NULL
  const uint32_t* entries;  // [row][entries_width(top)]
  uint32_t top;
  float* z;                 // [row][top]: the products there, before scale
};

// Whether a z log2 e lies where fp32 has whole numbers alone: its rounding is then no
// longer below the distance that an exponential takes, so what it is taken off is rounded
// the same way, and the largest is at distance 0.
__device__ __forceinline__ bool is_far(float z2) { return fabsf(z2) >= 0x1p23f && fabsf(z2) < INFINITY; }

// z of a tile of the vocabulary (m) and of rows of X (n), never in memory.  A lane holds
// MF x 4 logits of one row of X, a wave MF x 16, so a row's largest logit and sum over a
// wave's span are sums in registers and two exchanges, and the spans' join is left to the
// next kernel: nothing waits for another block.  Bound by the matrix units at the clock
// that power leaves them (1.95 GHz), a tile's 24 to 64 steps of 0.8 us and 6 us before and
// after them, in which the exponentials are the largest part: 12288 x 32000 x 768 fp16
// 673 us, 0.90 PFLOP/s; 16384 x 32000 x 2048 bf16 2.0 ms, 1.08 PFLOP/s.  8 rows: W's 49 MB
// go past in 12 us.
template <typename P>
__global__ __launch_bounds__(P::kLanes, 2) void logits_kernel(LogitsArgs a) {
  extern __shared__ __align__(1024) uint8_t lds[];
  uint32_t tm, tn, split;
  const uint32_t live = a.meta->live;
  const Tiles tiles = {a.tiles_m, (live + P::BN - 1) / P::BN};
  if (blockIdx.x >= tiles.m * tiles.n) return;
  tiles.find(blockIdx.x, tiles.m * tiles.n, &tm, &tn, &split);
  const uint32_t m0 = tm * P::BM, n0 = tn * P::BN;
  const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t w0 = m0 + wave % P::WM * 16 * P::MF;  // the wave's first of the vocabulary
  const uint32_t r0 = n0 + wave / P::WM * 16 * P::NF;  // and its first row
  uint32_t target = ~0u;  // lane i: of row r0 + i
  if (a.top == 1 && lane < 16 * P::NF && r0 + lane < live) target = a.entries[r0 + lane];
  P p;
  const Operand ow = {a.w + m0 * a.w_stride, a.w_stride, a.vocab - m0, 0};
  const Operand ox = {a.x + (uint64_t)n0 * a.padded, a.padded, P::BN, 0};
  p.run(ow, ox, 0, a.padded / kProductStep, (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds);
  const uint32_t span = tm * P::WM + wave % P::WM;
  if (m0 + P::BM > a.vocab) {
#pragma unroll
    for (uint32_t i = 0; i < P::MF; ++i)
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k)
        if (w0 + lane / 16 * 4 + i * 16 + k >= a.vocab) {
#pragma unroll
          for (uint32_t j = 0; j < P::NF; ++j) p.acc[i][j][k] = -INFINITY;
        }
  }
  // a lane's sixteen entries from k on, in four pieces, of one row
  const auto entries = [&](u32x4 (&v)[4], uint32_t row, uint32_t k) __attribute__((always_inline)) {
    const uint32_t width = entries_width(a.top);
#pragma unroll
    for (uint32_t q = 0; q < 4; ++q) {
      v[q] = u32x4{~0u, ~0u, ~0u, ~0u};
      if (k + q * 16 < width)
        v[q] = ld_g<u32x4>(a.entries + (uint64_t)row * width + k + q * 16);
    }
  };
  u32x4 begin[P::NF][4];  // those of every row's first 64, all on their way at once
  if (a.top > 1) {
#pragma unroll
    for (uint32_t j = 0; j < P::NF; ++j)
      entries(begin[j], min(r0 + j * 16 + lane / 4, live - 1), lane % 4 * 4);
  }
  __syncthreads();  // LDS is the epilogue's now
  // A wave's exponentials of 16 rows pass through LDS of its own, so that a row's
  // leave as whole lines: chunks of 16 bytes, permuted by the row against conflicts.
  constexpr uint32_t kRow = P::MF * 32, kChunks = kRow / 16;  // bytes of a row
  // Before them so do the logits of rows that may have a target in the wave's span (64
  // entries a token of 32000, looked for here: 4.5 us a tile, 256 x 256; gathered rows
  // of W times x: 55 us for 4096 tokens, of 16 tiles down and 8 rounds).
  constexpr uint32_t kZRow = P::MF * 64, kSpan = P::MF * 16;
  static_assert(16 * kZRow * P::WM * P::WN <= P::kLds, "a part of LDS for each wave");
  uint8_t* mine = lds + wave * 16 * kZRow;
  const float to2 = a.scale * kLog2e;
  const uint64_t hits = __ballot(target - w0 < kSpan);
#pragma unroll
  for (uint32_t j = 0; j < P::NF; ++j) {
    const uint32_t t0 = r0 + j * 16, t = t0 + lane % 16;
    if (a.top > 1 || hits >> (j * 16) & 0xFFFFu) {
#pragma unroll
      for (uint32_t i = 0; i < P::MF; ++i)
        *(f32x4*)(mine + lane % 16 * kZRow + ((i * 4 + lane / 16) ^ (lane % 16)) * 16) =
            p.acc[i][j];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      const auto z_at = [&](uint32_t row, uint32_t d) {
        return *(const float*)(mine + row * kZRow + ((d / 4) ^ row) * 16 + d % 4 * 4);
      };
      if (a.top == 1) {
        if (lane / 16 == j && target - w0 < kSpan) a.z[r0 + lane] = z_at(lane % 16, target - w0);
      } else if (t0 + lane / 4 < live) {
        const uint64_t row = t0 + lane / 4;
        const uint32_t width = entries_width(a.top);
        for (uint32_t k = lane % 4 * 4; k < width; k += 64) {
          u32x4 v[4];
          if (k < 16) {
#pragma unroll
            for (uint32_t q = 0; q < 4; ++q) v[q] = begin[j][q];
          } else {
            entries(v, (uint32_t)row, k);
          }
          // bits of those in the span, entry i in 1 << i; few
          uint32_t there = 0;
#pragma unroll
          for (uint32_t i = 0; i < 16; ++i) there |= v[i / 4][i % 4] - w0 < kSpan ? 1u << i : 0u;
          while (there) {
            const uint32_t i = (uint32_t)__ffs(there) - 1u;
            uint32_t d = 0;
#pragma unroll
            for (uint32_t h = 0; h < 16; ++h) d = h == i ? v[h / 4][h % 4] - w0 : d;
            a.z[row * a.top + k + i / 4 * 16 + i % 4] = z_at(lane / 4, d);
            there &= there - 1;
          }
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    float most = -INFINITY;
#pragma unroll
    for (uint32_t i = 0; i < P::MF; ++i)
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) most = fmaxf(most, p.acc[i][j][k]);
    most = fmaxf(most, __shfl_xor(most, 16));
    most = fmaxf(most, __shfl_xor(most, 32));
    // a whole power of two: no rounding of its own, which all of the span would share
    const float top = most == -INFINITY ? most : rintf(most * to2);
    float mul = to2, from = most == -INFINITY ? 0.0f : -top;
    if (is_far(top)) {
      mul = 1.0f, from = 0.0f;
#pragma unroll
      for (uint32_t i = 0; i < P::MF; ++i)
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) p.acc[i][j][k] = p.acc[i][j][k] * to2 - top;
    }
    float sum = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < P::MF; ++i)
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) {
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(p.acc[i][j][k], mul, from));
        p.acc[i][j][k] = e;
        sum += e;
      }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (lane < 16 && t < live) {
      float* s = a.stats + ((uint64_t)t * a.spans + span) * 2;
      s[0] = top, s[1] = sum;
    }
    if (!a.e) continue;
    const uint32_t row = lane % 16;
#pragma unroll
    for (uint32_t i = 0; i < P::MF; ++i) {
      const f32x4 v = p.acc[i][j];
      const uint32_t chunk = (i * 2 + lane / 32) ^ (row % kChunks);
      *(u32x2*)(mine + row * kRow + chunk * 16 + lane / 16 % 2 * 8) =
          u32x2{keep2<typename P::T>(v[0], v[1]), keep2<typename P::T>(v[2], v[3])};
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (uint32_t i = 0; i < kRow / 64; ++i) {
      const uint32_t q = i * 64 + lane, r = q / kChunks, c = q % kChunks;
      const u32x4 v = *(const u32x4*)(mine + r * kRow + (c ^ (r % kChunks)) * 16);
      if (t0 + r < live) st_nt<u32x4>(a.e + (t0 + r) * a.e_stride + w0 + c * 8, v);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// The sum of a row's exponentials.
struct RowSum {
  float top, log;  // log2 of it is top + log; top is whole, so that what is near it stays exact
  // log2 of the probability at a product x . w
  __device__ __forceinline__ float log2_q(float product, float to2) const {
    return (is_far(top) ? product * to2 - top : __builtin_fmaf(product, to2, -top)) - log;
  }
};

// It from its spans' (t, sum), by `LANES` lanes of a block (a wave or all of it; red: two
// values a wave).  One pass, eight spans a lane on their way at once.  Spans' t are
// whole, so that their sums join without rounding but the sum's own.
template <uint32_t LANES>
__device__ __forceinline__ RowSum join_spans(const float* stats, uint32_t spans, uint32_t lane,
                                             float* red) {
  typedef float V __attribute__((ext_vector_type(2)));
  constexpr uint32_t kEach = 8;
  float most = -INFINITY, sum = 0.0f;
  const auto join = [](float& m, float& s, float m2, float s2) {
    // a NaN among the sums stays; -inf on both sides has no distance
    const float top = fmaxf(m, m2);
    s = s * (m == top ? 1.0f : exp2f(m - top)) + s2 * (m2 == top ? 1.0f : exp2f(m2 - top));
    m = top;
  };
  for (uint32_t i0 = lane; i0 < spans; i0 += LANES * kEach) {
    V v[kEach];
#pragma unroll
    for (uint32_t k = 0; k < kEach; ++k) {
      const uint32_t i = i0 + k * LANES;
      v[k] = i < spans ? ld_g<V>(stats + 2 * i) : V{-INFINITY, 0.0f};
    }
    float m = most;
#pragma unroll
    for (uint32_t k = 0; k < kEach; ++k) m = fmaxf(m, v[k].x);
    sum *= most == m ? 1.0f : exp2f(most - m);
    most = m;
#pragma unroll
    for (uint32_t k = 0; k < kEach; ++k) sum += v[k].y * (v[k].x == m ? 1.0f : exp2f(v[k].x - m));
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) join(most, sum, __shfl_xor(most, o), __shfl_xor(sum, o));
  if constexpr (LANES > 64) {
    if (lane % 64 == 0) red[lane / 64 * 2] = most, red[lane / 64 * 2 + 1] = sum;
    __syncthreads();
    most = red[0], sum = red[1];
    for (uint32_t w = 1; w < LANES / 64; ++w) join(most, sum, red[2 * w], red[2 * w + 1]);
  }
  return {most, log2f(sum)};
}

// A token's loss: sum of p (log p - log q), by a wave.
__device__ __forceinline__ float row_loss(const Targets& g, uint32_t t, const float* z,
                                          const RowSum& sum, float to2, uint32_t lane) {
  float s = 0.0f;
  for (uint32_t k = lane; k < g.top; k += 64) {
    const float p = g.weight(t, k);
    if (p != 0.0f) s -= p * sum.log2_q(z[k], to2);
  }
  s = wave_sum(s) * kLn2;
  return g.targets ? s : s + g.self[t];
}

struct LossArgs {
  Targets targets;
  const uint32_t* rows;
  const Meta* meta;
  const float* stats;
  uint32_t spans;
  const float* z;
  float* loss;
  float scale;
};

// The loss alone, a wave a row.  Latency: 4099 rows of 250 spans 6 us.
__global__ __launch_bounds__(kLanes) void loss_kernel(LossArgs a) {
  const uint32_t row = blockIdx.x * (kLanes / 64) + threadIdx.x / 64, lane = threadIdx.x % 64;
  if (row >= a.meta->live) return;
  const uint32_t t = a.rows[row];
  const RowSum sum = join_spans<64>(a.stats + (uint64_t)row * a.spans * 2, a.spans, lane, nullptr);
  const float loss =
      row_loss(a.targets, t, a.z + (uint64_t)row * a.targets.top, sum, a.scale * kLog2e, lane);
  if (lane == 0) a.loss[t] = loss;
}

struct DzArgs {
  LossArgs loss;
  const float* grads;  // or NULL
  float grad;
  uint16_t* e;
  uint64_t e_stride;
  uint32_t written;  // columns that hold something
  uint32_t span;   // values a span covers
  uint32_t share;  // of a row, that a block takes: whole rounds of its lanes
};

// A row's exponentials to dz, by a block (or with few rows by several, each of which
// joins the spans for itself); rows past the live ones, up to a whole step of the
// products, to zeros.  Bound by HBM: 12288 rows of 32000, 1.57 GB, 276 us, 5.7 TB/s.
// LANES: a block's, or a wave's where a row is no more than a block's one round (6039
// rows of 377: 10 us, 18 by blocks; 738 of 1936: 7.9 both ways).
template <typename T, uint32_t LANES>
__global__ __launch_bounds__(kLanes) void dz_kernel(DzArgs a) {
  constexpr uint32_t DT = kTypeOf<T>, kTeams = kLanes / LANES;
  __shared__ float red[kLanes / 64 * 2];
  __shared__ uint32_t s_index_of[kTeams][ARK_HEAD_MAX_TOP];
  __shared__ float s_p_of[kTeams][ARK_HEAD_MAX_TOP];
  const LossArgs& l = a.loss;
  const uint32_t team = threadIdx.x / LANES, tid = threadIdx.x % LANES;
  const uint32_t row = blockIdx.x * kTeams + team, live = l.meta->live;
  uint32_t* const s_index = s_index_of[team];
  float* const s_p = s_p_of[team];
  const uint32_t second = l.meta->again;  // rows to dz's second part, or 0
  if (second + row >= RankArgs::whole(second + live)) return;
  uint16_t* e = a.e + row * a.e_stride;
  const uint64_t again = second * a.e_stride;
  const uint32_t from = blockIdx.y * a.share, to = min(from + a.share, a.written);
  if (row >= live) {
    for (uint32_t c = from + tid * 8; c < to; c += LANES * 8)
      *(u32x4*)(e + again + c) = u32x4{0, 0, 0, 0};
    return;
  }
  const uint32_t t = l.rows[row], top = l.targets.top;
  const float* stats = l.stats + (uint64_t)row * l.spans * 2;
  const float* z = l.z + (uint64_t)row * top;
  // four rounds of the lanes on their way, the first four while the spans join
  constexpr uint32_t kAhead = 4, kRound = LANES * 8;
  u32x4 v[kAhead];
  const auto fetch = [&](uint32_t c) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t q = 0; q < kAhead; ++q)
      if (c + q * kRound < to) v[q] = ld_nt<u32x4>(e + c + q * kRound);
  };
  fetch(from + tid * 8);
  const RowSum sum = join_spans<LANES>(stats, l.spans, tid, red);
  const float to2 = l.scale * kLog2e;
  if (tid < 64 && blockIdx.y == 0) {
    const float loss = row_loss(l.targets, t, z, sum, to2, tid);
    if (tid == 0) l.loss[t] = loss;
  }
  const float g = a.grads ? a.grads[t] : a.grad;
  const float f = fabsf(g) * l.scale < INFINITY ? g / l.meta->largest * l.meta->to : g * l.scale;
  for (uint32_t k = tid; k < top; k += LANES) {
    s_index[k] = l.targets.at(t, k);
    s_p[k] = l.targets.weight(t, k);
  }
  for (uint32_t c0 = from + tid * 8; c0 < to; c0 += kAhead * kRound) {
#pragma unroll
    for (uint32_t q = 0; q < kAhead; ++q) {
      const uint32_t c = c0 + q * kRound;
      if (c >= to) break;
      const float s = exp2f((stats[c / a.span * 2] - sum.top) - sum.log) * f * Kept<T>::kUp;
      u32x4 o;
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        float x, y;
        kept2<T>(v[q][i], x, y);
        o[i] = narrow2<DT>(x * s, y * s);
      }
      *(u32x4*)(e + c) = o;
      if (again) {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
          float x, y;
          kept2<T>(v[q][i], x, y);
          o[i] = left2<T>(x * s, y * s, o[i]);
        }
        *(u32x4*)(e + again + c) = o;
      }
    }
    fetch(c0 + kAhead * kRound);
  }
  if constexpr (LANES > 64)
    __syncthreads();
  else
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
  // the targets' own entries, from fp32 (an index that comes twice writes the same
  // value twice)
  for (uint32_t k = tid; k < top; k += LANES) {
    const uint32_t v = s_index[k];
    if (v < from || v >= to) continue;  // another block's, or left out
    float p = 0.0f;
    for (uint32_t i = 0; i < top; ++i) p += s_index[i] == v ? s_p[i] : 0.0f;
    // q - p without the difference of two numbers near 1
    const float d = (expm1f(sum.log2_q(z[k], to2) * kLn2) + (1.0f - p)) * f;
    const uint32_t o = narrow2<DT>(d, 0.0f);
    e[v] = (uint16_t)o;
    if (again) e[again + v] = (uint16_t)left2<T>(d, 0.0f, o);
  }
}

// Where a product goes.
struct Out {
  void* p;         // fp32 or 16 bits
  uint64_t stride;
  uint32_t dtype;
  const float* add;         // fp32 to add, of `add_stride`, or NULL
  uint64_t add_stride;
  const uint32_t* rows;     // row n goes to rows[n], or NULL
  uint32_t width, height;   // m and n that are stored
  const Meta* meta;

  // Four values at any element's alignment.
  __device__ __forceinline__ void put(uint32_t n, uint32_t m, f32x4 v) const {
    typedef float V4 __attribute__((ext_vector_type(4), aligned(4)));
    typedef uint32_t V2 __attribute__((ext_vector_type(2), aligned(2)));
    v *= meta->down;
    const uint64_t row = rows ? rows[n] : n;
    const uint32_t c = min(width - m, 4u);
    if (add) {
      const float* q = add + row * add_stride + m;
      if (c == 4) {
        v += *(const ARK_GLOBAL V4*)q;
      } else {
#pragma unroll
        for (uint32_t k = 0; k < 3; ++k)
          if (k < c) v[k] += q[k];
      }
    }
    if (dtype == ARK_HEAD_F32) {
      float* q = (float*)p + row * stride + m;
      if (c == 4) {
        *(ARK_GLOBAL V4*)q = v;
        return;
      }
#pragma unroll
      for (uint32_t k = 0; k < 3; ++k)
        if (k < c) q[k] = v[k];
      return;
    }
    const u32x2 h = dtype == ARK_HEAD_F16
                        ? u32x2{narrow2<ARK_ACT_F16>(v[0], v[1]), narrow2<ARK_ACT_F16>(v[2], v[3])}
                        : u32x2{narrow2<ARK_ACT_BF16>(v[0], v[1]), narrow2<ARK_ACT_BF16>(v[2], v[3])};
    uint16_t* q = (uint16_t*)p + row * stride + m;
    if (c == 4) {
      *(ARK_GLOBAL V2*)q = h;
      return;
    }
#pragma unroll
    for (uint32_t k = 0; k < 3; ++k)
      if (k < c) q[k] = (uint16_t)(h[k / 2] >> (k % 2 * 16));
  }
};

// dx (DX: a = W across its rows, b = dz along them) or dw (a = X, b = dz, both
// across).
struct ProductArgs {
  const uint16_t *a, *b;
  uint64_t a_stride, b_stride;
  uint32_t a_width;   // values of a row of a
  uint32_t b_width;   // dw: of a row of b
  uint32_t a_rows;    // dx: rows of W
  float* partial;     // [part][rows][width up to 4]
  Out out;            // p NULL: not formed
};
struct GradArgs {
  ProductArgs dx, dw;
  uint32_t tiles_m;
  const Meta* meta;
};

// One block of dx or dw: `block` of the blocks of its kind.
template <typename P, bool DX>
__device__ __forceinline__ void product_block(const ProductArgs& g, const Meta& meta,
                                              const Tiles& tiles, uint32_t block, uint8_t* lds) {
  const uint32_t parts = DX ? meta.dx_parts : meta.dw_parts;
  const uint32_t height = DX ? meta.again + meta.live : g.out.height;
  uint32_t tm, tn, part;
  tiles.find(block, tiles.m * tiles.n * parts, &tm, &tn, &part);
  const uint32_t m0 = tm * P::BM, n0 = tn * P::BN;
  const uint32_t ks = DX ? g.a_rows : RankArgs::whole(meta.again + meta.live);
  const uint32_t steps = (ks + kProductStep - 1) / kProductStep;
  const uint32_t s0 = (uint32_t)((uint64_t)steps * part / parts);
  const uint32_t s1 = (uint32_t)((uint64_t)steps * (part + 1) / parts);
  P p;
  const Operand oa = {g.a + m0, g.a_stride, g.a_width - m0, ks};
  const Operand ob = DX ? Operand{g.b + n0 * g.b_stride, g.b_stride, P::BN, 0}
                        : Operand{g.b + n0, g.b_stride, g.b_width - n0, ks};
  const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
  p.run(oa, ob, s0, s1, at);
  const uint64_t w4 = (g.out.width + 3) / 4 * 4;
  float* partial = g.partial + (uint64_t)part * height * w4;
  p.each(at, [&](uint32_t m, uint32_t n, f32x4 v) __attribute__((always_inline)) {
    m += m0, n += n0;
    if (m >= g.out.width || n >= height) return;
    if (parts > 1 || (DX && meta.again))
      *(f32x4*)(partial + n * w4 + m) = v;
    else
      g.out.put(n, m, v);
  });
}

// dx and dw in one launch, the longer blocks first (write_meta), so that the shorter ones
// fill the units that those leave (12288 x 32000 x 768: 7 % of the call less than with a
// launch each).  Bound as the logits are: 12288 x 32000 x 768 fp16 1.11 ms, 1.09 PFLOP/s;
// 16384 x 32000 x 2048 bf16 3.55 ms, 1.21 PFLOP/s, where a library product of 8192^3
// reaches 1.29 and 1.35.  (A rate of 1.94 is what these matrix instructions reach from
// registers alone; 32 x 32 x 16 ones reach 1.71.)
template <typename X, typename W>
__global__ __launch_bounds__(X::kLanes, 2) void grad_kernel(GradArgs g) {
  extern __shared__ __align__(1024) uint8_t lds[];
  const Meta meta = *g.meta;
  const Tiles x = {g.tiles_m, g.dx.out.p ? (meta.again + meta.live + X::BN - 1) / X::BN : 0u};
  const Tiles w = {g.tiles_m, g.dw.out.p ? (g.dw.out.height + W::BN - 1) / W::BN : 0u};
  const uint32_t nx = x.m * x.n * meta.dx_parts, nw = w.m * w.n * meta.dw_parts;
  // the second kind starts at a multiple of the XCDs
  const uint32_t first = meta.dw_first ? nw : nx, up = (first + 7) / 8 * 8;
  const bool second = blockIdx.x >= up;
  const uint32_t block = second ? blockIdx.x - up : blockIdx.x;
  if ((meta.dw_first != 0) != second) {
    if (block < nw) product_block<W, false>(g.dw, meta, w, block, lds);
  } else {
    if (block < nx) product_block<X, true>(g.dx, meta, x, block, lds);
  }
}

// The parts of both products, added in order, and then those of the rows `again` further on.
// Bound by the caches that the parts are still in: dw's two of 32000 x 768, 18 us.
template <uint32_t kBatch>  // on their way at once
__device__ __forceinline__ void join(const float* partial, uint32_t parts, uint32_t height,
                                     uint32_t again, const Out& out, uint64_t i, uint64_t step) {
  const uint32_t per = (out.width + 3) / 4;
  const uint64_t rows = (uint64_t)height * per, second = (uint64_t)again * per;
  const uint64_t all = second + rows;
  const uint32_t sums = again ? 2 * parts : parts;
  for (; i < rows; i += step) {
    const f32x4* p = (const f32x4*)partial + i;
    const auto at = [&](uint32_t s) { return s < parts ? s * all : (s - parts) * all + second; };
    f32x4 v = p[0];
    for (uint32_t s = 1; s < sums; s += kBatch) {
      f32x4 more[kBatch];
#pragma unroll
      for (uint32_t k = 0; k < kBatch; ++k)
        if (s + k < sums) more[k] = p[at(s + k)];
#pragma unroll
      for (uint32_t k = 0; k < kBatch; ++k)
        if (s + k < sums) v += more[k];
    }
    out.put((uint32_t)(i / per), (uint32_t)(i % per) * 4, v);
  }
}
// TWICE: dx's rows may come twice, whose longer chains have more parts on their way (for all
// calls dw's two take 23 us for 19, for their registers).
template <bool TWICE>
__global__ __launch_bounds__(kLanes) void join_kernel(GradArgs g) {
  constexpr uint32_t kBatch = TWICE ? 8 : 4;
  const Meta meta = *g.meta;
  const uint32_t again = TWICE ? meta.again : 0;
  const uint64_t i = (uint64_t)blockIdx.x * kLanes + threadIdx.x, step = (uint64_t)gridDim.x * kLanes;
  if (g.dx.out.p && (meta.dx_parts > 1 || again))
    join<kBatch>(g.dx.partial, meta.dx_parts, meta.live, again, g.dx.out, i, step);
  if (g.dw.out.p && meta.dw_parts > 1)
    join<kBatch>(g.dw.partial, meta.dw_parts, g.dw.out.height, 0, g.dw.out, i, step);
}

// ---- host -------------------------------------------------------------------

constexpr uint64_t kPieceBytes = 1ull << 30;  // of a piece's dz, or of its spans' sums, at most

struct Big {
  template <typename T, bool AMC, bool BMC>
  using P = Product<T, AMC, BMC, 8, 4, 2, 4, 4>;
};
struct Small {
  template <typename T, bool AMC, bool BMC>
  using P = Product<T, AMC, BMC, 4, 2, 2, 2, 4>;
};

// How a call is cut, and where things lie in its workspace (offsets of 256).
struct Plan {
  bool small_logits, small;     // tiles
  bool twice;                   // dz in two parts
  uint32_t piece;               // tokens
  uint32_t pieces;
  uint32_t padded;              // columns
  bool copy_w;
  uint32_t span, spans, written;  // written: columns of dz that hold something
  uint64_t e_stride;
  Cut cut;
  uint64_t meta, rank, rows, index, p, self, there, entries, z, x, w, stats, e, dx_parts, dw_parts, sums, bytes;
};

uint64_t up(uint64_t n, uint64_t to) { return (n + to - 1) / to * to; }

// The cut of a piece of `rows` tokens, with room for the parts that it asks for with
// every token live, and for some more of dx's when few are.  *best: what it costs.
Cut cut_of(bool small, uint32_t columns, uint32_t rows, uint32_t vocab, bool has_dx, bool has_dw,
           float* best_cost) {
  Cut c = {};
  // measured on MI355X: a large tile has a unit to itself, of small ones three share it;
  // partial sums go out and come back at 5 TB/s
  c.tiles_m = small ? (columns + 127) / 128 : (columns + 255) / 256;
  c.bn = small ? 64 : 256;
  c.units = small ? 768 : 256;
  c.step = small ? 0.59f : 0.85f;
  c.part = small ? 4.0f : 8.0f;
  c.row = (float)up(columns, 4) * 8.0f / 5e6f;
  c.vocab = vocab, c.has_dx = has_dx, c.has_dw = has_dw;
  c.dx_most = c.dw_most = ~0u;
  Cut::Parts best = Cut::candidate(0);
  float cost = c.cost(best, rows);
  for (uint32_t i = 1; i < 64; ++i) {
    const Cut::Parts p = Cut::candidate(i);
    if (!c.may(p, rows)) continue;
    const float t = c.cost(p, rows);
    if (t < cost) best = p, cost = t;
  }
  const uint32_t n = c.tiles_of(rows), some = (512 + c.tiles_m - 1) / c.tiles_m;
  c.dx_most = best.dx * n;
  if (c.dx_most < some) c.dx_most = some < 24 * n ? some : 24 * n;
  c.dw_most = best.dw * c.tiles_of(vocab);
  *best_cost = cost;
  return c;
}

// What the logits cost, in microseconds: large tiles one a unit; small ones three a
// unit, whose steps take 0.32 alone and 0.59 when three share it.  Measured: 300 rows,
// 5003 x 901: 26 with large tiles, 12 with small ones; 517, 32308 x 768: 29 and 52.
float logits_cost(bool small, uint64_t rows, uint64_t vocab, uint32_t padded) {
  const float steps = (float)(padded / kProductStep);
  if (!small) {
    const uint64_t tiles = (up(vocab, 256) / 256) * (up(rows, 256) / 256);
    return (float)((tiles + 255) / 256) * (steps * 0.8f + 6.0f);
  }
  const uint64_t tiles = (up(vocab, 128) / 128) * (up(rows, 64) / 64);
  float t = (float)(tiles / 768) * (steps * 0.59f + 3.0f);
  if (tiles % 768) t += steps * (0.18f + 0.137f * (float)((tiles % 768 + 255) / 256)) + 3.0f;
  return t;
}

Plan plan_of(const void* w, uint64_t w_stride, uint64_t tokens, uint64_t columns, uint64_t vocab,
             uint64_t top, uint32_t dw_dtype, bool grad, bool has_dx, bool has_dw) {
  Plan p = {};
  p.e_stride = up(vocab, 256);
  p.padded = (uint32_t)up(columns, kProductStep);
  p.copy_w = columns % kProductStep || w_stride % 8 || (uintptr_t)w % 16;
  // pieces of equal sizes, whole tiles, bounded by what a token's row takes: dz, or for the
  // loss alone its spans' sums (of the narrower spans)
  const uint64_t row = grad ? p.e_stride * 2 : p.e_stride / 64 * 8;
  uint64_t most = kPieceBytes / row / kRowPad * kRowPad;
  if (most < kRowPad) most = kRowPad;
  if (most > kMaxPiece) most = kMaxPiece;
  p.pieces = (uint32_t)((tokens + most - 1) / most);
  if (p.pieces == 0) p.pieces = 1;
  p.piece = (uint32_t)(p.pieces == 1 ? tokens : up((tokens + p.pieces - 1) / p.pieces, kRowPad));
  const uint32_t piece = p.piece ? p.piece : 1;
  const uint64_t rows = up(piece, kRowPad);
  p.small_logits = logits_cost(true, piece, vocab, p.padded) <
                   logits_cost(false, piece, vocab, p.padded);
  p.span = p.small_logits ? 64 : 128;
  p.written = (uint32_t)up(vocab, 2 * p.span);
  p.spans = p.written / p.span;
  uint64_t at = 0;
  const auto take = [&](uint64_t bytes) {
    const uint64_t here = at;
    at += up(bytes, 256);
    return here;
  };
  p.meta = take(sizeof(Meta));
  p.rank = take(rows * 4);
  p.rows = take(rows * 4);
  p.index = take(rows * top * 4);
  p.p = take(rows * top * 4);
  p.self = take(rows * 4);
  p.there = take(rows * 4);
  p.entries = take(rows * entries_width((uint32_t)top) * 4);
  p.z = take(rows * top * 4);
  p.x = take(rows * p.padded * 2);
  p.w = take(p.copy_w ? vocab * p.padded * 2 : 0);
  p.stats = take(rows * p.spans * 8);
  if (grad) {
    p.e = take(rows * p.e_stride * 2);
    float large, small = INFINITY;
    p.twice = tokens <= kTwice;
    const uint32_t dz_rows = p.twice ? piece * 2 : piece;
    p.cut = cut_of(false, (uint32_t)columns, dz_rows, (uint32_t)vocab, has_dx, has_dw, &large);
    if (large < 500.0f) {  // beyond it small tiles have no chance
      const Cut c = cut_of(true, (uint32_t)columns, dz_rows, (uint32_t)vocab, has_dx, has_dw, &small);
      p.small = small < large;
      if (p.small) p.cut = c;
    }
    const uint64_t tile = up(columns, 4) * 4 * p.cut.bn;
    p.dx_parts = take(has_dx ? p.cut.dx_most * tile : 0);
    p.dw_parts = take(has_dw && p.cut.dw_most > p.cut.tiles_of((uint32_t)vocab)
                          ? p.cut.dw_most * tile : 0);
    p.sums = take(dw_dtype != ARK_HEAD_F32 && p.pieces > 1 ? vocab * columns * 4 : 0);
  }
  p.bytes = at;
  return p;
}

struct Call {
  const void* x;
  uint64_t x_stride;
  const void* w;
  uint64_t w_stride;
  uint32_t dtype;
  uint64_t tokens, columns, vocab;
  const void* targets;  // NULL: a teacher's entries
  uint32_t target_bytes;
  int64_t ignore;
  const void* index;
  uint32_t index_bytes;
  uint64_t index_stride;
  const void* logits;
  uint32_t logits_dtype;
  uint64_t logits_stride, top;
  float scale;
  bool with_grad;
  float grad;
  const float* grads;
  float* loss;
  void* dx;
  uint64_t dx_stride;
  void* dw;
  uint32_t dw_dtype;
  uint64_t dw_stride;
  uint32_t flags;
  char* ws;
  uint64_t ws_bytes;
  hipStream_t stream;
  bool teacher;
};

template <typename K>
int with_lds(K kernel, uint32_t bytes, std::atomic<uint64_t>* ready) {
  int dev = 0;
  ARK_HIP(hipGetDevice(&dev));
  if (dev >= 64 || !(ready->load(std::memory_order_relaxed) >> dev & 1u)) {
    ARK_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                                (int)bytes));
    if (dev < 64) ready->fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  return ARK_OPT_OK;
}

template <typename P>
int launch_logits(const LogitsArgs& a, uint32_t blocks, hipStream_t s) {
  static std::atomic<uint64_t> ready{0};
  if (int rc = with_lds(logits_kernel<P>, P::kLds, &ready)) return rc;
  hipLaunchKernelGGL(logits_kernel<P>, dim3(blocks), dim3(P::kLanes), P::kLds, s, a);
  ARK_HIP(hipGetLastError());
  return ARK_OPT_OK;
}

template <typename X, typename W>
int launch_grad(const GradArgs& g, const Cut& cut, bool twice, uint32_t tokens, hipStream_t s) {
  static std::atomic<uint64_t> ready{0};
  static_assert(X::kLanes == W::kLanes && X::kLds == W::kLds && X::BN == W::BN, "one launch");
  if (int rc = with_lds(grad_kernel<X, W>, X::kLds, &ready)) return rc;
  // as many blocks as any number of live rows may ask for; the others leave at once
  const uint32_t rows = twice ? tokens * 2 : tokens;
  uint32_t nx = 0, nw = 0;
  if (g.dx.out.p) nx = cut.dx_most > cut.tiles_of(rows) ? cut.dx_most : cut.tiles_of(rows);
  if (g.dw.out.p) nw = cut.dw_most;
  const uint32_t blocks = (uint32_t)(up(g.tiles_m * nx, 8) + up(g.tiles_m * nw, 8));
  hipLaunchKernelGGL((grad_kernel<X, W>), dim3(blocks), dim3(X::kLanes), X::kLds, s, g);
  ARK_HIP(hipGetLastError());
  if ((g.dx.out.p && (cut.dx_most > 1 || twice)) || (g.dw.out.p && nw > cut.tiles_of(cut.vocab))) {
    const uint64_t rows_dx = g.dx.out.p ? tokens : 0, rows_dw = g.dw.out.p ? cut.vocab : 0;
    const uint64_t most = (rows_dx > rows_dw ? rows_dx : rows_dw) * ((g.dx.out.width + 3) / 4);
    const uint64_t join_blocks = (most + kLanes - 1) / kLanes;
    hipLaunchKernelGGL(twice ? join_kernel<true> : join_kernel<false>,
                       dim3(join_blocks < 2048 ? (uint32_t)join_blocks : 2048u), dim3(kLanes), 0, s, g);
    ARK_HIP(hipGetLastError());
  }
  return ARK_OPT_OK;
}

template <typename T, typename LSize, typename Size>
int run_piece(const Call& c, const Plan& p, uint32_t piece) {
  const hipStream_t s = c.stream;
  const uint64_t t0 = (uint64_t)piece * p.piece;
  const uint32_t tokens = (uint32_t)(c.tokens - t0 < p.piece ? c.tokens - t0 : p.piece);
  const uint32_t top = (uint32_t)c.top;
  char* ws = c.ws;
  Meta* meta = (Meta*)(ws + p.meta);
  uint32_t* rows = (uint32_t*)(ws + p.rows);
  uint16_t* x = (uint16_t*)(ws + p.x);
  float* z = (float*)(ws + p.z);
  Targets g = {};
  g.top = top;
  g.vocab = (uint32_t)c.vocab;
  if (c.teacher) {
    uint32_t* index = (uint32_t*)(ws + p.index);
    float *q = (float*)(ws + p.p), *self = (float*)(ws + p.self);
    uint32_t* there = (uint32_t*)(ws + p.there);
    if (tokens) {
      hipLaunchKernelGGL(teacher_kernel, dim3((tokens + 3) / 4), dim3(kLanes), 0, s,
                         (const char*)c.index + t0 * c.index_stride * c.index_bytes,
                         c.index_bytes, c.index_stride,
                         (const char*)c.logits +
                             t0 * c.logits_stride * ark::act_elem_size(c.logits_dtype),
                         c.logits_dtype, c.logits_stride, tokens, top, (uint32_t)c.vocab, c.scale,
                         index, q, self, there);
      ARK_HIP(hipGetLastError());
    }
    g.index = index, g.p = q, g.self = self, g.there = there;
  } else {
    g.targets = (const char*)c.targets + t0 * c.target_bytes;
    g.bytes = c.target_bytes;
    g.ignore = c.ignore;
  }
  const uint16_t* w = p.copy_w ? (const uint16_t*)(ws + p.w) : (const uint16_t*)c.w;
  const uint64_t w_stride = p.copy_w ? p.padded : c.w_stride;
  GatherArgs ga = {};
  RankArgs& ra = ga.rank;
  ra.targets = g;
  ra.tokens = tokens;
  ra.rank = (uint32_t*)(ws + p.rank), ra.rows = rows;
  ra.meta = meta;
  ra.grads = c.grads ? c.grads + t0 : nullptr;
  ra.grad = c.grad, ra.scale = c.scale;
  ra.with_grad = c.with_grad;
  ra.twice = p.twice;
  ra.cut = p.cut;
  ga.x = (const uint16_t*)c.x + t0 * c.x_stride;
  ga.x_stride = c.x_stride;
  ga.columns = (uint32_t)c.columns;
  ga.padded = p.padded;
  ga.out = x;
  ga.loss = c.loss + t0;
  ga.dx = c.dx ? (uint16_t*)c.dx + t0 * c.dx_stride : nullptr;
  ga.dx_stride = c.dx_stride;
  ga.w = (const uint16_t*)c.w, ga.w_stride = c.w_stride;
  ga.entries = (uint32_t*)(ws + p.entries);
  if (!tokens || tokens > kFew) {  // without tokens for what dw's zeros need
    hipLaunchKernelGGL(rank_kernel, dim3(1), dim3(kRankLanes), 0, s, ra);
    ARK_HIP(hipGetLastError());
  }
  if (tokens) {
    ga.blocks = (tokens + kProductStep - 1 + 3) / 4;
    uint64_t pad = 0;
    if (p.copy_w && piece == 0) {
      ga.w_out = (uint16_t*)(ws + p.w);
      pad = (c.vocab + kLanes / 64 - 1) / (kLanes / 64);
      if (pad > 8192) pad = 8192;
    }
    const dim3 grid(ga.blocks + (uint32_t)pad);
    if (tokens <= kFew)
      hipLaunchKernelGGL((gather_kernel<true>), grid, dim3(kLanes), 0, s, ga);
    else
      hipLaunchKernelGGL((gather_kernel<false>), grid, dim3(kLanes), 0, s, ga);
    ARK_HIP(hipGetLastError());
  }
  LogitsArgs la = {};
  la.x = x, la.w = w, la.w_stride = w_stride;
  la.padded = p.padded, la.vocab = (uint32_t)c.vocab, la.spans = p.spans;
  la.e_stride = p.e_stride;
  la.scale = c.scale;
  typedef typename LSize::template P<T, false, false> L;
  la.tiles_m = (uint32_t)((c.vocab + L::BM - 1) / L::BM);
  la.meta = meta;
  la.stats = (float*)(ws + p.stats);
  la.e = c.with_grad ? (uint16_t*)(ws + p.e) : nullptr;
  la.entries = ga.entries, la.top = top, la.z = z;
  int rc;
  if (tokens && (rc = launch_logits<L>(la, la.tiles_m * ((tokens + L::BN - 1) / L::BN), s))) return rc;
  LossArgs lo = {g, rows, meta, la.stats, p.spans, z, ga.loss, c.scale};
  if (!c.with_grad) {  // with tokens, or run() ends before
    hipLaunchKernelGGL(loss_kernel, dim3((tokens + 3) / 4), dim3(kLanes), 0, s, lo);
    ARK_HIP(hipGetLastError());
    return ARK_OPT_OK;
  }
  DzArgs da = {};
  da.loss = lo, da.grads = ra.grads;
  da.grad = c.grad;
  da.e = la.e, da.e_stride = p.e_stride, da.written = p.written, da.span = p.span;
  if (tokens) {
    // eight blocks for every compute unit, and two rounds of a block's lanes at least
    // rows with those up to a whole step of the products
    const uint64_t rows32 = p.twice ? up(tokens + kProductStep - 1, kLanes / 64) : up(tokens, kProductStep);
    const uint64_t round = kLanes * 8;
    uint64_t parts = (2048 + rows32 - 1) / rows32, rounds = (p.written + round - 1) / round;
    if (parts > (rounds + 1) / 2) parts = (rounds + 1) / 2;
    da.share = (uint32_t)((rounds + parts - 1) / parts * round);
    if (rounds == 1)
      hipLaunchKernelGGL((dz_kernel<T, 64>), dim3((uint32_t)(rows32 / (kLanes / 64))), dim3(kLanes),
                         0, s, da);
    else
      hipLaunchKernelGGL(
          (dz_kernel<T, kLanes>),
          dim3((uint32_t)rows32, (uint32_t)((p.written + da.share - 1) / da.share)), dim3(kLanes),
          0, s, da);
    ARK_HIP(hipGetLastError());
  }
  if (!c.dx && !c.dw) return ARK_OPT_OK;
  GradArgs gr = {};
  gr.tiles_m = p.cut.tiles_m;
  gr.meta = meta;
  for (ProductArgs* g : {&gr.dx, &gr.dw}) {
    g->b = la.e, g->b_stride = p.e_stride, g->b_width = (uint32_t)p.e_stride;
    g->a_width = p.padded;
    g->out.meta = meta;
    g->out.width = (uint32_t)c.columns;
  }
  if (c.dx && tokens) {
    Out& o = gr.dx.out;
    gr.dx.a = w, gr.dx.a_stride = w_stride, gr.dx.a_rows = (uint32_t)c.vocab;
    gr.dx.partial = (float*)(ws + p.dx_parts);
    o.p = ga.dx, o.stride = c.dx_stride, o.dtype = c.dtype, o.rows = rows, o.height = tokens;
  }
  if (c.dw) {
    Out& o = gr.dw.out;
    gr.dw.a = x, gr.dw.a_stride = p.padded;
    gr.dw.partial = (float*)(ws + p.dw_parts);
    o.height = (uint32_t)c.vocab;
    // fp32 sums over the pieces, in dw itself or beside it
    const bool last = piece + 1 == p.pieces, wide = c.dw_dtype == ARK_HEAD_F32;
    float* sums = wide ? (float*)c.dw : (float*)(ws + p.sums);
    const uint64_t sums_stride = wide ? c.dw_stride : c.columns;
    const bool add = piece > 0 || (c.flags & ARK_HEAD_ACCUMULATE);
    o.add = add ? sums : nullptr, o.add_stride = sums_stride;
    const bool final = wide || last;
    o.p = final ? c.dw : (void*)sums;
    o.stride = final ? c.dw_stride : sums_stride;
    o.dtype = final ? c.dw_dtype : ARK_HEAD_F32;
  }
  return launch_grad<typename Size::template P<T, true, false>,
                     typename Size::template P<T, true, true>>(gr, p.cut, p.twice, tokens, s);
}

template <typename T>
int run_call(const Call& c, const Plan& p) {
  for (uint32_t i = 0; i < p.pieces; ++i) {
    const int rc = p.small_logits ? p.small ? run_piece<T, Small, Small>(c, p, i)
                                            : run_piece<T, Small, Big>(c, p, i)
                   : p.small      ? run_piece<T, Big, Small>(c, p, i)
                                  : run_piece<T, Big, Big>(c, p, i);
    if (rc) return rc;
  }
  return ARK_OPT_OK;
}

// Bytes that rows x row elements at a row stride span; 0 for none.
int rows_bytes(uint64_t rows, uint64_t row, uint64_t stride, uint32_t es, bool written,
               const char* what, uint64_t* bytes) {
  *bytes = 0;
  if (rows == 0 || row == 0) return ARK_OPT_OK;
  if (rows > 1 && (stride >= (1ull << 32) || (rows - 1) * stride >= (1ull << 48)))
    return fail(ARK_OPT_EINVAL, "%s: stride %llu too large", what, (unsigned long long)stride);
  if (written && rows > 1 && stride < row)
    return fail(ARK_OPT_EINVAL, "%s: rows of %llu elements overlap at stride %llu", what,
                (unsigned long long)row, (unsigned long long)stride);
  *bytes = ((rows - 1) * stride + row) * es;
  return ARK_OPT_OK;
}

int check_sizes(uint64_t tokens, uint64_t columns, uint64_t vocab, uint64_t top, uint32_t dw_dtype) {
  if (dw_dtype > ARK_HEAD_F32) return fail(ARK_OPT_EINVAL, "dw_dtype %u unknown", dw_dtype);
  if (tokens >= (1ull << 31))
    return fail(ARK_OPT_EINVAL, "tokens = %llu too large", (unsigned long long)tokens);
  if (columns == 0 || columns > 65536)
    return fail(ARK_OPT_EINVAL, "columns = %llu: 1 to 65536", (unsigned long long)columns);
  if (vocab == 0 || vocab > (1ull << 21))
    return fail(ARK_OPT_EINVAL, "vocab = %llu: 1 to 2097152", (unsigned long long)vocab);
  if (top == 0 || top > ARK_HEAD_MAX_TOP)
    return fail(ARK_OPT_EINVAL, "top = %llu: 1 to %d", (unsigned long long)top, ARK_HEAD_MAX_TOP);
  return ARK_OPT_OK;
}

struct Range {
  const void* p;
  uint64_t bytes;
  const char* what;
};

int run(Call c) {
  int rc;
  if (c.dtype != ARK_HEAD_F16 && c.dtype != ARK_HEAD_BF16)
    return fail(ARK_OPT_EINVAL, "dtype %u: x and w are fp16 or bf16", c.dtype);
  if ((rc = check_sizes(c.tokens, c.columns, c.vocab, c.top, c.dw ? c.dw_dtype : c.dtype)))
    return rc;
  if (c.dw && c.dw_dtype != ARK_HEAD_F32 && c.dw_dtype != c.dtype)
    return fail(ARK_OPT_EINVAL, "dw_dtype %u: fp32, or that of w", c.dw_dtype);
  if (c.flags & ~ARK_HEAD_ACCUMULATE) return fail(ARK_OPT_EINVAL, "flags %#x unknown", c.flags);
  if ((c.flags & ARK_HEAD_ACCUMULATE) && c.dw && c.dw_dtype != ARK_HEAD_F32)
    return fail(ARK_OPT_EINVAL, "only an fp32 dw can be added to");
  const uint32_t ib = c.teacher ? c.index_bytes : c.target_bytes;
  if (ib != 4 && ib != 8)
    return fail(ARK_OPT_EINVAL, "%s of %u bytes: 4 or 8", c.teacher ? "indices" : "targets", ib);
  if (c.teacher && c.logits_dtype > ARK_HEAD_F32)
    return fail(ARK_OPT_EINVAL, "logits_dtype %u unknown", c.logits_dtype);
  if (!(c.scale > 0.0f) || !(c.scale < 0x1p126f))
    return fail(ARK_OPT_EINVAL, "%s must be positive, and %s below 2^126",
                c.teacher ? "temperature" : "scale", c.teacher ? "finite, its reciprocal" : "it");
  if (c.w_stride >= (1u << 22))
    return fail(ARK_OPT_EINVAL, "w: stride %llu too large", (unsigned long long)c.w_stride);
  const uint32_t les = c.teacher ? ark::act_elem_size(c.logits_dtype) : 1;
  uint64_t xb, wb, tb = 0, ixb = 0, lgb = 0, dxb = 0, dwb = 0;
  const uint32_t dwes = c.dw_dtype == ARK_HEAD_F32 ? 4 : 2;
  if ((rc = rows_bytes(c.tokens, c.columns, c.x_stride, 2, false, "x", &xb)) ||
      (rc = rows_bytes(c.vocab, c.columns, c.w_stride, 2, false, "w", &wb)))
    return rc;
  if (c.teacher) {
    if ((rc = rows_bytes(c.tokens, c.top, c.index_stride, ib, false, "index", &ixb)) ||
        (rc = rows_bytes(c.tokens, c.top, c.logits_stride, les, false, "logits", &lgb)))
      return rc;
  } else {
    tb = c.tokens * ib;
  }
  if (c.dx && (rc = rows_bytes(c.tokens, c.columns, c.dx_stride, 2, true, "dx", &dxb))) return rc;
  if (c.dw && (rc = rows_bytes(c.vocab, c.columns, c.dw_stride, dwes, true, "dw", &dwb))) return rc;
  if ((uintptr_t)c.x % 2 || (uintptr_t)c.w % 2 || (uintptr_t)c.dx % 2 || (uintptr_t)c.dw % dwes ||
      (uintptr_t)c.targets % ib || (uintptr_t)c.index % ib || (uintptr_t)c.logits % les ||
      (uintptr_t)c.loss % 4 || (uintptr_t)c.grads % 4)
    return fail(ARK_OPT_EINVAL, "an array is not aligned to its elements");
  const Plan p = plan_of(c.w, c.w_stride, c.tokens, c.columns, c.vocab, c.top,
                         c.dw ? c.dw_dtype : ARK_HEAD_F32, c.with_grad, c.dx, c.dw);
  if (c.tokens == 0 && (!c.dw || (c.flags & ARK_HEAD_ACCUMULATE))) return ARK_OPT_OK;
  if (c.ws_bytes < p.bytes)
    return fail(ARK_OPT_EINVAL, "workspace of %llu B, %llu B needed",
                (unsigned long long)c.ws_bytes, (unsigned long long)p.bytes);
  if ((uintptr_t)c.ws % 16)
    return fail(ARK_OPT_EINVAL, "workspace %p is not 16-byte aligned", (void*)c.ws);
  const Range written[] = {{c.loss, c.tokens * 4, "loss"},
                           {c.dx, dxb, "dx"},
                           {c.dw, dwb, "dw"},
                           {c.ws, p.bytes, "workspace"}};
  const Range read[] = {{c.x, xb, "x"},           {c.w, wb, "w"},
                        {c.targets, tb, "targets"}, {c.index, ixb, "index"},
                        {c.logits, lgb, "logits"},  {c.grads, c.grads ? c.tokens * 4 : 0, "grads"}};
  for (int i = 0; i < 4; ++i) {
    if (!written[i].bytes) continue;
    for (int k = 0; k < i; ++k)
      if (ark::overlaps(written[i].p, written[i].bytes, written[k].p, written[k].bytes))
        return fail(ARK_OPT_EINVAL, "%s overlaps %s", written[i].what, written[k].what);
    for (const Range& r : read)
      if (r.bytes && ark::overlaps(written[i].p, written[i].bytes, r.p, r.bytes))
        return fail(ARK_OPT_EINVAL, "%s overlaps %s", written[i].what, r.what);
  }
  ark::BufferChecker checker;
  for (const Range& r : read)
    if ((rc = checker.check(r.p, r.bytes, r.what, 0))) return rc;
  for (const Range& r : written)
    if ((rc = checker.check(r.p, r.bytes, r.what, 0))) return rc;
  {
    const void* d[4];
    uint64_t b[4];
    for (int i = 0; i < 4; ++i) d[i] = written[i].p, b[i] = written[i].bytes;
    ark::opt_units_invalidate(d, b, 4);
  }
  return c.dtype == ARK_HEAD_F16 ? run_call<_Float16>(c, p) : run_call<__bf16>(c, p);
}

}  // namespace

extern "C" {

int ark_head_workspace(const void* w, uint64_t w_stride, uint64_t tokens, uint64_t columns,
                       uint64_t vocab, uint64_t top, uint32_t dw_dtype, uint32_t grad,
                       uint64_t* bytes) {
  if (!bytes) return fail(ARK_OPT_EINVAL, "bytes is NULL");
  *bytes = 0;
  if (grad & ~(ARK_HEAD_GRAD | ARK_HEAD_DX | ARK_HEAD_DW))
    return fail(ARK_OPT_EINVAL, "grad %#x unknown", grad);
  if (int rc = check_sizes(tokens, columns, vocab, top, dw_dtype)) return rc;
  *bytes = plan_of(w, w_stride, tokens, columns, vocab, top, dw_dtype, grad != 0,
                   grad & ARK_HEAD_DX, grad & ARK_HEAD_DW).bytes;
  return ARK_OPT_OK;
}

int ark_head_cross_entropy(const void* x, uint64_t x_stride, const void* w, uint64_t w_stride,
                           uint32_t dtype, uint64_t tokens, uint64_t columns, uint64_t vocab,
                           const void* targets, uint32_t target_bytes, int32_t ignore, float scale,
                           float* loss, void* workspace, uint64_t workspace_bytes, void* stream) {
  Call c = {};
  c.x = x, c.x_stride = x_stride, c.w = w, c.w_stride = w_stride, c.dtype = dtype;
  c.tokens = tokens, c.columns = columns, c.vocab = vocab;
  c.targets = targets, c.target_bytes = target_bytes, c.ignore = ignore, c.top = 1;
  c.scale = scale, c.loss = loss;
  c.ws = (char*)workspace, c.ws_bytes = workspace_bytes, c.stream = (hipStream_t)stream;
  return run(c);
}

int ark_head_cross_entropy_grad(const void* x, uint64_t x_stride, const void* w, uint64_t w_stride,
                                uint32_t dtype, uint64_t tokens, uint64_t columns, uint64_t vocab,
                                const void* targets, uint32_t target_bytes, int32_t ignore,
                                float scale, float grad, const float* grads, float* loss, void* dx,
                                uint64_t dx_stride, void* dw, uint32_t dw_dtype,
                                uint64_t dw_stride, uint32_t flags, void* workspace,
                                uint64_t workspace_bytes, void* stream) {
  Call c = {};
  c.x = x, c.x_stride = x_stride, c.w = w, c.w_stride = w_stride, c.dtype = dtype;
  c.tokens = tokens, c.columns = columns, c.vocab = vocab;
  c.targets = targets, c.target_bytes = target_bytes, c.ignore = ignore, c.top = 1;
  c.scale = scale, c.with_grad = true, c.grad = grad, c.grads = grads, c.loss = loss;
  c.dx = dx, c.dx_stride = dx_stride, c.dw = dw, c.dw_dtype = dw_dtype, c.dw_stride = dw_stride;
  c.flags = flags;
  c.ws = (char*)workspace, c.ws_bytes = workspace_bytes, c.stream = (hipStream_t)stream;
  return run(c);
}

int ark_head_distill(const void* x, uint64_t x_stride, const void* w, uint64_t w_stride,
                     uint32_t dtype, uint64_t tokens, uint64_t columns, uint64_t vocab,
                     const void* index, uint32_t index_bytes, uint64_t index_stride,
                     const void* logits, uint32_t logits_dtype, uint64_t logits_stride,
                     uint64_t top, float temperature, float* loss, void* workspace,
                     uint64_t workspace_bytes, void* stream) {
  Call c = {};
  c.x = x, c.x_stride = x_stride, c.w = w, c.w_stride = w_stride, c.dtype = dtype;
  c.tokens = tokens, c.columns = columns, c.vocab = vocab;
  c.teacher = true, c.index = index, c.index_bytes = index_bytes, c.index_stride = index_stride;
  c.logits = logits, c.logits_dtype = logits_dtype, c.logits_stride = logits_stride, c.top = top;
  c.scale = temperature < INFINITY ? 1.0f / temperature : 0.0f, c.loss = loss;
  c.ws = (char*)workspace, c.ws_bytes = workspace_bytes, c.stream = (hipStream_t)stream;
  return run(c);
}

int ark_head_distill_grad(const void* x, uint64_t x_stride, const void* w, uint64_t w_stride,
                          uint32_t dtype, uint64_t tokens, uint64_t columns, uint64_t vocab,
                          const void* index, uint32_t index_bytes, uint64_t index_stride,
                          const void* logits, uint32_t logits_dtype, uint64_t logits_stride,
                          uint64_t top, float temperature, float grad, const float* grads,
                          float* loss, void* dx, uint64_t dx_stride, void* dw, uint32_t dw_dtype,
                          uint64_t dw_stride, uint32_t flags, void* workspace,
                          uint64_t workspace_bytes, void* stream) {
  Call c = {};
  c.x = x, c.x_stride = x_stride, c.w = w, c.w_stride = w_stride, c.dtype = dtype;
  c.tokens = tokens, c.columns = columns, c.vocab = vocab;
  c.teacher = true, c.index = index, c.index_bytes = index_bytes, c.index_stride = index_stride;
  c.logits = logits, c.logits_dtype = logits_dtype, c.logits_stride = logits_stride, c.top = top;
  c.scale = temperature < INFINITY ? 1.0f / temperature : 0.0f;
  c.with_grad = true, c.grad = grad, c.grads = grads, c.loss = loss;
  c.dx = dx, c.dx_stride = dx_stride, c.dw = dw, c.dw_dtype = dw_dtype, c.dw_stride = dw_stride;
  c.flags = flags;
  c.ws = (char*)workspace, c.ws_bytes = workspace_bytes, c.stream = (hipStream_t)stream;
  return run(c);
}

}  // extern "C"
