// ark_rope.hip -- rotary positions and the norms of queries and keys
// (include/ark_rope.h).
#include <math.h>

#include <new>
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

// One of a call's two tensors, q or k.
struct Part {
  Array x;           // the input; for the backward pass the norm's input
  Array dy;          // backward: the gradient of the output
  Array y;           // the output
  const void* gain;  // head_dim values
  uint8_t* act;      // 8-bit form written or read, or NULL
  float* partial;    // backward: the gain's gradient, one row of head_dim a block
  uint32_t heads;
};

struct Args {
  Part part[2];
  const uint64_t* turns;  // 2^64 inv_freq / (2 pi) of every pair
  const void* positions;
  uint64_t start, batch, tokens;
  float magnitude, eps;
  uint32_t position_bytes, head, rotary, inverse, gain_dtype;
  uint64_t rows[2];       // batch * tokens * heads
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

__device__ __forceinline__ int64_t position_at(const Args& a, uint64_t b, uint64_t t) {
  if (!a.positions) return (int64_t)(a.start + t);
  const uint64_t i = b * a.tokens + t;
  return a.position_bytes == 8 ? ((const int64_t*)a.positions)[i] : ((const int32_t*)a.positions)[i];
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

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
  return v;
}

enum Op { kRope, kNorm, kBack };

constexpr uint32_t kBlock = 256, kWaves = 4;
constexpr uint32_t kPairs = ARK_ROPE_MAX_HEAD / 2 / 64;  // pairs of a row a lane takes

// A wave takes rows (a head of a token) one after another; its lanes take the
// row's pairs 64 apart, the pairs past the rotary ones being neighbours.
template <uint32_t DT, uint32_t LAYOUT, Op OP>
__global__ __launch_bounds__(kBlock) void rows_kernel(Args a) {
  const Part& P = a.part[blockIdx.y];
  typedef elem_t<DT> T;
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const uint32_t half = a.rotary / 2, pairs = half + (a.head - a.rotary + 1) / 2;
  uint32_t ju[kPairs], jv[kPairs];
  bool hu[kPairs], hv[kPairs];
  float gu[kPairs], gv[kPairs], su[kPairs] = {}, sv[kPairs] = {};
#pragma unroll
  for (uint32_t i = 0; i < kPairs; ++i) {
    const uint32_t p = lane + 64 * i;
    const bool rot = p < half;
    ju[i] = rot ? (LAYOUT == ARK_ROPE_HALF ? p : 2 * p) : a.rotary + 2 * (p - half);
    jv[i] = rot && LAYOUT == ARK_ROPE_HALF ? p + half : ju[i] + 1;
    hu[i] = p < pairs;
    hv[i] = p < pairs && jv[i] < a.head;
    gu[i] = OP != kRope && hu[i] ? gain_at(a, P.gain, ju[i]) : 0.0f;
    gv[i] = OP != kRope && hv[i] ? gain_at(a, P.gain, jv[i]) : 0.0f;
  }
  const uint64_t columns = (uint64_t)P.heads * a.head;
  const uint64_t groups = (a.batch * a.tokens + ARK_ACT_GROUP - 1) / ARK_ACT_GROUP;
  const uint8_t* exps = P.act ? P.act + groups * columns * ARK_ACT_GROUP : nullptr;
  const uint64_t rows = a.rows[blockIdx.y];
  for (uint64_t row = (uint64_t)blockIdx.x * kWaves + wave; row < rows;
       row += (uint64_t)gridDim.x * kWaves) {
    const uint64_t bt = row / P.heads, h = row % P.heads;
    const uint64_t b = bt / a.tokens, t = bt % a.tokens;
    const int64_t pos = position_at(a, b, t);
    const T* x = (const T*)P.x.p + b * P.x.sb + t * P.x.st + h * P.x.sh;
    const T* dy = OP == kBack ? (const T*)P.dy.p + b * P.dy.sb + t * P.dy.st + h * P.dy.sh : x;
    float xu[kPairs], xv[kPairs], du[kPairs], dv[kPairs], sn[kPairs], cs[kPairs];
    float sq = 0.0f, along = 0.0f;
    const auto load = [&](uint32_t j) -> float {
      if (OP != kBack || !P.act) return (float)x[j];
      const uint64_t col = h * a.head + j, g = bt / ARK_ACT_GROUP;
      return act_value(P.act[(g * columns + col) * ARK_ACT_GROUP + bt % ARK_ACT_GROUP],
                       act_up(exps[g * columns + col]));
    };
#pragma unroll
    for (uint32_t i = 0; i < kPairs; ++i) {
      xu[i] = hu[i] ? load(ju[i]) : 0.0f;
      xv[i] = hv[i] ? load(jv[i]) : 0.0f;
      const uint32_t p = lane + 64 * i;
      sn[i] = 0.0f;
      cs[i] = 1.0f;
      if (p < half) {
        sincos_turns(phase_of(pos, a.turns[p]), &sn[i], &cs[i]);
        sn[i] *= a.inverse || OP == kBack ? -a.magnitude : a.magnitude;
        cs[i] *= a.magnitude;
      }
      if (OP == kBack) {
        const float u = hu[i] ? (float)dy[ju[i]] : 0.0f, v = hv[i] ? (float)dy[jv[i]] : 0.0f;
        du[i] = u * cs[i] - v * sn[i];
        dv[i] = u * sn[i] + v * cs[i];
        along += du[i] * gu[i] * xu[i] + dv[i] * gv[i] * xv[i];
      }
      sq += xu[i] * xu[i] + xv[i] * xv[i];
    }
    float r = 1.0f;
    if (OP != kRope) r = 1.0f / __builtin_sqrtf(wave_sum(sq) / (float)a.head + a.eps);
    if (OP == kBack) along = wave_sum(along) / (float)a.head * r * r;
    T* y = (T*)P.y.p + b * P.y.sb + t * P.y.st + h * P.y.sh;
#pragma unroll
    for (uint32_t i = 0; i < kPairs; ++i) {
      float u, v;
      if (OP == kBack) {
        su[i] += du[i] * xu[i] * r;
        sv[i] += dv[i] * xv[i] * r;
        u = r * (du[i] * gu[i] - xu[i] * along);
        v = r * (dv[i] * gv[i] - xv[i] * along);
      } else {
        const float nu = OP == kNorm ? xu[i] * r * gu[i] : xu[i];
        const float nv = OP == kNorm ? xv[i] * r * gv[i] : xv[i];
        u = nu * cs[i] - nv * sn[i];
        v = nu * sn[i] + nv * cs[i];
      }
      if (hu[i]) y[ju[i]] = narrow<T>(u);
      if (hv[i]) y[jv[i]] = narrow<T>(v);
    }
  }
  if (OP == kBack) {
    __shared__ float sum[kWaves][ARK_ROPE_MAX_HEAD];
#pragma unroll
    for (uint32_t i = 0; i < kPairs; ++i) {
      if (hu[i]) sum[wave][ju[i]] = su[i];
      if (hv[i]) sum[wave][jv[i]] = sv[i];
    }
    __syncthreads();
    for (uint32_t j = threadIdx.x; j < a.head; j += kBlock)
      P.partial[(uint64_t)blockIdx.x * a.head + j] =
          (sum[0][j] + sum[1][j]) + (sum[2][j] + sum[3][j]);
  }
}

// The 8-bit form of a part's input: a lane a column of a group, heads and
// batches wherever their strides put them.
template <uint32_t DT>
__global__ __launch_bounds__(kBlock) void keep_kernel(Args a) {
  const Part& P = a.part[blockIdx.z];
  if (!P.act) return;
  const uint64_t columns = (uint64_t)P.heads * a.head, n = a.batch * a.tokens;
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
  const float down = act_down(s);
#pragma unroll
  for (uint32_t r = 0; r < ARK_ACT_GROUP; ++r)
    P.act[i * ARK_ACT_GROUP + r] = (uint8_t)act_byte<DT>(v[r], s, down);
  P.act[groups * columns * ARK_ACT_GROUP + i] = (uint8_t)s;
}

// The gain's gradient from the blocks' rows, added in order.
__global__ __launch_bounds__(64) void gain_kernel(const float* __restrict__ partial, uint32_t rows,
                                                  uint32_t head, float* __restrict__ dq,
                                                  float* __restrict__ dk, uint32_t accumulate) {
  const uint32_t j = blockIdx.x * 64 + threadIdx.x;
  float* out = blockIdx.y ? dk : dq;
  if (j >= head || !out) return;
  const float* p = partial + (uint64_t)blockIdx.y * rows * head + j;
  float s = 0.0f;
  for (uint32_t i = 0; i < rows; ++i) s += p[(uint64_t)i * head];
  out[j] = accumulate ? out[j] + s : s;
}

constexpr uint32_t kMaxBlocks = 1024;

template <Op OP>
void launch_rows(uint32_t dtype, uint32_t layout, dim3 grid, hipStream_t s, const Args& a) {
#define ARK_ROWS(DT, LY)                                                                       \
  if (dtype == DT && layout == LY)                                                             \
    hipLaunchKernelGGL((rows_kernel<DT, LY, OP>), grid, dim3(kBlock), 0, s, a);
  ARK_ROWS(ARK_ACT_F16, ARK_ROPE_HALF)
  ARK_ROWS(ARK_ACT_BF16, ARK_ROPE_HALF)
  ARK_ROWS(ARK_ACT_F32, ARK_ROPE_HALF)
  ARK_ROWS(ARK_ACT_F16, ARK_ROPE_INTERLEAVED)
  ARK_ROWS(ARK_ACT_BF16, ARK_ROPE_INTERLEAVED)
  ARK_ROWS(ARK_ACT_F32, ARK_ROPE_INTERLEAVED)
#undef ARK_ROWS
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

// Blocks for the larger of the two parts; a third dimension is not needed, the
// kernel's loop takes what is left.
uint32_t row_blocks(const Args& a, uint32_t most) {
  const uint64_t rows = a.rows[0] > a.rows[1] ? a.rows[0] : a.rows[1];
  const uint64_t blocks = (rows + kWaves - 1) / kWaves;
  return (uint32_t)(blocks < most ? blocks : most);
}

Args base_args(const ark_rope* r, uint64_t batch, uint64_t tokens, const void* positions,
               uint32_t position_bytes, uint64_t start) {
  Args a = {};
  a.turns = r->turns;
  a.positions = positions;
  a.position_bytes = position_bytes;
  a.start = start;
  a.batch = batch;
  a.tokens = tokens;
  a.magnitude = r->magnitude;
  a.head = r->head;
  a.rotary = r->rotary;
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
  for (int i = 0; i < 2; ++i) {
    if (!heads[i]) continue;
    a.part[i].x = array_of(g[2 * i + 1]);
    a.part[i].y = array_of(g[2 * i]);
    a.part[i].heads = heads[i];
    a.rows[i] = batch * tokens * heads[i];
  }
  ark::DeviceGuard guard(r->device);
  if (!guard.ok) return ark::fail(ARK_OPT_EHIP, "cannot select device %d", r->device);
  launch_rows<kRope>(dtype, r->layout, dim3(row_blocks(a, 1u << 20), heads[1] ? 2 : 1),
                     (hipStream_t)stream, a);
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
  for (int i = 0; i < 2; ++i) {
    if (!heads[i]) continue;
    a.part[i].x = array_of(g[2 * i + 1]);
    a.part[i].y = array_of(g[2 * i]);
    a.part[i].heads = heads[i];
    a.part[i].gain = gains[i];
    a.rows[i] = n * heads[i];
    a.part[i].act = (uint8_t*)acts[i];
    const uint64_t values = ark::act_groups(n) * heads[i] * r->head;
    most = acts[i] && values > most ? values : most;
  }
  if (most) {
    const dim3 grid((uint32_t)((most + kBlock - 1) / kBlock), 1, heads[1] ? 2 : 1);
    if (dtype == ARK_ACT_F16)
      hipLaunchKernelGGL(keep_kernel<ARK_ACT_F16>, grid, dim3(kBlock), 0, (hipStream_t)stream, a);
    else if (dtype == ARK_ACT_BF16)
      hipLaunchKernelGGL(keep_kernel<ARK_ACT_BF16>, grid, dim3(kBlock), 0, (hipStream_t)stream, a);
    else
      hipLaunchKernelGGL(keep_kernel<ARK_ACT_F32>, grid, dim3(kBlock), 0, (hipStream_t)stream, a);
    ARK_HIP(hipGetLastError());
  }
  launch_rows<kNorm>(dtype, r->layout, dim3(row_blocks(a, 1u << 20), heads[1] ? 2 : 1),
                     (hipStream_t)stream, a);
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
  for (int i = 0; i < 2; ++i) {
    if (!has[i]) continue;
    if (!acts[i]) a.part[i].x = array_of(g[3 * i + 2]);
    a.part[i].dy = array_of(g[3 * i + 1]);
    a.part[i].y = array_of(g[3 * i]);
    a.part[i].heads = heads[i];
    a.part[i].gain = gains[i];
    a.part[i].act = (uint8_t*)acts[i];
    a.rows[i] = n * heads[i];
  }
  ark::DeviceGuard guard(r->device);
  if (!guard.ok) return ark::fail(ARK_OPT_EHIP, "cannot select device %d", r->device);
  const hipStream_t st = (hipStream_t)stream;
  const uint32_t blocks = row_blocks(a, kMaxBlocks);
  ark::StreamBuf buf;
  if (blocks) {
    const hipError_t e = buf.alloc((uint64_t)2 * blocks * r->head * 4, st);
    if (e != hipSuccess) return ark::hip_fail(e, "workspace of ark_rope_norm_backward");
    for (int i = 0; i < 2; ++i) a.part[i].partial = (float*)buf.p + (uint64_t)i * blocks * r->head;
    launch_rows<kBack>(dtype, r->layout, dim3(blocks, 2), st, a);
    ARK_HIP(hipGetLastError());
  }
  hipLaunchKernelGGL(gain_kernel, dim3((r->head + 63) / 64, dk_layout ? 2 : 1), dim3(64), 0, st,
                     (const float*)buf.p, blocks, r->head, dgain_q, dgain_k, accumulate);
  ARK_HIP(hipGetLastError());
  return ARK_OPT_OK;
}

}  // extern "C"
