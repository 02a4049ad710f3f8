// ark_embed.hip -- token lookup and its gradient (include/ark_embed.h).
#include "ark_act.hpp"
#include "ark_common.hpp"
#include "ark_embed.h"

namespace {

using namespace ark::dev;
using ark::fail;

constexpr uint32_t kLanes = 256;

// Eight neighbouring values, in fp32.
struct Eight {
  float v[8];
  template <uint32_t DT>
  __device__ __forceinline__ void load(const void* row, uint64_t c, uint32_t n, bool vec) {
    typedef elem_t<DT> T;
    const T* p = (const T*)row + c;
    if (vec && n >= 8) {
      if constexpr (DT == ARK_EMBED_F32) {
        const f32x4 a = ld_g<f32x4>(p), b = ld_g<f32x4>(p + 4);
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
      } else {
        typedef T V __attribute__((ext_vector_type(8)));
        const V a = ld_g<V>(p);
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) v[i] = (float)a[i];
      }
      return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) v[i] = i < n ? (float)p[i] : 0.0f;
  }
  template <uint32_t DT>
  __device__ __forceinline__ void store(void* row, uint64_t c, uint32_t n, bool vec) const {
    typedef elem_t<DT> T;
    T* p = (T*)row + c;
    if (vec && n >= 8) {
      if constexpr (DT == ARK_EMBED_F32) {
        st_g<f32x4>(p, f32x4{v[0], v[1], v[2], v[3]});
        st_g<f32x4>(p + 4, f32x4{v[4], v[5], v[6], v[7]});
      } else {
        st_g<u32x4>(p, u32x4{narrow2<DT>(v[0], v[1]), narrow2<DT>(v[2], v[3]),
                             narrow2<DT>(v[4], v[5]), narrow2<DT>(v[6], v[7])});
      }
      return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i)
      if (i < n) p[i] = (T)v[i];
  }
};

struct Tokens {
  const void* p;
  uint32_t bytes, vocab;
  // ~0: no row
  __device__ __forceinline__ uint32_t at(uint64_t t) const {
    const int64_t v = bytes == 8 ? ld_g<int64_t>((const int64_t*)p + t)
                                 : ld_g<int32_t>((const int32_t*)p + t);
    return v >= 0 && v < (int64_t)vocab ? (uint32_t)v : ~0u;
  }
};

struct LookupArgs {
  Tokens tokens;
  const void* table;
  void* out;
  uint64_t table_stride, out_stride, n;
  uint32_t columns, vec_in, vec_out;
  float scale;
};

template <uint32_t IN, uint32_t OUT>
__global__ __launch_bounds__(kLanes) void lookup_kernel(LookupArgs a) {
  const uint32_t per = (a.columns + 7) / 8;
  const uint64_t all = a.n * per;
  for (uint64_t i = (uint64_t)blockIdx.x * kLanes + threadIdx.x; i < all;
       i += (uint64_t)gridDim.x * kLanes) {
    const uint64_t t = i / per;
    const uint32_t c = (uint32_t)(i % per) * 8, n = min(a.columns - c, 8u);
    const uint32_t v = a.tokens.at(t);
    Eight e = {};
    if (v != ~0u) {
      e.load<IN>((const elem_t<IN>*)a.table + v * a.table_stride, c, n, a.vec_in);
#pragma unroll
      for (uint32_t k = 0; k < 8; ++k) e.v[k] *= a.scale;
    }
    e.store<OUT>((elem_t<OUT>*)a.out + t * a.out_stride, c, n, a.vec_out);
  }
}

// ---- the gradient -------------------------------------------------------------
//
// Positions sorted by token: a block takes kGroup rows of the table, goes through
// the tokens twice, first counting its own rows' and those of rows before its own,
// then placing the positions of its rows, each wave a stretch of the tokens, so
// that a token's positions stay in order.  Then sums of whole windows of 64 sorted
// positions of one token (frequent ones: text's most frequent token takes a tenth
// of all), and a row's sum from its windows' and the positions beside them.

constexpr uint32_t kGroup = 128;
constexpr uint32_t kSortLanes = 1024;
constexpr uint32_t kSortWaves = kSortLanes / 64;
constexpr uint32_t kWindow = 64;

__global__ __launch_bounds__(kSortLanes) void sort_kernel(Tokens tokens, uint32_t n,
                                                          uint32_t* __restrict__ start,
                                                          uint32_t* __restrict__ pos) {
  __shared__ uint32_t s_at[kSortWaves][kGroup], s_below[kSortWaves];
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const uint32_t v0 = blockIdx.x * kGroup;
  const uint32_t per = (n + kSortLanes - 1) / kSortLanes * 64;  // tokens a wave takes
  const uint32_t lo = min(n, wave * per), hi = min(n, lo + per);
  for (uint32_t i = lane; i < kGroup; i += 64) s_at[wave][i] = 0;
  uint32_t below = 0;
  for (uint32_t t = lo + lane; t < hi; t += 64) {
    const uint32_t v = tokens.at(t);
    if (v < v0)
      ++below;
    else if (v - v0 < kGroup)
      atomicAdd(&s_at[wave][v - v0], 1u);
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) below += __shfl_xor(below, o);
  if (lane == 0) s_below[wave] = below;
  __syncthreads();
  // starts: of the group's rows, and of each wave's positions in them
  if (wave == 0) {
    uint32_t at = 0;
    for (uint32_t w = 0; w < kSortWaves; ++w) at += s_below[w];
    uint32_t mine[2] = {0, 0};  // rows 2 lane, 2 lane + 1
#pragma unroll
    for (uint32_t k = 0; k < 2; ++k)
      for (uint32_t w = 0; w < kSortWaves; ++w) mine[k] += s_at[w][2 * lane + k];
    uint32_t incl = mine[0] + mine[1];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t y = __shfl_up(incl, o);
      if (lane >= (uint32_t)o) incl += y;
    }
    uint32_t from = at + incl - mine[0] - mine[1];
#pragma unroll
    for (uint32_t k = 0; k < 2; ++k) {
      const uint32_t v = v0 + 2 * lane + k;
      if (v <= tokens.vocab) start[v] = from;
      for (uint32_t w = 0; w < kSortWaves; ++w) {
        const uint32_t c = s_at[w][2 * lane + k];
        s_at[w][2 * lane + k] = from;
        from += c;
      }
    }
    if (lane == 63 && v0 + kGroup == tokens.vocab) start[tokens.vocab] = from;
  }
  __syncthreads();
  for (uint32_t t0 = lo; t0 < hi; t0 += 64) {
    const uint32_t t = t0 + lane;
    const uint32_t v = t < hi ? tokens.at(t) : ~0u;
    const uint32_t r = v - v0;
    uint64_t left = __ballot(v != ~0u && v >= v0 && r < kGroup);
    while (left) {
      const uint32_t first = (uint32_t)__ffsll((unsigned long long)left) - 1u;
      const uint32_t row = __builtin_amdgcn_readlane(r, first);
      const uint64_t same = __ballot(r == row) & left;
      const uint32_t at = s_at[wave][row];
      if (same >> lane & 1u) pos[at + __popcll(same & ((1ull << lane) - 1ull))] = t;
      if (lane == first) s_at[wave][row] = at + (uint32_t)__popcll(same);
      left &= ~same;
    }
  }
}

struct SumArgs {
  Tokens tokens;
  const void* dy;
  uint64_t dy_stride;
  const uint32_t *start, *pos;
  float* windows;  // [n / 64][columns up to 8]
  float* dw;
  uint64_t dw_stride;
  uint32_t n, columns, vec_in, vec_out, accumulate;
  float scale;
};

constexpr uint32_t kBatch = 8;  // rows in flight

// e = the rows at sorted positions [lo, hi), added in order, columns [c, c + n).
template <uint32_t DT>
__device__ __forceinline__ void add_rows(const SumArgs& a, Eight* e, uint32_t lo, uint32_t hi,
                                         uint32_t c, uint32_t n) {
  for (uint32_t i = lo; i < hi; i += kBatch) {
    Eight v[kBatch];
#pragma unroll
    for (uint32_t k = 0; k < kBatch; ++k)
      if (i + k < hi)
        v[k].load<DT>((const elem_t<DT>*)a.dy + a.pos[i + k] * a.dy_stride, c, n, a.vec_in);
#pragma unroll
    for (uint32_t k = 0; k < kBatch; ++k)
      if (i + k < hi) {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) e->v[j] += v[k].v[j];
      }
  }
}

// Columns a wave takes: 512.
__device__ __forceinline__ uint32_t wave_tiles(uint32_t columns) { return (columns + 511) / 512; }

template <uint32_t DT>
__global__ __launch_bounds__(kLanes) void window_kernel(SumArgs a) {
  const uint32_t tiles = wave_tiles(a.columns);
  const uint64_t id = (uint64_t)blockIdx.x * (kLanes / 64) + threadIdx.x / 64;
  const uint64_t w = id / tiles;
  const uint32_t c = ((uint32_t)(id % tiles) * 64 + threadIdx.x % 64) * 8;
  if ((w + 1) * kWindow > a.start[a.tokens.vocab]) return;
  const uint32_t lo = (uint32_t)w * kWindow;
  if (a.tokens.at(a.pos[lo]) != a.tokens.at(a.pos[lo + kWindow - 1])) return;
  if (c >= a.columns) return;
  Eight e = {};
  add_rows<DT>(a, &e, lo, lo + kWindow, c, min(a.columns - c, 8u));
  const uint64_t width = (a.columns + 7) / 8 * 8;
  e.store<ARK_EMBED_F32>(a.windows + w * width, c, 8, true);
}

template <uint32_t DT>
__global__ __launch_bounds__(kLanes) void sum_kernel(SumArgs a) {
  const uint32_t tiles = wave_tiles(a.columns);
  const uint64_t all = (uint64_t)a.tokens.vocab * tiles;
  for (uint64_t id = (uint64_t)blockIdx.x * (kLanes / 64) + threadIdx.x / 64; id < all;
       id += (uint64_t)gridDim.x * (kLanes / 64)) {
    const uint32_t v = (uint32_t)(id / tiles);
    const uint32_t c = ((uint32_t)(id % tiles) * 64 + threadIdx.x % 64) * 8;
    const uint32_t lo = a.start[v], hi = a.start[v + 1];
    if ((a.accumulate && lo == hi) || c >= a.columns) continue;
    const uint32_t n = min(a.columns - c, 8u);
    Eight e = {};
    const uint32_t w0 = (lo + kWindow - 1) / kWindow, w1 = hi / kWindow;  // whole windows
    if (w0 < w1) {
      const uint64_t width = (a.columns + 7) / 8 * 8;
      add_rows<DT>(a, &e, lo, w0 * kWindow, c, n);
      for (uint32_t w = w0; w < w1; ++w) {
        Eight s;
        s.load<ARK_EMBED_F32>(a.windows + w * width, c, 8, true);
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) e.v[j] += s.v[j];
      }
      add_rows<DT>(a, &e, w1 * kWindow, hi, c, n);
    } else {
      add_rows<DT>(a, &e, lo, hi, c, n);
    }
    float* row = a.dw + v * a.dw_stride;
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) e.v[j] *= a.scale;
    if (a.accumulate) {
      Eight old;
      old.load<ARK_EMBED_F32>(row, c, n, a.vec_out);
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) e.v[j] += old.v[j];
    }
    e.store<ARK_EMBED_F32>(row, c, n, a.vec_out);
  }
}

// ---- host -------------------------------------------------------------------

struct Layout {
  uint64_t start, pos, windows, bytes;
};
Layout layout_of(uint64_t n, uint64_t vocab, uint64_t columns) {
  Layout l;
  l.start = 0;
  l.pos = ark::align_up((vocab + 1) * 4, 256);
  l.windows = l.pos + ark::align_up(n * 4, 256);
  l.bytes = l.windows + n / kWindow * ((columns + 7) / 8 * 8) * 4;
  return l;
}

int check_sizes(uint64_t n, uint64_t vocab, uint64_t columns) {
  if (n >= (1ull << 31)) return fail(ARK_OPT_EINVAL, "n = %llu too large", (unsigned long long)n);
  if (vocab == 0 || vocab >= (1ull << 31))
    return fail(ARK_OPT_EINVAL, "vocab = %llu: 1 to 2^31 - 1", (unsigned long long)vocab);
  if (columns == 0 || columns > 65536)
    return fail(ARK_OPT_EINVAL, "columns = %llu: 1 to 65536", (unsigned long long)columns);
  return ARK_OPT_OK;
}

int rows_bytes(uint64_t rows, uint64_t row, uint64_t stride, uint32_t es, bool written,
               const char* what, uint64_t* bytes) {
  *bytes = 0;
  if (rows == 0) return ARK_OPT_OK;
  if (rows > 1 && stride >= (1ull << 31))
    return fail(ARK_OPT_EINVAL, "%s: stride %llu too large", what, (unsigned long long)stride);
  if (written && rows > 1 && stride < row)
    return fail(ARK_OPT_EINVAL, "%s: rows of %llu elements overlap at stride %llu", what,
                (unsigned long long)row, (unsigned long long)stride);
  *bytes = ((rows - 1) * stride + row) * es;
  return ARK_OPT_OK;
}

bool vec16(const void* p, uint64_t stride, uint32_t es) {
  return (uintptr_t)p % 16 == 0 && stride * es % 16 == 0;
}

int check_types(uint32_t a, uint32_t b, uint32_t token_bytes) {
  if (a > ARK_EMBED_F32 || b > ARK_EMBED_F32)
    return fail(ARK_OPT_EINVAL, "dtype %u unknown", a > ARK_EMBED_F32 ? a : b);
  if (token_bytes != 4 && token_bytes != 8)
    return fail(ARK_OPT_EINVAL, "tokens of %u bytes: 4 or 8", token_bytes);
  return ARK_OPT_OK;
}

template <uint32_t IN>
void launch_lookup(const LookupArgs& a, uint32_t out, dim3 grid, hipStream_t s) {
  if (out == ARK_EMBED_F16)
    hipLaunchKernelGGL((lookup_kernel<IN, ARK_EMBED_F16>), grid, dim3(kLanes), 0, s, a);
  else if (out == ARK_EMBED_BF16)
    hipLaunchKernelGGL((lookup_kernel<IN, ARK_EMBED_BF16>), grid, dim3(kLanes), 0, s, a);
  else
    hipLaunchKernelGGL((lookup_kernel<IN, ARK_EMBED_F32>), grid, dim3(kLanes), 0, s, a);
}

template <uint32_t DT>
int launch_sums(const SumArgs& a, hipStream_t s) {
  const uint64_t tiles = (a.columns + 511) / 512, windows = a.n / kWindow * tiles;
  if (windows) {
    hipLaunchKernelGGL(window_kernel<DT>, dim3((uint32_t)((windows + 3) / 4)), dim3(kLanes), 0, s, a);
    ARK_HIP(hipGetLastError());
  }
  const uint64_t blocks = ((uint64_t)a.tokens.vocab * tiles + 3) / 4;
  hipLaunchKernelGGL(sum_kernel<DT>, dim3((uint32_t)(blocks < (1u << 23) ? blocks : 1u << 23)),
                     dim3(kLanes), 0, s, a);
  ARK_HIP(hipGetLastError());
  return ARK_OPT_OK;
}

}  // namespace

extern "C" {

int ark_embed_lookup(const void* table, uint64_t table_stride, uint32_t table_dtype,
                     uint64_t vocab, uint64_t columns, const void* tokens, uint32_t token_bytes,
                     uint64_t n, float scale, void* out, uint64_t out_stride, uint32_t out_dtype,
                     void* stream) {
  int rc;
  if ((rc = check_types(table_dtype, out_dtype, token_bytes))) return rc;
  if ((rc = check_sizes(n, vocab, columns))) return rc;
  if (n == 0) return ARK_OPT_OK;
  const uint32_t es = ark::act_elem_size(table_dtype), eo = ark::act_elem_size(out_dtype);
  uint64_t tb, ob;
  if ((rc = rows_bytes(vocab, columns, table_stride, es, false, "table", &tb)) ||
      (rc = rows_bytes(n, columns, out_stride, eo, true, "out", &ob)))
    return rc;
  if ((uintptr_t)table % es || (uintptr_t)out % eo || (uintptr_t)tokens % token_bytes)
    return fail(ARK_OPT_EINVAL, "table, out or tokens not aligned to their elements");
  if (ark::overlaps(out, ob, table, tb) || ark::overlaps(out, ob, tokens, n * token_bytes))
    return fail(ARK_OPT_EINVAL, "out overlaps table or tokens");
  ark::BufferChecker checker;
  if ((rc = checker.check(table, tb, "table", 0)) || (rc = checker.check(out, ob, "out", 0)) ||
      (rc = checker.check(tokens, n * token_bytes, "tokens", 0)))
    return rc;
  {
    const void* d = out;
    ark::opt_units_invalidate(&d, &ob, 1);
  }
  LookupArgs a = {};
  a.tokens = {tokens, token_bytes, (uint32_t)vocab};
  a.table = table, a.out = out;
  a.table_stride = table_stride, a.out_stride = out_stride, a.n = n;
  a.columns = (uint32_t)columns;
  a.vec_in = vec16(table, table_stride, es), a.vec_out = vec16(out, out_stride, eo);
  a.scale = scale;
  const uint64_t blocks = (n * ((columns + 7) / 8) + kLanes - 1) / kLanes;
  const dim3 grid((uint32_t)(blocks < (1u << 20) ? blocks : 1u << 20));
  const hipStream_t s = (hipStream_t)stream;
  if (table_dtype == ARK_EMBED_F16)
    launch_lookup<ARK_EMBED_F16>(a, out_dtype, grid, s);
  else if (table_dtype == ARK_EMBED_BF16)
    launch_lookup<ARK_EMBED_BF16>(a, out_dtype, grid, s);
  else
    launch_lookup<ARK_EMBED_F32>(a, out_dtype, grid, s);
  ARK_HIP(hipGetLastError());
  return ARK_OPT_OK;
}

int ark_embed_grad_workspace(uint64_t n, uint64_t vocab, uint64_t columns, uint64_t* bytes) {
  if (!bytes) return fail(ARK_OPT_EINVAL, "bytes is NULL");
  *bytes = 0;
  if (int rc = check_sizes(n, vocab, columns)) return rc;
  *bytes = layout_of(n, vocab, columns).bytes;
  return ARK_OPT_OK;
}

int ark_embed_grad(const void* dy, uint64_t dy_stride, uint32_t dy_dtype, const void* tokens,
                   uint32_t token_bytes, uint64_t n, uint64_t vocab, uint64_t columns, float scale,
                   float* dw, uint64_t dw_stride, uint32_t flags, void* workspace,
                   uint64_t workspace_bytes, void* stream) {
  int rc;
  if ((rc = check_types(dy_dtype, dy_dtype, token_bytes))) return rc;
  if (flags & ~ARK_EMBED_ACCUMULATE) return fail(ARK_OPT_EINVAL, "flags %#x unknown", flags);
  if ((rc = check_sizes(n, vocab, columns))) return rc;
  const uint32_t es = ark::act_elem_size(dy_dtype);
  uint64_t yb, wb;
  if ((rc = rows_bytes(n, columns, dy_stride, es, false, "dy", &yb)) ||
      (rc = rows_bytes(vocab, columns, dw_stride, 4, true, "dw", &wb)))
    return rc;
  if ((uintptr_t)dy % es || (uintptr_t)dw % 4 || (uintptr_t)tokens % token_bytes)
    return fail(ARK_OPT_EINVAL, "dy, dw or tokens not aligned to their elements");
  if (n == 0 && (flags & ARK_EMBED_ACCUMULATE)) return ARK_OPT_OK;
  const Layout l = layout_of(n, vocab, columns);
  if (workspace_bytes < l.bytes)
    return fail(ARK_OPT_EINVAL, "workspace of %llu B, %llu B needed",
                (unsigned long long)workspace_bytes, (unsigned long long)l.bytes);
  if ((uintptr_t)workspace % 16)
    return fail(ARK_OPT_EINVAL, "workspace %p is not 16-byte aligned", workspace);
  const uint64_t kb = n * token_bytes;
  if (ark::overlaps(dw, wb, dy, yb) || ark::overlaps(dw, wb, tokens, kb))
    return fail(ARK_OPT_EINVAL, "dw overlaps dy or tokens");
  if (ark::overlaps(workspace, l.bytes, dy, yb) || ark::overlaps(workspace, l.bytes, tokens, kb) ||
      ark::overlaps(workspace, l.bytes, dw, wb))
    return fail(ARK_OPT_EINVAL, "workspace overlaps dy, tokens or dw");
  ark::BufferChecker checker;
  if ((rc = checker.check(dy, yb, "dy", 0)) || (rc = checker.check(dw, wb, "dw", 0)) ||
      (rc = checker.check(tokens, kb, "tokens", 0)) ||
      (rc = checker.check(workspace, l.bytes, "workspace", 0)))
    return rc;
  {
    const void* d[2] = {dw, workspace};
    const uint64_t b[2] = {wb, l.bytes};
    ark::opt_units_invalidate(d, b, 2);
  }
  const hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)workspace;
  SumArgs a = {};
  a.tokens = {tokens, token_bytes, (uint32_t)vocab};
  a.dy = dy, a.dy_stride = dy_stride;
  a.start = (uint32_t*)(ws + l.start), a.pos = (uint32_t*)(ws + l.pos);
  a.windows = (float*)(ws + l.windows);
  a.dw = dw, a.dw_stride = dw_stride;
  a.n = (uint32_t)n, a.columns = (uint32_t)columns;
  a.vec_in = vec16(dy, dy_stride, es), a.vec_out = vec16(dw, dw_stride, 4);
  a.accumulate = flags & ARK_EMBED_ACCUMULATE ? 1u : 0u;
  a.scale = scale;
  hipLaunchKernelGGL(sort_kernel, dim3((uint32_t)((vocab + kGroup - 1) / kGroup)), dim3(kSortLanes),
                     0, s, a.tokens, a.n, (uint32_t*)a.start, (uint32_t*)a.pos);
  ARK_HIP(hipGetLastError());
  if (dy_dtype == ARK_EMBED_F16) return launch_sums<ARK_EMBED_F16>(a, s);
  if (dy_dtype == ARK_EMBED_BF16) return launch_sums<ARK_EMBED_BF16>(a, s);
  return launch_sums<ARK_EMBED_F32>(a, s);
}

}  // extern "C"
