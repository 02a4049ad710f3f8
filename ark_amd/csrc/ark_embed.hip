// ark_embed.hip -- token lookup and its gradient (include/ark_embed.h).
#include <type_traits>

#include "ark_act.hpp"
#include "ark_common.hpp"
#include "ark_embed.h"

namespace {

using namespace ark::dev;
using ark::fail;

constexpr uint32_t kLanes = 256;
constexpr uint64_t kMostBlocks = 1ull << 23;  // a launch has fewer than 2^32 lanes

typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

// N neighbouring values of a row, in fp32, at any element's alignment (gfx950 takes
// unaligned global accesses).
template <uint32_t N>
struct Some {
  float v[N];
  template <uint32_t DT>
  __device__ __forceinline__ void load(const void* row, uint64_t c) {
    typedef elem_t<DT> T;
    typedef T V __attribute__((ext_vector_type(N < 8 || DT != ARK_EMBED_F32 ? N : 4),
                               aligned(sizeof(T))));
    constexpr uint32_t kEach = sizeof(V) / sizeof(T);
#pragma unroll
    for (uint32_t i = 0; i < N; i += kEach) {
      const V a = *(const ARK_GLOBAL V*)((const T*)row + c + i);
#pragma unroll
      for (uint32_t k = 0; k < kEach; ++k) v[i + k] = (float)a[k];
    }
  }
  template <uint32_t DT>
  __device__ __forceinline__ void store(void* row, uint64_t c) const {
    typedef elem_t<DT> T;
    if constexpr (DT == ARK_EMBED_F32) {
#pragma unroll
      for (uint32_t i = 0; i < N; i += 4)
        st_g<f32x4_a4>((T*)row + c + i, f32x4_a4{v[i], v[i + 1], v[i + 2], v[i + 3]});
    } else {
      typedef uint32_t V __attribute__((ext_vector_type(N / 2), aligned(2)));
      V a;
#pragma unroll
      for (uint32_t i = 0; i < N / 2; ++i) a[i] = narrow2<DT>(v[2 * i], v[2 * i + 1]);
      *(ARK_GLOBAL V*)((T*)row + c) = a;
    }
  }
};

struct Tokens {
  const void* p;
  uint32_t bytes, vocab;
  // ~0: no row
  __device__ __forceinline__ uint32_t row(int64_t v) const {
    return v >= 0 && v < (int64_t)vocab ? (uint32_t)v : ~0u;
  }
  __device__ __forceinline__ uint32_t at(uint64_t t) const {
    return row(bytes == 8 ? ld_g<int64_t>((const int64_t*)p + t)
                          : ld_g<int32_t>((const int32_t*)p + t));
  }
  // Those at t, t + 64, ..., past `last` the last one's; their loads all together, which
  // a branch on the size for each would keep apart.
  template <uint32_t N>
  __device__ __forceinline__ void each(uint32_t t, uint32_t last, uint32_t (&out)[N]) const {
    const auto load = [&](auto kind) __attribute__((always_inline)) {
      typedef decltype(kind) T;
      T v[N];
#pragma unroll
      for (uint32_t k = 0; k < N; ++k) v[k] = ld_g<T>((const T*)p + min(t + k * 64, last));
#pragma unroll
      for (uint32_t k = 0; k < N; ++k) out[k] = row(v[k]);
    };
    if (bytes == 8)
      load(int64_t());
    else
      load(int32_t());
  }
};

struct LookupArgs {
  Tokens tokens;
  const void* table;
  void* out;
  uint64_t table_stride, out_stride, n;
  uint32_t columns;
  float scale;
};

// A lane takes eight values of a row; those past the last whole eight are the last
// eight again, written twice alike.  Bound by HBM: 16384 rows of 2048 bf16, 18 us
// with the call, 7.3 TB/s (rows that occur twice come from cache).
template <uint32_t IN, uint32_t OUT>
__global__ __launch_bounds__(kLanes) void lookup_kernel(LookupArgs a) {
  const uint32_t per = (a.columns + 7) / 8;
  const uint64_t all = a.n * per;
  for (uint64_t i = (uint64_t)blockIdx.x * kLanes + threadIdx.x; i < all;
       i += (uint64_t)gridDim.x * kLanes) {
    const uint64_t t = i / per;
    const uint32_t c = min((uint32_t)(i % per) * 8, a.columns - 8);
    const uint32_t v = a.tokens.at(t);
    Some<8> e = {};
    if (v != ~0u) {
      e.load<IN>((const elem_t<IN>*)a.table + v * a.table_stride, c);
#pragma unroll
      for (uint32_t k = 0; k < 8; ++k) e.v[k] *= a.scale;
    }
    e.store<OUT>((elem_t<OUT>*)a.out + t * a.out_stride, c);
  }
}
// Rows of fewer than eight values, a lane a value.
template <uint32_t IN, uint32_t OUT>
__global__ __launch_bounds__(kLanes) void lookup_short_kernel(LookupArgs a) {
  const uint64_t all = a.n * a.columns;
  for (uint64_t i = (uint64_t)blockIdx.x * kLanes + threadIdx.x; i < all;
       i += (uint64_t)gridDim.x * kLanes) {
    const uint64_t t = i / a.columns;
    const uint32_t c = (uint32_t)(i % a.columns), v = a.tokens.at(t);
    const float x =
        v != ~0u ? (float)((const elem_t<IN>*)a.table)[v * a.table_stride + c] * a.scale : 0.0f;
    ((elem_t<OUT>*)a.out)[t * a.out_stride + c] = (elem_t<OUT>)x;
  }
}

// ---- the gradient -------------------------------------------------------------
//
// Positions sorted by token: a block takes kGroup rows of the table, goes through
// the tokens twice, first counting its own rows' and those of rows before its own,
// then placing the positions of its rows, each wave a stretch of the tokens, so
// that a token's positions stay in order.  Then sums of whole windows of sixteen
// sorted positions of one token (text's most frequent token takes a tenth of all:
// its rows are added by many waves at once), and a row's sum from its windows' and
// the positions beside them.

constexpr uint32_t kGroup = 128;
constexpr uint32_t kSortLanes = 1024;
constexpr uint32_t kSortWaves = kSortLanes / 64;
constexpr uint32_t kKept = 16;  // tokens a lane asks for at once
constexpr uint32_t kWindow = 16;

// n is 1 at least: lanes past it read the last token again.
// KEEP: each lane has kKept tokens at most, which stay in registers for the second
// time.  Bound by a block's latency: 16384 tokens into 250 groups 10.6 us, 16 without.
template <bool KEEP>
__global__ __launch_bounds__(kSortLanes) void sort_kernel(Tokens tokens, uint32_t n,
                                                          uint32_t* __restrict__ start,
                                                          uint32_t* __restrict__ pos) {
  __shared__ uint32_t s_at[kSortWaves][kGroup], s_below[kSortWaves], s_first;
  static_assert(kGroup == 128, "two waves' rows");
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const uint32_t v0 = blockIdx.x * kGroup;
  const uint32_t per = (n + kSortLanes - 1) / kSortLanes * 64;  // tokens a wave takes
  const uint32_t lo = min(n, wave * per), hi = min(n, lo + per);
  for (uint32_t i = lane; i < kGroup; i += 64) s_at[wave][i] = 0;
  uint32_t below = 0, v[kKept];
  const auto ask = [&](uint32_t t0) __attribute__((always_inline)) {
    tokens.each<kKept>(t0 + lane, n - 1, v);
#pragma unroll
    for (uint32_t k = 0; k < kKept; ++k)
      if (t0 + k * 64 + lane >= hi) v[k] = ~0u;
  };
  if (KEEP) ask(lo);
  for (uint32_t t0 = lo; t0 < hi; t0 += 64 * kKept) {
    if (!KEEP) ask(t0);
#pragma unroll
    for (uint32_t k = 0; k < kKept; ++k) {
      if (v[k] < v0)
        ++below;
      else if (v[k] - v0 < kGroup)
        atomicAdd(&s_at[wave][v[k] - v0], 1u);
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) below += __shfl_xor(below, o);
  if (lane == 0) s_below[wave] = below;
  __syncthreads();
  // starts: of the group's rows, and of each wave's positions in them, a lane a row
  const uint32_t row = threadIdx.x;
  uint32_t count[kSortWaves], total = 0, incl = 0;
  if (row < kGroup) {
#pragma unroll
    for (uint32_t w = 0; w < kSortWaves; ++w) count[w] = s_at[w][row];
#pragma unroll
    for (uint32_t w = 0; w < kSortWaves; ++w) total += count[w];
    incl = total;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t y = __shfl_up(incl, o);
      if (lane >= (uint32_t)o) incl += y;
    }
    if (row == 63) s_first = incl;
  }
  __syncthreads();
  if (row < kGroup) {
    uint32_t from = incl - total + (row < 64 ? 0u : s_first);
#pragma unroll
    for (uint32_t w = 0; w < kSortWaves; ++w) from += s_below[w];
    if (v0 + row <= tokens.vocab) start[v0 + row] = from;
    if (row + 1 == kGroup && v0 + kGroup == tokens.vocab) start[tokens.vocab] = from + total;
#pragma unroll
    for (uint32_t w = 0; w < kSortWaves; ++w) s_at[w][row] = from, from += count[w];
  }
  __syncthreads();
  for (uint32_t t0 = lo; t0 < hi; t0 += 64 * kKept) {
    if (!KEEP) ask(t0);
#pragma unroll
    for (uint32_t k = 0; k < kKept; ++k) {
      const uint32_t r = v[k] - v0;
      uint64_t left = __ballot(v[k] != ~0u && v[k] >= v0 && r < kGroup);
      while (left) {
        const uint32_t first = (uint32_t)__ffsll((unsigned long long)left) - 1u;
        const uint32_t row = __builtin_amdgcn_readlane(r, first);
        const uint64_t same = __ballot(r == row) & left;
        const uint32_t at = s_at[wave][row];
        if (same >> lane & 1u)
          pos[at + __popcll(same & ((1ull << lane) - 1ull))] = t0 + k * 64 + lane;
        if (lane == first) s_at[wave][row] = at + (uint32_t)__popcll(same);
        left &= ~same;
      }
    }
  }
}

struct SumArgs {
  Tokens tokens;
  const void* dy;
  uint64_t dy_stride;
  const uint32_t *start, *pos;
  float* windows;  // [n / 16][columns up to 4]
  float* dw;
  uint64_t dw_stride;
  uint32_t n, columns, accumulate;
  float scale;
};

// A wave takes 256 columns, a lane four; those past the last whole four are the
// last four again.  Rows of fewer than four values: a lane one of them (WIDE false).
template <bool WIDE>
struct Column {
  static constexpr uint32_t kEach = WIDE ? 4 : 1, kWave = WIDE ? 256 : 64;
  uint32_t own, c;  // the first that is the lane's alone, and that it loads (lanes
                    // past the last column load with the others and store nothing)
  __device__ __forceinline__ Column(uint32_t tile, uint32_t columns) {
    own = (tile * 64 + threadIdx.x % 64) * kEach;
    c = min(own, columns - kEach);
  }
};

__device__ __forceinline__ auto sorted(const SumArgs& a) {
  return [p = a.pos](uint32_t i) { return ld_g<uint32_t>(p + i); };
}

// e = e + the rows at sorted positions [lo, hi), in order, kBatch in flight, as they are
// in memory until they are added.  pos(i): the i-th position.
template <uint32_t DT, bool WIDE, uint32_t kBatch, typename F>
__device__ __forceinline__ void add_rows(const SumArgs& a, const Column<WIDE>& col,
                                         float (&e)[Column<WIDE>::kEach], uint32_t lo,
                                         uint32_t hi, F pos) {
  constexpr uint32_t E = Column<WIDE>::kEach;
  typedef elem_t<DT> T;
  typedef T V __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  typedef typename std::conditional<WIDE, V, T>::type R;
  for (uint32_t i = lo; i < hi; i += kBatch) {
    // the positions of the rows, a lane one
    const uint32_t k = i + threadIdx.x % kBatch;
    const uint32_t p = pos(min(k, hi - 1));
    R v[kBatch];
    const auto load = [&](uint32_t k) __attribute__((always_inline)) {
      const uint32_t t = __builtin_amdgcn_readlane(p, k);
      v[k] = *(const ARK_GLOBAL R*)((const T*)a.dy + t * a.dy_stride + col.c);
    };
    const auto add = [&](uint32_t k) __attribute__((always_inline)) {
      if constexpr (WIDE) {
#pragma unroll
        for (uint32_t j = 0; j < E; ++j) e[j] += (float)v[k][j];
      } else {
        e[0] += (float)v[k];
      }
    };
    if (i + kBatch <= hi) {
#pragma unroll
      for (uint32_t k = 0; k < kBatch; ++k) load(k);
#pragma unroll
      for (uint32_t k = 0; k < kBatch; ++k) add(k);
    } else {
#pragma unroll
      for (uint32_t k = 0; k < kBatch; ++k)
        if (i + k < hi) load(k);
#pragma unroll
      for (uint32_t k = 0; k < kBatch; ++k)
        if (i + k < hi) add(k);
    }
  }
}

__device__ __forceinline__ uint64_t window_width(uint32_t columns) {
  return (columns + 3) / 4 * 4;
}

// Latency: 16384 of text's tokens, of which a third of the windows are one token's, 768
// columns of fp16, 5 us.
template <uint32_t DT, bool WIDE>
__global__ __launch_bounds__(kLanes) void window_kernel(SumArgs a) {
  typedef Column<WIDE> C;
  const uint32_t tiles = (a.columns + C::kWave - 1) / C::kWave;
  const uint64_t all = (uint64_t)a.start[a.tokens.vocab] / kWindow * tiles;
  for (uint64_t id = (uint64_t)blockIdx.x * (kLanes / 64) +
                     __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
       id < all; id += (uint64_t)gridDim.x * (kLanes / 64)) {
    const uint64_t w = id / tiles;
    const uint32_t lo = (uint32_t)w * kWindow;
    if (a.tokens.at(a.pos[lo]) != a.tokens.at(a.pos[lo + kWindow - 1])) continue;
    const C col((uint32_t)(id % tiles), a.columns);
    float e[C::kEach] = {};
    add_rows<DT, WIDE, kWindow>(a, col, e, lo, lo + kWindow, sorted(a));
    float* out = a.windows + w * window_width(a.columns) + col.c;
    // a lane's last four may be another's too: written twice alike
#pragma unroll
    for (uint32_t j = 0; j < C::kEach; ++j) out[j] = e[j];
  }
}

constexpr uint32_t kBatch = 8;  // half the registers of sixteen, twice the waves

constexpr uint32_t kRows = 4;     // rows of the table a wave takes, their starts read at once

// e to row v, or added there; zeros.
template <bool WIDE>
__device__ __forceinline__ void put_row(const SumArgs& a, const Column<WIDE>& col, uint32_t v,
                                        float (&e)[Column<WIDE>::kEach]) {
  typedef Column<WIDE> C;
  float* row = a.dw + v * a.dw_stride;
#pragma unroll
  for (uint32_t j = 0; j < C::kEach; ++j) e[j] *= a.scale;
  if constexpr (WIDE) {
    if (col.c == col.own) {
      Some<4> out;
      if (a.accumulate) out.load<ARK_EMBED_F32>(row, col.c);
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) out.v[j] = a.accumulate ? out.v[j] + e[j] : e[j];
      out.store<ARK_EMBED_F32>(row, col.c);
      return;
    }
  }
#pragma unroll
  for (uint32_t j = 0; j < C::kEach; ++j)
    if (col.c + j >= col.own) row[col.c + j] = a.accumulate ? row[col.c + j] + e[j] : e[j];
}
template <bool WIDE>
__device__ __forceinline__ void put_zeros(const SumArgs& a, const Column<WIDE>& col, uint32_t v) {
  float* row = a.dw + v * a.dw_stride;
  if (WIDE && col.c == col.own) {
    const Some<4> none = {};
    none.store<ARK_EMBED_F32>(row, col.c);
  } else {
#pragma unroll
    for (uint32_t j = 0; j < Column<WIDE>::kEach; ++j)
      if (col.c + j >= col.own) row[col.c + j] = 0.0f;
  }
}

template <uint32_t DT, bool WIDE>
__device__ __forceinline__ void sum_row(const SumArgs& a, const Column<WIDE>& col, uint32_t v,
                                        uint32_t lo, uint32_t hi) {
  typedef Column<WIDE> C;
  float e[C::kEach] = {};
  const uint32_t w0 = (lo + kWindow - 1) / kWindow, w1 = hi / kWindow;  // whole windows
  const bool windows = w0 < w1;
  add_rows<DT, WIDE, kBatch>(a, col, e, lo, windows ? w0 * kWindow : hi, sorted(a));
  if (windows) {
    const uint64_t width = window_width(a.columns);
    for (uint32_t w = w0; w < w1; w += kBatch) {
      float s[kBatch][C::kEach];
#pragma unroll
      for (uint32_t k = 0; k < kBatch; ++k)
        if (w + k < w1) {
          const float* in = a.windows + (w + k) * width + col.c;
#pragma unroll
          for (uint32_t j = 0; j < C::kEach; ++j) s[k][j] = in[j];
        }
#pragma unroll
      for (uint32_t k = 0; k < kBatch; ++k)
        if (w + k < w1) {
#pragma unroll
          for (uint32_t j = 0; j < C::kEach; ++j) e[j] += s[k][j];
        }
    }
    add_rows<DT, WIDE, kBatch>(a, col, e, w1 * kWindow, hi, sorted(a));
  }
  put_row(a, col, v, e);
}

// Every row of the table, or those of tokens that occur.  Most rows have no token
// (a vocabulary is larger than a batch's words), so what counts is the zeros'
// way to memory: 16384 tokens into 32000 x 768, 98 MB written and 25 read in 29 us.
template <uint32_t DT, bool WIDE>
__global__ __launch_bounds__(kLanes) void sum_kernel(SumArgs a) {
  typedef Column<WIDE> C;
  const uint32_t tiles = (a.columns + C::kWave - 1) / C::kWave, vocab = a.tokens.vocab;
  const uint64_t all = (uint64_t)((vocab + kRows - 1) / kRows) * tiles;
  for (uint64_t id = (uint64_t)blockIdx.x * (kLanes / 64) +
                     __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
       id < all; id += (uint64_t)gridDim.x * (kLanes / 64)) {
    const uint32_t v0 = (uint32_t)(id / tiles) * kRows;
    const C col((uint32_t)(id % tiles), a.columns);
    uint32_t at[kRows + 1];
#pragma unroll
    for (uint32_t k = 0; k <= kRows; ++k) at[k] = a.start[min(v0 + k, vocab)];
    if (!a.accumulate) {
#pragma unroll
      for (uint32_t k = 0; k < kRows; ++k)
        if (at[k] == at[k + 1] && v0 + k < vocab) put_zeros(a, col, v0 + k);
    }
    for (uint32_t k = 0; k < kRows; ++k)
      if (at[k] != at[k + 1]) sum_row<DT, WIDE>(a, col, v0 + k, at[k], at[k + 1]);
  }
}

// The whole gradient of few tokens in one launch: a block takes kFewRows rows of the
// table and a tile of columns for each of its waves, finds the rows' positions among all
// tokens and puts them in order by counting, for each, those before it.  A row's sums are
// by sixteen positions.  305 tokens into 14862 x 1837 19.7 us (109 MB of zeros), 276 into
// 604 x 64 9; sorted and summed in three launches 26 and 16.  512 equal tokens, a row by
// four waves, take longer than by windows, more of them much longer.
constexpr uint32_t kFew = 512;
constexpr uint32_t kFewRows = 16;

template <uint32_t DT, bool WIDE>
__global__ __launch_bounds__(kLanes) void few_kernel(SumArgs a) {
  typedef Column<WIDE> C;
  constexpr uint32_t kWaves = kLanes / 64, kEach = kFew / kLanes;
  __shared__ uint64_t s_mask[kEach * kWaves];
  constexpr uint32_t kAtOnce = 16;  // of the ones found, compared with
  __shared__ __align__(16) uint32_t s_found[kFew + kAtOnce];
  __shared__ uint32_t s_pos[kFew], s_start[kFewRows + 1];
  const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t v0 = blockIdx.x * kFewRows, rows = min(kFewRows, a.tokens.vocab - v0);
  uint32_t row[kEach];
#pragma unroll
  for (uint32_t k = 0; k < kEach; ++k) {
    const uint32_t t = k * kLanes + threadIdx.x;
    row[k] = t < a.n ? a.tokens.at(t) - v0 : ~0u;  // ~0, no row, stays past them
    const uint64_t mask = __ballot(row[k] < rows);
    if (lane == 0) s_mask[k * kWaves + wave] = mask;
  }
  __syncthreads();
  uint32_t all = 0;
#pragma unroll
  for (uint32_t i = 0; i < kEach * kWaves; ++i) {
    const uint64_t mask = s_mask[i];
    if (i % kWaves == wave && row[i / kWaves] < rows)
      s_found[all + __popcll(mask & ((1ull << lane) - 1ull))] =
          row[i / kWaves] << 16 | (i / kWaves * kLanes + threadIdx.x);
    all += __popcll(mask);
  }
  if (threadIdx.x < kAtOnce) s_found[all + threadIdx.x] = ~0u;
  __syncthreads();
  // those found that are below a key
  const auto below = [&](uint32_t key) {
    uint32_t at = 0;
    for (uint32_t j = 0; j < all; j += kAtOnce) {
      u32x4 v[kAtOnce / 4];
#pragma unroll
      for (uint32_t q = 0; q < kAtOnce / 4; ++q) v[q] = *(const u32x4*)(s_found + j + q * 4);
#pragma unroll
      for (uint32_t q = 0; q < kAtOnce; ++q) at += v[q / 4][q % 4] < key ? 1 : 0;
    }
    return at;
  };
  for (uint32_t i = threadIdx.x; i < all; i += kLanes) s_pos[below(s_found[i])] = s_found[i] & 0xFFFFu;
  if (threadIdx.x <= kFewRows) s_start[threadIdx.x] = below(threadIdx.x << 16);
  __syncthreads();
  const uint32_t tile0 = blockIdx.y * kWaves;
  const uint32_t tiles = min((a.columns + C::kWave - 1) / C::kWave - tile0, kWaves);
  for (uint32_t i = wave; i < rows * tiles; i += kWaves) {
    const uint32_t r = i / tiles, lo = s_start[r], hi = s_start[r + 1];
    const C col(tile0 + i % tiles, a.columns);
    if (lo == hi) {
      if (!a.accumulate) put_zeros(a, col, v0 + r);
      continue;
    }
    float e[C::kEach] = {};
    for (uint32_t g = lo; g < hi; g += kWindow) {
      float s[C::kEach] = {};
      add_rows<DT, WIDE, kWindow>(a, col, s, g, min(g + kWindow, hi),
                                  [&](uint32_t k) { return s_pos[k]; });
#pragma unroll
      for (uint32_t j = 0; j < C::kEach; ++j) e[j] += s[j];
    }
    put_row(a, col, v0 + r, e);
  }
}

// The gradient of no tokens: every row zeros, with nothing to count or to read.
template <bool WIDE>
__global__ __launch_bounds__(kLanes) void zero_kernel(SumArgs a) {
  typedef Column<WIDE> C;
  const uint32_t tiles = (a.columns + C::kWave - 1) / C::kWave;
  const uint64_t all = (uint64_t)a.tokens.vocab * tiles;
  for (uint64_t id = (uint64_t)blockIdx.x * (kLanes / 64) +
                     __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
       id < all; id += (uint64_t)gridDim.x * (kLanes / 64))
    put_zeros(a, C((uint32_t)(id % tiles), a.columns), (uint32_t)(id / tiles));
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
  l.bytes = l.windows + n / kWindow * ((columns + 3) / 4 * 4) * 4;
  return l;
}

int check_sizes(uint64_t n, uint64_t vocab, uint64_t columns) {
  if (n >= (1ull << 31)) return fail(ARK_OPT_EINVAL, "n = %llu too large", (unsigned long long)n);
  if (vocab == 0 || vocab > (1ull << 28))
    return fail(ARK_OPT_EINVAL, "vocab = %llu: 1 to 2^28", (unsigned long long)vocab);
  if (columns == 0 || columns > 65536)
    return fail(ARK_OPT_EINVAL, "columns = %llu: 1 to 65536", (unsigned long long)columns);
  return ARK_OPT_OK;
}

int rows_bytes(uint64_t rows, uint64_t row, uint64_t stride, uint32_t es, bool written,
               const char* what, uint64_t* bytes) {
  *bytes = 0;
  if (rows == 0) return ARK_OPT_OK;
  if (rows > 1 && (stride >= (1ull << 31) || (rows - 1) * stride >= (1ull << 48)))
    return fail(ARK_OPT_EINVAL, "%s: stride %llu too large", what, (unsigned long long)stride);
  if (written && rows > 1 && stride < row)
    return fail(ARK_OPT_EINVAL, "%s: rows of %llu elements overlap at stride %llu", what,
                (unsigned long long)row, (unsigned long long)stride);
  *bytes = ((rows - 1) * stride + row) * es;
  return ARK_OPT_OK;
}

int check_types(uint32_t a, uint32_t b, uint32_t token_bytes) {
  if (a > ARK_EMBED_F32 || b > ARK_EMBED_F32)
    return fail(ARK_OPT_EINVAL, "dtype %u unknown", a > ARK_EMBED_F32 ? a : b);
  if (token_bytes != 4 && token_bytes != 8)
    return fail(ARK_OPT_EINVAL, "tokens of %u bytes: 4 or 8", token_bytes);
  return ARK_OPT_OK;
}

template <uint32_t IN, uint32_t OUT>
void launch_lookup(const LookupArgs& a, dim3 grid, hipStream_t s) {
  if (a.columns < 8)
    hipLaunchKernelGGL((lookup_short_kernel<IN, OUT>), grid, dim3(kLanes), 0, s, a);
  else
    hipLaunchKernelGGL((lookup_kernel<IN, OUT>), grid, dim3(kLanes), 0, s, a);
}
template <uint32_t IN>
void launch_lookup(const LookupArgs& a, uint32_t out, dim3 grid, hipStream_t s) {
  if (out == ARK_EMBED_F16)
    launch_lookup<IN, ARK_EMBED_F16>(a, grid, s);
  else if (out == ARK_EMBED_BF16)
    launch_lookup<IN, ARK_EMBED_BF16>(a, grid, s);
  else
    launch_lookup<IN, ARK_EMBED_F32>(a, grid, s);
}

dim3 blocks_of(uint64_t n) { return dim3((uint32_t)(n < kMostBlocks ? n : kMostBlocks)); }

template <uint32_t DT, bool WIDE>
int launch_sums(const SumArgs& a, hipStream_t s) {
  const uint64_t tiles = (a.columns + Column<WIDE>::kWave - 1) / Column<WIDE>::kWave;
  if (a.n == 0) {
    hipLaunchKernelGGL(zero_kernel<WIDE>, blocks_of((a.tokens.vocab * tiles + 3) / 4),
                       dim3(kLanes), 0, s, a);
    ARK_HIP(hipGetLastError());
    return ARK_OPT_OK;
  }
  const uint32_t blocks = (a.tokens.vocab + kFewRows - 1) / kFewRows;
  if (a.n <= kFew && blocks <= kMostBlocks) {
    const uint32_t tiles4 = (uint32_t)((tiles + kLanes / 64 - 1) / (kLanes / 64));
    hipLaunchKernelGGL((few_kernel<DT, WIDE>), dim3(blocks, tiles4), dim3(kLanes), 0, s, a);
    ARK_HIP(hipGetLastError());
    return ARK_OPT_OK;
  }
  const dim3 groups((a.tokens.vocab + kGroup - 1) / kGroup);
  if (a.n <= kSortLanes * kKept)
    hipLaunchKernelGGL(sort_kernel<true>, groups, dim3(kSortLanes), 0, s, a.tokens, a.n,
                       (uint32_t*)a.start, (uint32_t*)a.pos);
  else
    hipLaunchKernelGGL(sort_kernel<false>, groups, dim3(kSortLanes), 0, s, a.tokens, a.n,
                       (uint32_t*)a.start, (uint32_t*)a.pos);
  ARK_HIP(hipGetLastError());
  const uint64_t windows = a.n / kWindow * tiles;
  if (windows) {
    hipLaunchKernelGGL((window_kernel<DT, WIDE>), blocks_of((windows + 3) / 4), dim3(kLanes), 0,
                       s, a);
    ARK_HIP(hipGetLastError());
  }
  const uint64_t waves = ((uint64_t)a.tokens.vocab + kRows - 1) / kRows * tiles;
  hipLaunchKernelGGL((sum_kernel<DT, WIDE>), blocks_of((waves + 3) / 4), dim3(kLanes), 0, s, a);
  ARK_HIP(hipGetLastError());
  return ARK_OPT_OK;
}
template <uint32_t DT>
int launch_sums(const SumArgs& a, hipStream_t s) {
  return a.columns < 4 ? launch_sums<DT, false>(a, s) : launch_sums<DT, true>(a, s);
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
  a.scale = scale;
  const dim3 grid = blocks_of((n * (columns < 8 ? columns : (columns + 7) / 8) + kLanes - 1) / kLanes);
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
  a.accumulate = flags & ARK_EMBED_ACCUMULATE ? 1u : 0u;
  a.scale = scale;
  if (dy_dtype == ARK_EMBED_F16) return launch_sums<ARK_EMBED_F16>(a, s);
  if (dy_dtype == ARK_EMBED_BF16) return launch_sums<ARK_EMBED_BF16>(a, s);
  return launch_sums<ARK_EMBED_F32>(a, s);
}

}  // extern "C"
