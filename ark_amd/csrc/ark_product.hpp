// ark_product.hpp -- a block's tile of a matrix product of 16-bit operands on
// gfx950's matrix instructions, from operands in either order in memory.
//
//   out[n][m] = sum over k of a[m][k] b[n][k], in fp32
//
// An operand lies in memory with k along its rows (KC: a row is an m or n, its k
// follow one another) or across them (MC: a row is a k).  A block forms BM x BN
// outputs, a wave 16 MF x 16 NF of them; a lane ends up with four neighbouring m
// of one n.  A step is 32 k of both operands, which go from memory into LDS
// without passing through registers (global_load_lds), into one of BUFS buffers.
//
// LDS holds a KC operand as rows of 32 k, four 16-byte chunks each, permuted by
// the row's bits so that a fragment's 16-byte reads meet in no bank, and an MC
// operand as it comes, rows of BM or BN values; its fragments are read through
// the transposing read, which gives lane i of sixteen the values of column i in
// four rows, its 32-byte pieces permuted by the row's bits for the same reason.
// As loads into LDS write 64 x 16 bytes in lane order, the permutations are of
// the addresses that are loaded from.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "ark_device.hpp"

namespace ark {
namespace dev {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

#define ARK_LDS_AT(T, byte) (*(__attribute__((address_space(3))) T*)(uintptr_t)(byte))

template <typename T>
struct Frag;
template <>
struct Frag<_Float16> {
  typedef f16x8 V;
  static __device__ __forceinline__ f32x4 mul(V a, V b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Frag<__bf16> {
  typedef bf16x8 V;
  static __device__ __forceinline__ f32x4 mul(V a, V b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

constexpr uint32_t kProductStep = 32;  // k a step

// An operand of one block: `at` is its first value (of the tile's first row and
// first k when KC, of the first k's row and the tile's first column when MC).
struct Operand {
  const uint16_t* at;
  uint64_t stride;  // of its rows, in elements, below 2^22
  uint32_t rows;    // KC: rows from `at` on that may be read; MC: values of a row, at least 8
  uint32_t ks;      // MC: rows from the first k on that may be read
};

// B rows (KC) or columns (MC) of an operand, staged by LANES lanes.
template <uint32_t B, bool MC, uint32_t LANES>
struct Staged {
  static constexpr uint32_t kBytes = B * kProductStep * 2;
  static constexpr uint32_t kLoads = kBytes / (LANES * 16);
  static_assert(kLoads * LANES * 16 == kBytes, "whole loads");
  static constexpr uint32_t kRow = MC ? B * 2 : kProductStep * 2;  // bytes of a row in LDS
  uint32_t off[kLoads];  // bytes from the step's first value

  static __device__ __forceinline__ uint32_t swizzle(uint32_t row) {
    if constexpr (MC) return ((row & 3u) | (row >> 3 & 1u) << 2) & (B / 16 - 1);
    // LDS takes 16-byte reads sixteen lanes at a time, of each 32 lanes 0-3, 12-15 and
    // 20-27 and then the others (measured: which pairs meet); lanes 16 on are a chunk
    // on.  Four rows are 256 bytes, a row of all banks: of rows 4 apart the four that
    // are read together get four different places.
    return ((row >> 2 ^ row >> 3) & 1u) << 1 | (row >> 3 & 1u);
  }
  // The offsets; of an MC operand's rows past `ks` from the step's first, the
  // last one's again.
  __device__ __forceinline__ void place(const Operand& o, uint32_t ks) {
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) {
      const uint32_t q = i * LANES + threadIdx.x, row = q / (kRow / 16), pos = q % (kRow / 16);
      if constexpr (MC) {
        const uint32_t col = ((pos / 2) ^ swizzle(row)) * 16 + pos % 2 * 8;
        off[i] = (min(row, ks - 1u) * (uint32_t)o.stride + min(col, o.rows - 8u)) * 2;
      } else {
        off[i] = (min(row, o.rows - 1u) * (uint32_t)o.stride + (pos ^ swizzle(row)) * 8) * 2;
      }
    }
  }
  // The k of `step`, into LDS at byte `to`.  The load writes LDS at m0
  // plus 16 bytes a lane; nothing returns to registers, and meet() waits for it by
  // count.  (One wait state between m0 and a load; the first load's others are those
  // between a vector instruction that writes an address's scalar registers and a load
  // that reads them, which the compiler does not see inside the block.)
  __device__ __forceinline__ void load(const Operand& o, uint32_t step, uint32_t to) {
    const uint16_t* p = o.at + (uint64_t)step * kProductStep * (MC ? o.stride : 1);
    if constexpr (MC) {
      const uint32_t left = o.ks - step * kProductStep;
      if (left < kProductStep) place(o, left);
    }
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) {
      const uint32_t at = to + (i * LANES + wave * 64) * 16;
      if (i == 0)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2"
                     :
                     : "s"(at), "v"(off[i]), "s"(p));
      else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                     :
                     : "s"(at), "v"(off[i]), "s"(p));
    }
  }
};

// Where a lane reads fragment f (16 rows or columns) of a wave's part.
template <typename T, uint32_t B, bool MC>
struct Reader {
  uint32_t at;
  // first: the wave's first row or column, a multiple of 16 times its fragments,
  // of which there is a power of two
  __device__ __forceinline__ explicit Reader(uint32_t first) {
    const uint32_t lane = threadIdx.x % 64, i = lane % 16, g = lane / 16;
    typedef Staged<B, MC, 64> S;
    if constexpr (MC) {
      const uint32_t row = 8 * g + i / 4;
      at = row * S::kRow + ((first * 2) ^ (S::swizzle(row) * 32)) + i % 4 * 8;
    } else {
      at = (first + i) * S::kRow + (g ^ S::swizzle(first + i)) * 16;
    }
  }
  __device__ __forceinline__ typename Frag<T>::V get(uint32_t buf, uint32_t f) const {
    typedef typename Frag<T>::V V;
    typedef Staged<B, MC, 64> S;
    if constexpr (MC) {
      const uint32_t a = buf + (at ^ (f * 32));
      typedef __attribute__((address_space(3))) s16x4 L;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L*)(uintptr_t)a);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L*)(uintptr_t)(a + 4 * S::kRow));
      return __builtin_bit_cast(V, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    return ARK_LDS_AT(V, buf + at + f * 16 * S::kRow);
  }
};

// A block's shape: WM x WN waves of MF x NF fragments, BUFS steps in LDS.
template <typename T_, bool AMC_, bool BMC_, uint32_t MF_, uint32_t NF_, uint32_t WM_, uint32_t WN_,
          uint32_t BUFS_>
struct Product {
  typedef T_ T;
  static constexpr uint32_t MF = MF_, NF = NF_, WM = WM_, WN = WN_, BUFS = BUFS_;
  static constexpr bool AMC = AMC_, BMC = BMC_;
  static constexpr uint32_t kLanes = 64 * WM * WN;
  static constexpr uint32_t BM = 16 * MF * WM, BN = 16 * NF * WN;
  typedef Staged<BM, AMC, kLanes> A;
  typedef Staged<BN, BMC, kLanes> B;
  static constexpr uint32_t kBuffer = A::kBytes + B::kBytes;
  static constexpr uint32_t kLds = BUFS * kBuffer;
  static constexpr uint32_t kLoads = A::kLoads + B::kLoads;
  static_assert(BUFS >= 3, "one read, one arriving, one asked for");

  f32x4 acc[MF][NF];

  // All but the newest `left` loads of this wave have arrived, and so have every
  // other wave's.
  template <uint32_t LEFT>
  static __device__ __forceinline__ void meet() {
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" : : "n"(LEFT) : "memory");
  }

  // acc = the product over steps [s0, s1).  lds: kLds bytes, aligned to 1024; the
  // caller's to use again after a barrier.
  __device__ __forceinline__ void run(const Operand& oa, const Operand& ob, uint32_t s0,
                                      uint32_t s1, uint32_t lds) {
#pragma unroll
    for (uint32_t i = 0; i < MF; ++i)
#pragma unroll
      for (uint32_t j = 0; j < NF; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    if (s0 >= s1) return;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    A a;
    B b;
    a.place(oa, kProductStep);
    b.place(ob, kProductStep);
    const Reader<T, BM, AMC> ra(wave % WM * 16 * MF);
    const Reader<T, BN, BMC> rb(wave / WM * 16 * NF);
    typename Frag<T>::V fa[MF], fb[2][NF];
    const auto load = [&](uint32_t s, uint32_t buf) __attribute__((always_inline)) {
      a.load(oa, s, buf);
      b.load(ob, s, buf + A::kBytes);
    };
    const uint32_t end = lds + kLds;
    uint32_t to = lds;  // the buffer of the next load
    const auto next = [&](uint32_t buf) { return buf + kBuffer == end ? lds : buf + kBuffer; };
    uint32_t s = s0;
    for (; s < s1 && s < s0 + BUFS - 1; ++s) load(s, to), to = next(to);
    if (s1 - s0 >= BUFS - 1)
      meet<(BUFS - 2) * kLoads>();
    else
      meet<0>();
    uint32_t from = lds;  // the buffer of the next fragments
    const auto read_b = [&](auto set) __attribute__((always_inline)) {
#pragma unroll
      for (uint32_t j = 0; j < NF; ++j) fb[decltype(set)::value][j] = rb.get(from + A::kBytes, j);
    };
    // A step is multiplied from registers while the next one's fragments take their
    // places: b's into the other set, each of a's when its products are done.  The
    // barrier before says that the next step is there, and that the buffer of the one
    // before is free: its fragments have been multiplied.  (The last step reads what
    // is in the buffer after its own and does not use it.)
    s = s0;
    const auto step = [&](auto set) __attribute__((always_inline)) {
      constexpr uint32_t p = decltype(set)::value;
      if (s + BUFS - 1 <= s1)
        meet<(BUFS - 3) * kLoads>();
      else
        meet<0>();
#pragma unroll
      for (uint32_t i = 0; i < MF; ++i) {
#pragma unroll
        for (uint32_t j = 0; j < NF; ++j) acc[i][j] = Frag<T>::mul(fa[i], fb[p][j], acc[i][j]);
        __builtin_amdgcn_sched_barrier(0);
        // between the products, so that they start right behind the barrier
        if (i == 0) read_b(std::integral_constant<uint32_t, p ^ 1>());
        fa[i] = ra.get(from, i);
        if (i == 1 && s + BUFS - 1 < s1) load(s + BUFS - 1, to), to = next(to);
        __builtin_amdgcn_sched_barrier(0);
      }
      from = next(from);
      ++s;
    };
    const auto first = [&](auto set) __attribute__((always_inline)) {
      read_b(set);
#pragma unroll
      for (uint32_t i = 0; i < MF; ++i) fa[i] = ra.get(from, i);
      from = next(from);
    };
    typedef std::integral_constant<uint32_t, 0> S0;
    typedef std::integral_constant<uint32_t, 1> S1;
    if ((s1 - s0) % 2) {
      first(S1());
      step(S1());
    } else {
      first(S0());
    }
    // nothing on its way from LDS that the compiler would wait for in the loop
    __builtin_amdgcn_s_waitcnt(0xC07F);
    while (s < s1) {
      step(S0());
      step(S1());
    }
  }

  // f(m, n, v): four outputs at m .. m + 3 of row n, both from the tile's start.  They
  // pass through LDS (the block's own again, after a barrier), sixteen rows of a wave
  // at a time, so that neighbouring lanes have neighbouring m: a row's come as whole
  // lines of memory (1.3B gradients 3.50 ms, 3.58 straight from the sums' lanes).
  template <typename F>
  __device__ __forceinline__ void each(uint32_t lds, F f) const {
    constexpr uint32_t kRowBytes = MF * 64, kChunks = kRowBytes / 16, kMask = kChunks < 16 ? kChunks - 1 : 15;
    static_assert(16 * kRowBytes * WM * WN <= kLds, "a part of LDS for each wave");
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, row = lane % 16;
    const uint32_t mine = lds + wave * 16 * kRowBytes;
    const uint32_t m0 = wave % WM * 16 * MF, n0 = wave / WM * 16 * NF;
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < NF; ++j) {
#pragma unroll
      for (uint32_t i = 0; i < MF; ++i)
        ARK_LDS_AT(f32x4, mine + row * kRowBytes + ((i * 4 + lane / 16) ^ (row & kMask)) * 16) =
            acc[i][j];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (uint32_t i = 0; i < kRowBytes / 64; ++i) {
        const uint32_t q = i * 64 + lane, r = q / kChunks, c = q % kChunks;
        f(m0 + c * 4, n0 + j * 16 + r,
          ARK_LDS_AT(f32x4, mine + r * kRowBytes + (c ^ (r & kMask)) * 16));
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
};

}  // namespace dev
}  // namespace ark
