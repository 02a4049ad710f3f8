// ark_act.hip -- activations kept in 8 bits and the weight gradient that reads
// them (include/ark_act.h).
#include "ark_act.hpp"
#include "ark_common.hpp"

namespace {

using namespace ark::dev;

constexpr uint32_t kLanes = 256;

// One lane per column of a group: 32 loads, the largest magnitude, 32 bytes.
template <uint32_t DT>
__global__ __launch_bounds__(kLanes) void pack_kernel(const elem_t<DT>* __restrict__ x,
                                                      uint64_t stride, uint64_t tokens,
                                                      uint32_t columns, uint8_t* __restrict__ q,
                                                      uint8_t* __restrict__ e) {
  const uint32_t c = blockIdx.x * kLanes + threadIdx.x;
  const uint64_t g = blockIdx.y + (uint64_t)gridDim.y * blockIdx.z;
  const uint64_t t0 = g * ARK_ACT_GROUP;
  if (c >= columns || t0 >= tokens) return;
  const uint32_t n = (uint32_t)(tokens - t0 < ARK_ACT_GROUP ? tokens - t0 : ARK_ACT_GROUP);
  const elem_t<DT>* row = x + t0 * stride + c;
  float v[ARK_ACT_GROUP];
  uint32_t most = 0;
#pragma unroll
  for (uint32_t i = 0; i < ARK_ACT_GROUP; ++i) {
    v[i] = i < n ? (float)row[i * stride] : 0.0f;
    const uint32_t a = __float_as_uint(v[i]) & 0x7FFFFFFFu;
    most = a > most ? a : most;
  }
  const uint32_t s = act_exponent<DT>(most);
  const float down = act_down(s);
  uint32_t w[ARK_ACT_GROUP / 4] = {};
#pragma unroll
  for (uint32_t i = 0; i < ARK_ACT_GROUP; ++i)
    w[i / 4] |= act_byte<DT>(v[i], s, down) << (i % 4 * 8);
  u32x4* out = (u32x4*)(q + (g * columns + c) * ARK_ACT_GROUP);
  out[0] = u32x4{w[0], w[1], w[2], w[3]};
  out[1] = u32x4{w[4], w[5], w[6], w[7]};
  e[g * columns + c] = (uint8_t)s;
}

template <uint32_t DT>
__global__ __launch_bounds__(kLanes) void unpack_kernel(const uint8_t* __restrict__ q,
                                                        const uint8_t* __restrict__ e,
                                                        uint64_t tokens, uint32_t columns,
                                                        elem_t<DT>* __restrict__ x,
                                                        uint64_t stride) {
  const uint32_t c = blockIdx.x * kLanes + threadIdx.x;
  const uint64_t g = blockIdx.y + (uint64_t)gridDim.y * blockIdx.z;
  const uint64_t t0 = g * ARK_ACT_GROUP;
  if (c >= columns || t0 >= tokens) return;
  const uint32_t n = (uint32_t)(tokens - t0 < ARK_ACT_GROUP ? tokens - t0 : ARK_ACT_GROUP);
  const u32x4* in = (const u32x4*)(q + (g * columns + c) * ARK_ACT_GROUP);
  const u32x4 a = in[0], b = in[1];
  const float up = act_up(e[g * columns + c]);
  elem_t<DT>* row = x + t0 * stride + c;
#pragma unroll
  for (uint32_t i = 0; i < ARK_ACT_GROUP; ++i) {
    const uint32_t w = i < 16 ? a[i / 4] : b[i / 4 - 4];
    if (i < n) row[i * stride] = narrow<elem_t<DT>>(act_value(w >> (i % 4 * 8) & 255u, up));
  }
}

// 16 x 16 outputs a block, one a lane; both operands' tiles staged in LDS one
// group of rows at a time.
template <typename T>
__global__ __launch_bounds__(256) void grad_kernel(const uint8_t* __restrict__ q,
                                                   const uint8_t* __restrict__ e, uint64_t tokens,
                                                   uint32_t columns, const T* __restrict__ dy,
                                                   uint64_t dy_stride, uint32_t outputs,
                                                   float* __restrict__ dw, uint64_t dw_stride,
                                                   uint32_t flags) {
  __shared__ float xs[16][ARK_ACT_GROUP + 1], ys[ARK_ACT_GROUP][17];
  const uint32_t lc = threadIdx.x / 16, lo = threadIdx.x % 16;
  const uint32_t c = blockIdx.x * 16 + lc, o = blockIdx.y * 16 + lo;
  float sum = 0.0f;
  for (uint64_t t0 = 0, g = 0; t0 < tokens; t0 += ARK_ACT_GROUP, ++g) {
    for (uint32_t i = threadIdx.x; i < 16 * ARK_ACT_GROUP; i += 256) {
      const uint32_t cc = i / ARK_ACT_GROUP, t = i % ARK_ACT_GROUP;
      const uint32_t col = blockIdx.x * 16 + cc;
      xs[cc][t] = col < columns ? act_value(q[(g * columns + col) * ARK_ACT_GROUP + t],
                                            act_up(e[g * columns + col]))
                                : 0.0f;
      const uint32_t tt = i / 16, oo = blockIdx.y * 16 + i % 16;
      ys[tt][i % 16] = t0 + tt < tokens && oo < outputs ? (float)dy[(t0 + tt) * dy_stride + oo]
                                                        : 0.0f;
    }
    __syncthreads();
    for (uint32_t t = 0; t < ARK_ACT_GROUP; ++t) sum = __builtin_fmaf(xs[lc][t], ys[t][lo], sum);
    __syncthreads();
  }
  if (c < columns && o < outputs) {
    float* p = dw + (flags & ARK_ACT_TRANSPOSED ? o * dw_stride + c : c * dw_stride + o);
    *p = flags & ARK_ACT_ACCUMULATE ? *p + sum : sum;
  }
}

int check_dtype(uint32_t dtype, const char* what) {
  if (dtype > ARK_ACT_F32) return ark::fail(ARK_OPT_EINVAL, "%s %u unknown", what, dtype);
  return ARK_OPT_OK;
}

// Sizes for which no address below wraps: at most 2^32 - 1 columns and 2^47
// values, so any byte offset fits 64 bits with room to spare.
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

// Blocks over groups in y and z: y stays within a launch's 65535.
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
  const uint32_t es = ark::act_elem_size(dtype);
  if ((uintptr_t)x % es) return ark::fail(ARK_OPT_EINVAL, "x not aligned to its element");
  if ((rc = rows_bytes(tokens, columns, x_stride, es, unpack, "x", x_bytes))) return rc;
  if (ark::overlaps(x, *x_bytes, act, 33 * ark::act_groups(tokens) * columns))
    return ark::fail(ARK_OPT_EINVAL, "x and act overlap");
  ark::BufferChecker checker;
  if ((rc = check_act(act, tokens, columns, &checker))) return rc;
  return checker.check(x, *x_bytes, "x", 0);
}

template <uint32_t DT>
void launch_pack(const void* x, uint64_t stride, uint64_t tokens, uint64_t columns, uint8_t* act,
                 hipStream_t s) {
  const uint64_t groups = ark::act_groups(tokens);
  hipLaunchKernelGGL(pack_kernel<DT>, group_grid((columns + kLanes - 1) / kLanes, groups),
                     dim3(kLanes), 0, s, (const elem_t<DT>*)x, stride, tokens, (uint32_t)columns,
                     act, act + groups * columns * ARK_ACT_GROUP);
}

template <uint32_t DT>
void launch_unpack(const uint8_t* act, uint64_t tokens, uint64_t columns, void* x, uint64_t stride,
                   hipStream_t s) {
  const uint64_t groups = ark::act_groups(tokens);
  hipLaunchKernelGGL(unpack_kernel<DT>, group_grid((columns + kLanes - 1) / kLanes, groups),
                     dim3(kLanes), 0, s, act, act + groups * columns * ARK_ACT_GROUP, tokens,
                     (uint32_t)columns, (elem_t<DT>*)x, stride);
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
  ark::BufferChecker checker;
  if (tokens && (rc = check_act(act, tokens, columns, &checker))) return rc;
  if ((rc = checker.check(dy, dyb, "dy", 0))) return rc;
  if ((rc = checker.check(dw, dwb, "dw", 0))) return rc;
  {
    const void* d = dw;  // dw may be an optimizer's gradient
    ark::opt_units_invalidate(&d, &dwb, 1);
  }
  const hipStream_t s = (hipStream_t)stream;
  const uint8_t* q = (const uint8_t*)act;
  const uint8_t* e = q + ark::act_groups(tokens) * columns * ARK_ACT_GROUP;
  const dim3 grid((uint32_t)((columns + 15) / 16), (uint32_t)((outputs + 15) / 16));
  if (dy_dtype == ARK_ACT_F16)
    hipLaunchKernelGGL(grad_kernel<_Float16>, grid, dim3(256), 0, s, q, e, tokens,
                       (uint32_t)columns, (const _Float16*)dy, dy_stride, (uint32_t)outputs, dw,
                       dw_stride, flags);
  else
    hipLaunchKernelGGL(grad_kernel<__bf16>, grid, dim3(256), 0, s, q, e, tokens,
                       (uint32_t)columns, (const __bf16*)dy, dy_stride, (uint32_t)outputs, dw,
                       dw_stride, flags);
  ARK_HIP(hipGetLastError());
  return ARK_OPT_OK;
}

}  // extern "C"
