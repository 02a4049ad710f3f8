/*
 * ark_act.h -- activations kept in 8 bits for the backward pass, on MI355X
 * (gfx950), and the weight gradient that reads them.  No counterpart in the
 * reference, which recomputes or keeps its activations inside MPSGraph.
 *
 * The 8-bit form of an array x of tokens rows and columns columns.  32
 * consecutive rows (ARK_ACT_GROUP; the last group may be shorter) of one
 * column share an exponent e, and each value keeps a whole number q:
 *
 *   a = max |x| over the group
 *   e = the smallest whole number with a <= 127 * 2^e, at least -24 (fp16) or
 *       -126 (bf16, fp32) and at most 121
 *   q = x / 2^e rounded to nearest, ties to even, held to |q| <= 127 (63 where
 *       e = 10 and x is fp16: 64 * 2^10 is not a finite fp16)
 *
 * and stands for q * 2^e, which is exact in x's type, in bf16 and in fp32.  A
 * group that holds an inf or a NaN reads back as NaN in all its values, so a
 * gradient formed from it is not finite and the optimizer step skips, as it
 * would have for x itself.
 *
 * Rows of a group follow one another in memory, so a column's outliers cost
 * other columns nothing, and the weight gradient, which sums over rows, finds
 * 32 values under one exponent.  The buffer (ark_act_bytes; any device memory
 * aligned to 16 bytes) holds, with G = ceil(tokens / 32), the bytes q + 128 as
 * [G][columns][32], rows past the last as q = 0, and then the bytes e + 133
 * (255: NaN) as [G][columns].
 *
 * Every function is stream ordered and returns an ARK_OPT_* status code
 * (include/ark_opt.h), with the message in ark_opt_last_error().  Pointers
 * are device pointers of the current device, and stream is one of its streams.
 * Row strides are in elements.
 */
#ifndef ARK_ACT_H
#define ARK_ACT_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
#define ARK_ACT_F16 0u
#define ARK_ACT_BF16 1u
#define ARK_ACT_F32 2u

#define ARK_ACT_GROUP 32 /* rows that share an exponent */

/* Bytes of the 8-bit form: 33 * ceil(tokens / 32) * columns. */
int ark_act_bytes(uint64_t tokens, uint64_t columns, uint64_t *bytes);

/* act <- x.  act must not overlap x. */
int ark_act_pack(const void *x, uint64_t x_stride, uint32_t dtype, uint64_t tokens,
                 uint64_t columns, void *act, void *stream);

/* x <- the values of act, rounded to dtype (exact in the type they were
 * packed from, in bf16 and in fp32).  Rows of x must not overlap each other
 * or act. */
int ark_act_unpack(const void *act, uint64_t tokens, uint64_t columns, uint32_t dtype, void *x,
                   uint64_t x_stride, void *stream);

/* Flags of ark_act_weight_grad. */
#define ARK_ACT_ACCUMULATE 1u /* add to dw instead of overwriting it */
#define ARK_ACT_TRANSPOSED 2u /* dw is [outputs][columns] */

/* The weight gradient of y = x w from x's 8-bit form and dy [tokens][outputs]:
 *   dw[c][o] (+)= sum over t of act[t][c] * dy[t][o]
 * with fp32 products' sums in an order that depends on the sizes alone, so a
 * call repeated gives the same bits.  dw is [columns][outputs] (the
 * order of the reference's weights, proyecto_ark/ark01/src/memory.rs:227-255)
 * or transposed.  act_dtype is the type act was
 * packed from; dy is fp16 (act packed from fp16) or bf16 (from any): every
 * product is then exact in fp32.  A sum of T products is within (T + 1) 2^-23 of
 * the sum of their magnitudes, in which, with fp16 dy, a dy below 2^-14 (but not
 * 0) counts as 2^-14 and an act more than 2^23 below its column's largest 2^e as
 * 2^-23 of that: additions align by the factors' exponent fields, and a
 * subnormal's is that of 2^-14.  (Such a dy is itself given to half a place of
 * 2^-25, 2^12 times as much.)  tokens = 0 writes zeros, or leaves an
 * accumulated dw as it is.  dw must not overlap act or dy; a dw that is a
 * gradient of an optimizer is one the step may read at once, on the same
 * stream. */
int ark_act_weight_grad(const void *act, uint32_t act_dtype, uint64_t tokens, uint64_t columns,
                        const void *dy, uint64_t dy_stride, uint32_t dy_dtype, uint64_t outputs,
                        float *dw, uint64_t dw_stride, uint32_t flags, void *stream);

/* ark_act_weight_grad with the same arguments and bits, for callers that keep
 * their own workspace (loops whose host time counts, code that cannot
 * allocate): ark_act_weight_grad_workspace bytes of device memory, aligned to
 * 16, that the call's work uses until it ends.  Few or one large sum need
 * none (0 bytes; workspace may then be NULL).  The other call takes such memory
 * from the library's kept slots or the stream-ordered pool. */
int ark_act_weight_grad_workspace(uint64_t tokens, uint64_t columns, uint64_t dy_stride,
                                  uint64_t outputs, uint64_t *bytes);
int ark_act_weight_grad_noalloc(const void *act, uint32_t act_dtype, uint64_t tokens,
                                uint64_t columns, const void *dy, uint64_t dy_stride,
                                uint32_t dy_dtype, uint64_t outputs, float *dw,
                                uint64_t dw_stride, uint32_t flags, void *workspace,
                                uint64_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* ARK_ACT_H */
