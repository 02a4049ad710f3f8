/*
 * ark_embed.h -- the lookup of tokens in an embedding table and its gradient, on
 * MI355X (gfx950).  The reference gathers rows on the CPU (proyecto_ark/ark01/
 * asm/kern.s) and scatters their gradients back there (objc/bridge.m:922-928;
 * ark_grad_embed_scatter is that loop, bit for bit); these are this library's own
 * definitions, for rows of any type, scaled.
 *
 *   out[t] = scale * table[tokens[t]]            in fp32, rounded to out's type
 *   dw[v] (+)= scale * sum over t with tokens[t] = v of dy[t]      in fp32
 *
 * A token outside [0, vocab) has no row: its out is zeros, and its dy is not read.
 *
 * The gradient's sums are of fp32: positions of a token in increasing order, by
 * groups of 16 whose sums are added in order, so equal calls give equal bits, and
 * a sum of n rows is within (min(n, 64) + n / 16 + 2) 2^-24 of the sum of their
 * magnitudes.
 *
 * Every function is stream ordered and returns an ARK_OPT_* status code
 * (include/ark_opt.h), with the message in ark_opt_last_error().  Pointers are
 * device pointers of the current device, and stream is one of its streams.
 * Strides are of rows, in elements, below 2^31; tokens are int32 (token_bytes 4) or
 * int64 (8).  n is below 2^31, vocab 1 to 2^28, columns 1 to 65536.
 */
#ifndef ARK_EMBED_H
#define ARK_EMBED_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
#define ARK_EMBED_F16 0u
#define ARK_EMBED_BF16 1u
#define ARK_EMBED_F32 2u

/* Flags. */
#define ARK_EMBED_ACCUMULATE 1u /* add to dw instead of overwriting all of it */

/* table is [vocab][columns], out [n][columns]; out overlaps neither table nor
 * tokens. */
int ark_embed_lookup(const void *table, uint64_t table_stride, uint32_t table_dtype,
                     uint64_t vocab, uint64_t columns, const void *tokens, uint32_t token_bytes,
                     uint64_t n, float scale, void *out, uint64_t out_stride, uint32_t out_dtype,
                     void *stream);

/* Bytes of workspace of the gradient. */
int ark_embed_grad_workspace(uint64_t n, uint64_t vocab, uint64_t columns, uint64_t *bytes);

/* dy is [n][columns], dw fp32 [vocab][columns]; dw, which may be a gradient of an
 * optimizer, overlaps nothing else.  With ARK_EMBED_ACCUMULATE rows of tokens that
 * do not occur stay as they are, otherwise they become zeros.  workspace: device
 * memory aligned to 16 bytes, in use until the call's work ends. */
int ark_embed_grad(const void *dy, uint64_t dy_stride, uint32_t dy_dtype, const void *tokens,
                   uint32_t token_bytes, uint64_t n, uint64_t vocab, uint64_t columns, float scale,
                   float *dw, uint64_t dw_stride, uint32_t flags, void *workspace,
                   uint64_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* ARK_EMBED_H */
