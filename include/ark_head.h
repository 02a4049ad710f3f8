/*
 * ark_head.h -- the loss over a vocabulary from a model's last hidden rows and
 * its output layer, and the gradients of both, on MI355X (gfx950).  The logits
 * are never in memory; the gradients' dz, of their size in 16 bits, is, in pieces.
 * The reference forms the logits with a tied 1x1 convolution
 * (proyecto_ark/ark01/objc/bridge.m:414-503) and its cross entropy on the CPU
 * (:954-976); these are this library's own definitions.
 *
 * x is [tokens][columns], w [vocab][columns] (the tied embedding), both fp16 or
 * both bf16, and the logits are z = scale * x w^T, summed in fp32.
 *
 * Cross entropy: a token with a target y has
 *     loss = log(sum over v of exp(z_v)) - z_y
 *     dz_v = grad * scale * (softmax(z)_v - [v = y])
 * A token whose target is `ignore`, or outside [0, vocab), has loss 0, no
 * gradient, and its row of x is not used: NaN there reaches nothing.
 *
 * Distillation: a token with `top` entries (index, logit) of a teacher has the
 * divergence of the student's distribution q = softmax(z), z = x w^T /
 * temperature, from the teacher's p = softmax(logit / temperature) over the
 * entries:
 *     loss = sum over k of p_k (log p_k - log q_index_k)
 *     dz_v = grad / temperature * (q_v - sum over k of p_k [v = index_k])
 * Entries whose index is outside [0, vocab) are left out, whatever their logit;
 * those of logit -inf count for nothing; an index that comes twice counts twice.
 * A token with no entry, or only such of logit -inf, has loss 0 and no gradient.
 * (The factor temperature^2 that keeps gradients' sizes alike is the caller's,
 * in grad.)
 *
 * The gradients of x and w are
 *     dx = dz w          in x's type
 *     dw (+)= dz^T x     in fp32, or in w's type (not added to)
 * dz is rounded to the 16 bits of x's type, relative to the largest gradient, which is
 * taken as 2^14; until a row's sum is known its exponentials are kept in 16 bits of
 * their own, to 2^-13 (fp16) or 2^-10 (bf16) of each, a quarter of what dz's rounding is
 * off by.  With at most 64 tokens, whose sums show a rounding in full, what is left of dz
 * is 16 bits of its own in the products too.
 * Entries at targets are formed in fp32.  A loss or gradient formed
 * from an inf or NaN is not finite, and the optimizer step then skips; other tokens'
 * losses and dx stay what they are.  (A token whose grad * scale is past fp32's range
 * does not count for the largest gradient either.)  Sums run
 * in an order that depends on the sizes and on which tokens have a loss: equal
 * calls give equal bits.
 *
 * A call works through the tokens in pieces, whose copied rows and 16-bit dz (of the
 * logits' size, at most 1 GiB; for the loss alone sums of 64 or 128 logits each, at most
 * 1 GiB) lie in the caller's workspace (ark_head_workspace), in use until the call's
 * work ends.  Tokens without a loss cost no products.
 *
 * Every function is stream ordered and returns an ARK_OPT_* status code
 * (include/ark_opt.h), with the message in ark_opt_last_error().  Pointers are
 * device pointers of the current device, and stream is one of its streams.
 * Strides are in elements, below 2^32, and w's below 2^22.  columns are 1 to 65536,
 * vocab 1 to 2097152, tokens below 2^31; scale and 1 / temperature are positive and
 * below 2^126.
 */
#ifndef ARK_HEAD_H
#define ARK_HEAD_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types: of x, w (ARK_HEAD_F16, ARK_HEAD_BF16), dw and a teacher's logits. */
#define ARK_HEAD_F16 0u
#define ARK_HEAD_BF16 1u
#define ARK_HEAD_F32 2u

#define ARK_HEAD_MAX_TOP 256 /* entries of a teacher's distribution */

/* Flags. */
#define ARK_HEAD_ACCUMULATE 1u /* add to dw (fp32) instead of overwriting it */

/* What a call forms besides the loss, for its workspace. */
#define ARK_HEAD_DX 1u
#define ARK_HEAD_DW 2u
#define ARK_HEAD_GRAD 4u

/* Bytes of workspace of a call: top is 1 for cross entropy; grad is 0 for the
 * loss alone, otherwise ARK_HEAD_GRAD, with ARK_HEAD_DX and ARK_HEAD_DW for the
 * gradients that are formed.  The address and stride of w count, as the
 * products read w itself where rows of 16-byte pieces allow it and a copy
 * otherwise. */
int ark_head_workspace(const void *w, uint64_t w_stride, uint64_t tokens, uint64_t columns,
                       uint64_t vocab, uint64_t top, uint32_t dw_dtype, uint32_t grad,
                       uint64_t *bytes);

/* loss[t] for every token.  targets are int32 (target_bytes 4) or int64 (8). */
int ark_head_cross_entropy(const void *x, uint64_t x_stride, const void *w, uint64_t w_stride,
                           uint32_t dtype, uint64_t tokens, uint64_t columns, uint64_t vocab,
                           const void *targets, uint32_t target_bytes, int32_t ignore, float scale,
                           float *loss, void *workspace, uint64_t workspace_bytes, void *stream);

/* The same, and the gradients, times grads[t] for each token, or grad for all
 * when grads is NULL.  dx or dw may be NULL: not formed.  dw is fp32
 * (ARK_HEAD_F32) or of w's type; one that is a gradient of an optimizer may be
 * stepped on at once, on the same stream.  No written array may overlap another
 * one or an input.  tokens = 0 writes zeros to dw, or leaves an accumulated dw. */
int ark_head_cross_entropy_grad(const void *x, uint64_t x_stride, const void *w, uint64_t w_stride,
                                uint32_t dtype, uint64_t tokens, uint64_t columns, uint64_t vocab,
                                const void *targets, uint32_t target_bytes, int32_t ignore,
                                float scale, float grad, const float *grads, float *loss, void *dx,
                                uint64_t dx_stride, void *dw, uint32_t dw_dtype,
                                uint64_t dw_stride, uint32_t flags, void *workspace,
                                uint64_t workspace_bytes, void *stream);

/* Distillation: index (int32 or int64) and logits (fp16, bf16 or fp32) are
 * [tokens][top], top <= ARK_HEAD_MAX_TOP, rows of any stride. */
int ark_head_distill(const void *x, uint64_t x_stride, const void *w, uint64_t w_stride,
                     uint32_t dtype, uint64_t tokens, uint64_t columns, uint64_t vocab,
                     const void *index, uint32_t index_bytes, uint64_t index_stride,
                     const void *logits, uint32_t logits_dtype, uint64_t logits_stride,
                     uint64_t top, float temperature, float *loss, void *workspace,
                     uint64_t workspace_bytes, void *stream);
int ark_head_distill_grad(const void *x, uint64_t x_stride, const void *w, uint64_t w_stride,
                          uint32_t dtype, uint64_t tokens, uint64_t columns, uint64_t vocab,
                          const void *index, uint32_t index_bytes, uint64_t index_stride,
                          const void *logits, uint32_t logits_dtype, uint64_t logits_stride,
                          uint64_t top, float temperature, float grad, const float *grads,
                          float *loss, void *dx, uint64_t dx_stride, void *dw, uint32_t dw_dtype,
                          uint64_t dw_stride, uint32_t flags, void *workspace,
                          uint64_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* ARK_HEAD_H */
