/*
 * ark_rope.h -- rotary positions, and the RMS norm of every query and key head
 * with the rotation in the same pass, forward and backward, on MI355X
 * (gfx950).
 *
 * The reference rotates its queries and keys inside its per-layer MPSGraph
 * (proyecto_ark/ark01/objc/bridge.m:229-411) and has no norm of heads.
 *
 * Arrays are [batch][tokens][heads][head_dim] in the order of their strides,
 * not necessarily of memory: a layout is four numbers,
 *   { heads, batch stride, token stride, head stride }   (elements),
 * and the head_dim values of a head follow one another.  Inputs may repeat
 * (stride 0); an output may be its input with the same layout (in place), or
 * must not share a byte with any other array of the call.
 *
 * Positions are int32 or int64 (position_bytes 4 or 8), one for each batch and
 * token, of any sign; positions = NULL means start + token.
 *
 * Rotation, with R = rotary_dim, pairs i < R / 2, a = position * inv_freq[i]
 * and m = magnitude:
 *   half:         (u, v) = (x[i], x[i + R/2])
 *   interleaved:  (u, v) = (x[2i], x[2i + 1])
 *   u' = m (u cos a - v sin a),   v' = m (u sin a + v cos a)
 * and x[R..head_dim) stays as it is.  The angle is formed in 64-bit fixed point
 * in turns: at any position it is as exact as inv_freq itself (no tables).
 *
 * Every function is stream ordered and returns an ARK_OPT_* status code
 * (include/ark_opt.h), with the message in ark_opt_last_error().  Pointers are
 * device pointers of the rotation's device, and stream is one of its streams.
 * Element types are ARK_ACT_F16, ARK_ACT_BF16 and ARK_ACT_F32
 * (include/ark_act.h); all arithmetic is fp32, rounded once where a result is
 * stored.
 */
#ifndef ARK_ROPE_H
#define ARK_ROPE_H

#include <stdint.h>

#include "ark_act.h"

#ifdef __cplusplus
extern "C" {
#endif

#define ARK_ROPE_HALF 0u
#define ARK_ROPE_INTERLEAVED 1u

#define ARK_ROPE_MAX_HEAD 512 /* largest head_dim */

/* Scalings of the frequencies for contexts longer than the trained one, and
 * their parameters, with f_i = base^(-2i/R):
 *   NONE    -
 *   LINEAR  { factor }: f_i / factor
 *   NTK     { factor }: base * factor^(R / (R - 2)) in place of base
 *   YARN    { factor, original length L, fast turns, slow turns }: pairs that
 *           turn more often than `fast` over L keep f_i, those below `slow`
 *           take f_i / factor, linear in i between floor and ceil of
 *           R ln(L / (2 pi turns)) / (2 ln base), held to 0 and R - 1;
 *           magnitude 0.1 ln(factor) + 1, and 1 for a factor up to 1
 *   BANDS   { factor, original length L, low, high }: with n = L f_i / (2 pi)
 *           turns, f_i where n > high, f_i / factor where n < low, and between
 *           them linear in n
 */
#define ARK_ROPE_SCALE_NONE 0u
#define ARK_ROPE_SCALE_LINEAR 1u
#define ARK_ROPE_SCALE_NTK 2u
#define ARK_ROPE_SCALE_YARN 3u
#define ARK_ROPE_SCALE_BANDS 4u

/* inv_freq[0 .. rotary_dim / 2) and *magnitude of a scaling (host only). */
int ark_rope_frequencies(uint32_t rotary_dim, double base, uint32_t scaling, const double *params,
                         double *inv_freq, double *magnitude);

/* A model's rotation: head_dim up to ARK_ROPE_MAX_HEAD, rotary_dim even and at
 * most head_dim (0: no rotation), its frequencies copied to the current
 * device. */
typedef struct ark_rope ark_rope;
int ark_rope_create(uint32_t head_dim, uint32_t rotary_dim, uint32_t layout,
                    const double *inv_freq, double magnitude, ark_rope **out);
int ark_rope_destroy(ark_rope *rope);

/* q_out <- q rotated and, unless k_layout is NULL, k_out <- k rotated.  inverse != 0
 * applies the transpose, which takes gradients of q_out and k_out to those of
 * q and k. */
int ark_rope_apply(const ark_rope *rope, uint32_t dtype, uint64_t batch, uint64_t tokens,
                   const void *positions, uint32_t position_bytes, uint64_t start, const void *q,
                   const uint64_t *q_layout, void *q_out, const uint64_t *q_out_layout,
                   const void *k, const uint64_t *k_layout, void *k_out,
                   const uint64_t *k_out_layout, uint32_t inverse, void *stream);

/* n[j] = x[j] / sqrt(mean(x^2) + eps) * gain[j] for every head of q and k
 * (gain_q, gain_k: head_dim values of gain_dtype), then the rotation; q alone
 * where k_layout is NULL.  With
 * q_act (and k_act) not NULL, the 8-bit form of q (of k) as ark_act_pack gives
 * it for tokens = batch * tokens rows of heads * head_dim columns is written
 * in the same call. */
int ark_rope_norm(const ark_rope *rope, uint32_t dtype, uint64_t batch, uint64_t tokens,
                  const void *positions, uint32_t position_bytes, uint64_t start, float eps,
                  const void *gain_q, const void *gain_k, uint32_t gain_dtype, const void *q,
                  const uint64_t *q_layout, void *q_out, const uint64_t *q_out_layout,
                  void *q_act, const void *k, const uint64_t *k_layout, void *k_out,
                  const uint64_t *k_out_layout, void *k_act, void *stream);

/* The gradients of ark_rope_norm: from dq (the gradient of q_out) and the q the
 * norm was given, or with q_act not NULL its 8-bit form (q is then unused), to
 * q_grad, the gradient of q, and dgain_q, the gradient of gain_q in fp32,
 * summed over batch, tokens and heads in an order that depends on the sizes
 * alone; the same for k unless dk_layout is NULL.  accumulate != 0 adds to dgain_q
 * and dgain_k instead of overwriting them.  q_grad may be dq (in place). */
int ark_rope_norm_backward(const ark_rope *rope, uint32_t dtype, uint64_t batch, uint64_t tokens,
                           const void *positions, uint32_t position_bytes, uint64_t start,
                           float eps, const void *gain_q, const void *gain_k,
                           uint32_t gain_dtype, const void *dq, const uint64_t *dq_layout,
                           const void *q, const uint64_t *q_layout, const void *q_act,
                           void *q_grad, const uint64_t *q_grad_layout, float *dgain_q,
                           const void *dk, const uint64_t *dk_layout, const void *k,
                           const uint64_t *k_layout, const void *k_act, void *k_grad,
                           const uint64_t *k_grad_layout, float *dgain_k, uint32_t accumulate,
                           void *stream);

#ifdef __cplusplus
}
#endif

#endif /* ARK_ROPE_H */
