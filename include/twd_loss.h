/*
 * twd_loss.h -- C-ABI of an LM head's softmax cross entropy with its gradients on MI355X (gfx950), without the logits
 * being kept. Conventions as in twd_head.h (status codes, twd_last_error, device pointers, streams); types as in twd_mx.h.
 */
#ifndef TWD_LOSS_H
#define TWD_LOSS_H

#include "twd_mx.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- softmax cross entropy of a head's logits --------------------------------------------------
 * No counterpart in the reference. With hidden rows h_m and a head's weights w_v, both bf16:
 *   z_mv = softcap(h_m . w_v),  lse_m = ln sum_v exp(z_mv),  losses_m = lse_m - z_m,targets[m]
 * so -losses is the log-probability of each target. Rows whose target lies outside 0..vocab-1 (-100, -1) are left
 * out: their loss and lse are 0, they have no part in d_weight and their row of d_hidden is 0, whatever they hold.
 * A row with a NaN gives a NaN loss, and the gradients that have a part in it are NaN; so does, without a softcap, one with an
 * infinity. With a softcap an infinite sum is a logit of +-softcap, as tanh has it: unless one of its sums is NaN (0 times
 * infinity, infinities of both signs), such a row has a finite loss and d_hidden, and d_weight is not finite in the
 * infinity's column alone.
 *
 * The logits are computed a piece of the vocabulary at a time, summed in fp32, and again for the gradients, which are
 *   dz_mv = grad_m (exp(z_mv - lse_m) - [v = targets[m]]) softcap'(z_mv)
 *   d_hidden = dz W,  d_weight = dz^T H
 * with dz rounded to bf16 (by at most 2^-8 of each term, for a d_weight of fp32 too) for products summed in fp32.
 *
 * An object holds the scratch of calls of up to max_rows (65,536) rows with heads of up to vocab x d_model; d_model is a
 * multiple of 32, at most 2^20, vocab at most 2^24, max_rows x vocab at most 2^38; softcap 0 (none) or in 1e-30..1e30.
 * Without `backward` the scratch is the forward pass's alone: 2 max_rows d_model bytes and 8 max_rows for each 256 of the
 * vocabulary (of up to 128 rows, for each 64). The gradients take, on top of it, up to 256 MB for dz, and d_hidden in
 * fp32, once or for each of the up to 16 parts (up to 128 rows: 32) that its product is cut into where tiles are few.
 * Its calls are ordered across streams as a selector's are, and replays of captured calls are ordered by the caller. */
typedef struct twd_headloss twd_headloss;
TWD_API int twd_headloss_create(uint32_t max_rows, uint32_t vocab, uint32_t d_model, float softcap, int backward,
                                twd_headloss** out);
TWD_API void twd_headloss_destroy(twd_headloss* loss);
TWD_API int twd_headloss_info(const twd_headloss* loss, uint64_t* device_bytes);
/* losses and lse (device, one float a row; lse is what the backward pass needs). hidden_bf16 and weight_bf16 start at
 * multiples of 16 bytes, their rows hidden_stride and weight_stride elements apart (multiples of 8, at most 2^22); targets
 * are device int32. Asynchronous on `stream`. */
TWD_API int twd_headloss_forward(twd_headloss* loss, const uint16_t* hidden_bf16, uint32_t rows, uint64_t hidden_stride,
                                 const uint16_t* weight_bf16, uint64_t weight_stride, const int32_t* targets,
                                 float* losses, float* lse, void* stream);
/* The gradients of sum_m grad[m] losses[m] (grad NULL: all 1), given the same inputs and the lse of the forward pass.
 * d_hidden: bf16 rows; d_weight: rows of d_weight_type (TWD_F32 or TWD_BF16), with accumulate added to what is there.
 * Either may be NULL and is then not computed. Both start at multiples of 16 bytes, strides multiples of 8. Asynchronous
 * on `stream`. */
TWD_API int twd_headloss_backward(twd_headloss* loss, const uint16_t* hidden_bf16, uint32_t rows, uint64_t hidden_stride,
                                  const uint16_t* weight_bf16, uint64_t weight_stride, const int32_t* targets,
                                  const float* lse, const float* grad, uint16_t* d_hidden_bf16, uint64_t d_hidden_stride,
                                  void* d_weight, int d_weight_type, uint64_t d_weight_stride, int accumulate, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TWD_LOSS_H */
