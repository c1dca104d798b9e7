/*
 * twd_fp8.h -- C-ABI of 8-bit floating point with a scale for each block of 128 on MI355X (gfx950): rows and weights to
 * the format, and an LM head whose weights are held in it. Conventions as in twd_head.h (status codes, twd_last_error,
 * device pointers, streams); types as in twd_mx.h.
 */
#ifndef TWD_FP8_H
#define TWD_FP8_H

#include "twd_mx.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- 8-bit floating point in blocks of 128 ----------------------------------------------------
 * No counterpart in the reference. Elements are e4m3 codes (OCP: sign, four exponent bits with bias 7, three mantissa
 * bits, up to 448; 0x7F and 0xFF are NaN), one to a byte, [rows][cols] and contiguous, at a multiple of 16 bytes. A scale is
 * an fp32 number that a block's elements are multiplied by. Rows (hidden states) have a scale for each 128 columns, scales
 * [rows][cols / 128]; weights one for each 128 x 128, [rows / 128, rounded up][cols / 128]. cols is a multiple of 128.
 *
 * Quantises rows of `type` (device, unit column stride, row_stride elements between rows, at least one row), block_rows 1 or
 * 128 to a scale. With A the block's largest magnitude the scale is A / 448 in fp32, not below 2^-126; an element is x /
 * scale, as an exact quotient, rounded to the nearest value, ties to the even code. A block that holds a NaN or an infinity
 * gets a NaN scale and codes 0. Asynchronous on `stream`. */
TWD_API int twd_fp8_quantize(const void* x, int type, uint64_t rows, uint32_t cols, uint64_t row_stride, uint32_t block_rows,
                             uint8_t* codes, float* scales, void* stream);

/* An LM head whose weights [vocab][d_model] are held in the format, beside twd_head and twd_mxhead. The codes and scales
 * (device; block_rows 128) are copied into the layout the kernels read and may be freed after the call, which is
 * synchronous. d_model is a multiple of 128, at most 2^20; vocab at most 2^30. Scales that are negative, above 2^8 or NaN
 * are rejected with TWD_E_UNSUPPORTED: up to 2^8, times the largest scale of a hidden row, they stay within fp32. softcap 0
 * (none) or in 1e-30..1e30. */
typedef struct twd_fp8head twd_fp8head;
TWD_API int twd_fp8head_create(const uint8_t* codes, const float* scales, uint32_t vocab, uint32_t d_model, float softcap,
                               void* stream, twd_fp8head** out);
TWD_API void twd_fp8head_destroy(twd_fp8head* head);
TWD_API int twd_fp8head_info(const twd_fp8head* head, uint32_t* vocab, uint32_t* d_model, float* softcap,
                             uint64_t* device_bytes);
/* logits[m][v] = softcap(sum_c w[v][c] h[m][c]) of 1 to 65,536 hidden rows held in the format too (twd_fp8_quantize with
 * block_rows 1: codes [rows][d_model], scales [rows][d_model / 128]), each 128 columns' products summed on matrix
 * instructions and the sums, times their scales, added up in fp32; logits_type TWD_F32 or TWD_BF16 with logits_stride >=
 * vocab elements between rows. The products are exact and added in fp32, but for bf16 logits of more than 128 rows: those run
 * on 8-bit instructions, which cut the products of eight neighbouring columns at 2^-13 of the largest of the eight (2e-5 of
 * sum |w h| for normal products). Hidden scales are twd_fp8_quantize's, at most FLT_MAX / 448; the product of two scales is
 * rounded to fp32 (below 2^-126 to a multiple of 2^-149, which takes less than 2^-125 from a block's sum). A row with a NaN scale
 * gives NaN logits. The call keeps no state: calls on one head may overlap, on any streams, and may be
 * captured. Asynchronous on `stream`. */
TWD_API int twd_fp8head_logits(const twd_fp8head* head, const uint8_t* codes, const float* scales, uint32_t rows,
                               void* logits, int logits_type, uint64_t logits_stride, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TWD_FP8_H */
