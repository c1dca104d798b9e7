/*
 * twd_mx.h -- C-ABI of microscaled 4-bit floating point on MI355X (gfx950): rows to the format and
 * back, and an LM head whose weights are held in it. Conventions as in twd_head.h (status codes,
 * twd_last_error, device pointers, streams).
 */
#ifndef TWD_MX_H
#define TWD_MX_H

#include "twd_head.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- microscaled 4-bit floating point ------------------------------------------------------
 * No counterpart in the reference. The format is OCP Microscaling's MXFP4: a block is 32
 * consecutive columns of a row; its elements are e2m1 codes (sign, two exponent bits, one mantissa
 * bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), two to a byte with the lower column in the lower four bits; its
 * scale is one byte s that stands for 2^(s - 127) (255: NaN). A matrix of rows x cols is `codes`
 * [rows][cols / 2] and `scales` [rows][cols / 32], both contiguous; codes start at a multiple of
 * 16 bytes. */
#define TWD_F32 0
#define TWD_BF16 1
#define TWD_F16 2

/* Quantises rows of `type` (device, unit column stride, row_stride elements between rows; cols a
 * multiple of 32, at least one row). With A the block's largest magnitude the scale is 2^e,
 * e = floor(log2 A) - 2, not below 2^-127 (A = 0: byte 0); an element is x 2^-e rounded to the
 * nearest value, ties to the even code, 6 above that, with x's sign. A block that holds a NaN or an
 * infinity gets scale byte 255 and codes 0. Asynchronous on `stream`. */
TWD_API int twd_mx_quantize(const void* x, int type, uint64_t rows, uint32_t cols, uint64_t row_stride,
                            uint8_t* codes, uint8_t* scales, void* stream);
/* The values that codes and scales stand for, rounded to `type` (exact in fp32 and bf16, but for
 * magnitudes of 2^128 and more, which become infinity). Asynchronous on `stream`. */
TWD_API int twd_mx_dequantize(const uint8_t* codes, const uint8_t* scales, uint64_t rows, uint32_t cols,
                              void* out, int type, uint64_t row_stride, void* stream);

/* An LM head whose weights [vocab][d_model] are held in the format: beside twd_head, for models
 * published in it. The codes and scales (device) are copied into the layout the kernels read and
 * may be freed after the call, which is synchronous. d_model is a multiple of 32, at most 2^20;
 * vocab at most 2^30. Scales above 2^100, and NaN, are rejected with TWD_E_UNSUPPORTED, as
 * twd_head_create rejects such groups. softcap 0 (none) or in 1e-30..1e30. */
typedef struct twd_mxhead twd_mxhead;
TWD_API int twd_mxhead_create(const uint8_t* codes, const uint8_t* scales, uint32_t vocab, uint32_t d_model,
                              float softcap, void* stream, twd_mxhead** out);
TWD_API void twd_mxhead_destroy(twd_mxhead* head);
TWD_API int twd_mxhead_info(const twd_mxhead* head, uint32_t* vocab, uint32_t* d_model, float* softcap,
                            uint64_t* device_bytes);
/* logits[m][v] = softcap(sum_c w[v][c] h[m][c]), 1 to 65,536 rows, summed in fp32; logits_type TWD_F32
 * or TWD_BF16 with logits_stride >= vocab elements between rows. hidden_bf16: rows of d_model bf16
 * values, hidden_stride (a multiple of 8, at most 2^26) elements apart, starting at a multiple of 16
 * bytes; every product is exact. The call keeps no state: calls on one head may overlap, on any streams, and may be
 * captured. Asynchronous on `stream`. */
TWD_API int twd_mxhead_logits(const twd_mxhead* head, const uint16_t* hidden_bf16, uint32_t rows,
                              uint64_t hidden_stride, void* logits, int logits_type, uint64_t logits_stride,
                              void* stream);
/* The same of hidden rows held in the format too (twd_mx_quantize's codes [rows][d_model / 2] and
 * scales [rows][d_model / 32]): the product then runs on 4-bit matrix instructions. A row with a NaN
 * scale gives NaN logits. */
TWD_API int twd_mxhead_logits_mx(const twd_mxhead* head, const uint8_t* codes, const uint8_t* scales,
                                 uint32_t rows, void* logits, int logits_type, uint64_t logits_stride,
                                 void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TWD_MX_H */
