/*
 * twd_embed.h -- C-ABI of the embedding lookup with scaling and its gradient on MI355X (gfx950). Conventions as in
 * twd_head.h (status codes, twd_last_error, device pointers, streams); types as in twd_mx.h.
 */
#ifndef TWD_EMBED_H
#define TWD_EMBED_H

#include "twd_mx.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- embedding lookup -------------------------------------------------------------------------
 * out[i] = scale * table[ids[i]], the product in fp32, rounded to out_type; a row of zeros where ids[i] lies outside
 * 0..vocab-1 (-1: padding). table: vocab rows (1 to 2^31 - 1) of d_model elements (1 to 2^20) of table_type, table_stride
 * elements apart, at any alignment of the type; rows that are aligned to 16 bytes, as their strides are, move faster. ids:
 * device int32, ids_count of them (none: nothing is done), at most 2^23. Asynchronous on `stream`. */
TWD_API int twd_embed(const void* table, int table_type, uint32_t vocab, uint32_t d_model, uint64_t table_stride,
                      const int32_t* ids, uint32_t ids_count, float scale, void* out, int out_type, uint64_t out_stride,
                      void* stream);

/* The lookup's gradient: d_table[v] = scale * (the sum of d_rows[i] over the i with ids[i] = v), by sorted ids: each sum in
 * fp32 and in an order that depends on the ids alone, so results do not change from run to run. Every row of d_table is
 * written, or with accumulate only those that have an id, on top of what is there. Rows of d_rows whose id lies outside
 * 0..vocab-1 are not read.
 *
 * An object holds the scratch of calls of up to max_ids (262,144) ids and rows of up to max_d_model elements (2^20), 16
 * bytes an id and 1/8 of a byte for each element of that many rows. Its calls are ordered across streams as a
 * selector's are, and replays of captured calls are ordered by the caller. */
typedef struct twd_embedgrad twd_embedgrad;
TWD_API int twd_embedgrad_create(uint32_t max_ids, uint32_t max_d_model, twd_embedgrad** out);
TWD_API void twd_embedgrad_destroy(twd_embedgrad* grad);
TWD_API int twd_embedgrad_info(const twd_embedgrad* grad, uint64_t* device_bytes);
TWD_API int twd_embedgrad_run(twd_embedgrad* grad, const void* d_rows, int rows_type, uint32_t ids_count, uint32_t d_model,
                              uint64_t rows_stride, const int32_t* ids, float scale, void* d_table, int table_type,
                              uint32_t vocab, uint64_t table_stride, int accumulate, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TWD_EMBED_H */
