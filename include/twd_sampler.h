/*
 * twd_sampler.h -- C-ABI of sampling with temperature, top-k, top-p and min-p from given random
 * numbers on MI355X (gfx950). Conventions as in twd_head.h; the logits' types are twd_mx.h's.
 */
#ifndef TWD_SAMPLER_H
#define TWD_SAMPLER_H

#include "twd_mx.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- sampling from given random numbers ------------------------------------------------------
 * No counterpart in the reference, whose sample_token (twd_select) cuts by top_p before top_k and the
 * temperature. Here, per row: weights w_i = exp((l_i - max) / T); in the order of falling logit, equal
 * logits by rising index, three limits each keep a prefix -- the first top_k ids, the shortest prefix
 * whose weights reach top_p of the top-k's sum, the weights of at least min_p of the largest -- and the
 * shortest of them is kept, at least one id. tokens[m] is the first kept id, by index, at which the
 * running sum of kept weights exceeds uniform[m] of their sum; logprobs[m] (may be NULL) is ln of its
 * share of that sum, kept[m] (may be NULL) the number of kept ids. Entries of -inf are masked: they are
 * never kept.
 *
 * All parameters are device arrays of one value per row, so a captured call reads them anew at every
 * replay; any but `uniform` may be NULL: T = 1 and no limit. T <= 0 takes the largest logit, the lowest
 * index on ties (logprob 0, one id kept); T = +inf weighs all ids alike. top_k <= 0, top_p >= 1 and
 * min_p <= 0 are no limit. uniform lies in [0, 1); values outside act as its nearest end. A row that
 * holds a NaN or +inf logit or no entry above -inf, and one whose T, top_p, min_p or uniform is NaN,
 * gives TWD_TOKEN_DEGENERATE, a NaN logprob and 0 kept.
 *
 * Sums are integers (weights of 37 bits; a weight under 2^-66 of the largest, of a logit 45.7 T and more
 * below it, may count as nothing in them, but for a draw of 0, which takes the first kept id down to
 * 745 T below), so results do not depend on the launch, the batch or the run. logits are rows of `type`
 * with row_stride elements between them, at any alignment of that type, and stay as they are. A sampler
 * holds the scratch of up to max_rows (4,096) rows of up to max_vocab (524,288) entries, about 330 KB a
 * row of 262,144; its calls are ordered across streams as a selector's are, and replays of captured
 * calls are ordered by the caller. Asynchronous on `stream`.
 *
 * A row of 262,144 takes some 30 us, 64 of them under 60. A row of which more than 32,768 entries lie in the
 * eighth of an octave of weight where a limit cuts takes 1 to 4 ms, and its batch with it: equal logits under any
 * limit, or T so high that the weights are nearly equal (T = +inf with a limit among them). */
typedef struct twd_sampler twd_sampler;
TWD_API int twd_sampler_create(uint32_t max_vocab, uint32_t max_rows, twd_sampler** out);
TWD_API void twd_sampler_destroy(twd_sampler* sampler);
TWD_API int twd_sampler_sample(twd_sampler* sampler, const void* logits, int type, uint32_t vocab, uint32_t rows,
                               uint64_t row_stride, const float* temperature, const int32_t* top_k,
                               const float* top_p, const float* min_p, const float* uniform, uint32_t* tokens,
                               float* logprobs, int32_t* kept, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TWD_SAMPLER_H */
