/* Attention over parts of a context that dance_kv.h's cache holds: rows that see
 * all of another sequence (an encoder's states, a prefix that many sequences share),
 * and the join of attentions over several parts. Arrays are device pointers, structs
 * lie on the host; calls behave as dance_kv.h's do: they check their arguments, launch on
 * `stream`, allocate nothing, wait for nothing and can be recorded into a HIP
 * graph; 0 on success, -1 on error with a message on stderr. */
#ifndef DANCE_KV_PARTS_H
#define DANCE_KV_PARTS_H

#include "dance_kv.h"

#ifdef __cplusplus
extern "C" {
#endif

/* dance_kv_attention whose rows see all of their sequence's tokens, whatever their
 * own place: an encoder's states, or a prefix that the rows of many sequences
 * share. lengths[b] has no rows of this call in it; a sequence without tokens gives zeros
 * and -infinity. */
int dance_kv_cross_attention(const DanceKvCache *cache, const DanceKvBatch *batch, const DanceKvRows *queries, float scale,
                             void *out, float *lse, void *work, size_t work_bytes, void *stream);
size_t dance_kv_cross_attention_work(const DanceKvCache *cache, const DanceKvBatch *batch, uint32_t heads);

/* Attention over one part of a context, for dance_kv_join: `tokens` rows x heads x
 * dim with strides in elements, adjacent dimensions, and the logarithms lse
 * [tokens][heads]. rows (may be null) has an entry for each joined row: the part's
 * row, none where it is outside [0, tokens). */
typedef struct DanceKvPart {
    const void *data;
    int64_t token_stride, head_stride;
    const float *lse;
    const int32_t *rows;
    uint64_t tokens;
} DanceKvPart;

/* The attention over all parts of a context from those over each of them: with
 * l_i a row's logarithms, out = sum_i exp(l_i - l) o_i and lse (may be null) l =
 * log sum_i exp(l_i), in float32 and rounded once. A part whose l_i is -infinity counts
 * for nothing, whatever its row holds; where all are, the row is zeros and
 * -infinity; a NaN among them makes the row NaN. 1 to 8 parts, all of `dtype`; a part
 * without `rows` has `tokens` rows; out is tokens x heads x dim of dtype and lse
 * tokens x heads, packed, and neither overlaps a part. */
int dance_kv_join(const DanceKvPart *parts, uint32_t count, uint32_t tokens, uint32_t heads, uint32_t dim, int dtype,
                  void *out, float *lse, void *stream);

#ifdef __cplusplus
}
#endif

#endif
