/* A key-value cache in 8-bit codes and the operators that write it and read
 * it: append, attention over all of a sequence, the selection of the blocks
 * worth reading by a bound on their keys' products with the query, and
 * attention over selected blocks (attention over parts of a context: dance_kv_parts.h; the
 * blocks' owners, copies and compaction: dance_kv_pages.h). No counterpart in the reference: beside the
 * library's searches over vectors in 8-bit codes, the same idea for the keys and
 * values of a language model's cache, with layouts and kernels of their own.
 *
 * All pointers are device pointers. A call checks its arguments on the host,
 * launches its kernels on `stream` and returns; it allocates nothing, waits
 * for nothing and keeps nothing, so it can be recorded into a HIP graph.
 * All return 0 on success and -1 on error (message on stderr).
 *
 * The cache holds `blocks` blocks of `block_tokens` tokens. For block p, kv
 * head h, token slot t and dimension d:
 *   k     [blocks][kv_heads][block_tokens][dim]   int8 codes of the keys
 *   v     [blocks][kv_heads][dim][block_tokens]   int8 codes of the values
 *   scale [blocks][kv_heads][2]                   a key is k * scale[0], a value v * scale[1]
 *   bound [blocks][kv_heads][2][dim]              largest and least key code of the block's tokens
 * all aligned to 16 bytes. dim is 64, 96, 128, 192 or 256; block_tokens 16,
 * 32, 64 or 128.
 *
 * A batch holds `seqs` sequences. table[b * table_width + j] is the block with
 * tokens [j * block_tokens, (j + 1) * block_tokens) of sequence b; an entry
 * outside [0, blocks) is a hole, whose tokens are neither read nor written.
 * lengths[b] counts the sequence's tokens, those that this call brings or asks
 * for included; what lies beyond the table's width is not there. The call's
 * token rows of sequence b are offsets[b] .. offsets[b + 1] - 1 (offsets[0] =
 * 0, not decreasing, none beyond `tokens`), or row b alone where offsets is
 * null (then tokens = seqs); row i of n stands at position lengths[b] - n + i
 * and sees the positions up to its own. A row at a negative position sees
 * nothing and is not written into the cache; the outputs of rows of no sequence
 * (beyond the last offset) are undefined. max_tokens is at least the most rows of a
 * sequence, max_length at least the longest length (0: the table's width).
 * A call is one launch of fewer than 2^32 threads (and a join of splits, where there are any), and refuses a batch that
 * needs more: attention has room for 2^23 single rows x kv heads (of up to 16 heads each), and for prompts of
 * some 2^30 rows x heads. */
#ifndef DANCE_KV_H
#define DANCE_KV_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of queries, new keys and values, and outputs (the first is
 * DANCE_DTYPE_F16 of dance_hip.h). */
enum { DANCE_KV_F16 = 2, DANCE_KV_BF16 = 3 };

typedef struct DanceKvCache {
    int8_t *k, *v;
    float *scale;
    int8_t *bound;
    uint32_t blocks, kv_heads, dim, block_tokens;
} DanceKvCache;

typedef struct DanceKvBatch {
    const int32_t *table;
    const int32_t *lengths;
    const int32_t *offsets; /* seqs + 1 entries, or null */
    uint32_t seqs, tokens, table_width, max_tokens;
    uint64_t max_length;
} DanceKvBatch;

/* Rows of tokens x heads x dim; strides in elements, the dimensions of a row
 * adjacent. heads is a multiple of kv_heads: head i belongs to kv head i /
 * (heads / kv_heads). */
typedef struct DanceKvRows {
    const void *data;
    int64_t token_stride, head_stride;
    uint32_t heads;
    int dtype;
} DanceKvRows;

/* Writes the rows' keys and values (heads = kv_heads) into the cache. In a
 * block with new tokens, per head and for keys and values apart: with a the
 * largest magnitude of the new tokens and e the least integer >= -100 with
 * a <= 127 * 2^e, the scale becomes s' = max(s, 2^e) (2^e where the block held
 * none of the sequence's tokens before), its old codes c become rint(c * s / s')
 * and the new ones rint(x / s'), halves to even. Not finite: infinities take
 * the code +-127, NaN the code 0, and neither counts for a. The bounds follow.
 * A block that the call opens holds zeros behind its last token, others hold
 * anything there (tokens that a shorter length gave up are not kept). Two
 * sequences, or two places of one, must not share a block that is written. */
int dance_kv_append(const DanceKvCache *cache, const DanceKvBatch *batch, const DanceKvRows *keys,
                    const DanceKvRows *values, void *stream);

/* out[t][head] = sum over the visible tokens of softmax(scale * q . k) v, and
 * lse[t][head] (may be null) the natural logarithm of the sum of
 * exp(scale * q . k). out is tokens x heads x dim of the queries' type, packed.
 * A row that sees nothing gives zeros and -infinity. `work` holds at least
 * dance_kv_attention_work() bytes, aligned to 16 (null where that is 0), and
 * may be used again once the call's work on the stream has completed. */
int dance_kv_attention(const DanceKvCache *cache, const DanceKvBatch *batch, const DanceKvRows *queries, float scale,
                       void *out, float *lse, void *work, size_t work_bytes, void *stream);
size_t dance_kv_attention_work(const DanceKvCache *cache, const DanceKvBatch *batch, uint32_t heads);

/* For each token row and kv head the `count` blocks with the best scores,
 * as logical blocks (indices into the sequence's table row), ascending, -1
 * behind them: chosen is tokens x kv_heads x count. The score of a block is
 * the largest over the group's heads of sum_d max(c_d * hi_d, c_d * lo_d) *
 * scale * 2^e, where c = rint(q / 2^e) are the head's codes (rounded as in
 * append) and hi, lo the block's bounds: no token of the block has a larger
 * product with the rounded query. The sum is exact; equal scores go to the
 * lower index. The first `sink` and the last `recent` blocks that the row
 * sees are chosen before all others; holes and blocks the row does not see
 * never are. */
int dance_kv_select(const DanceKvCache *cache, const DanceKvBatch *batch, const DanceKvRows *queries, uint32_t count,
                    uint32_t sink, uint32_t recent, int32_t *chosen, void *work, size_t work_bytes, void *stream);
size_t dance_kv_select_work(const DanceKvCache *cache, const DanceKvBatch *batch, uint32_t heads, uint32_t count);

/* dance_kv_attention over the blocks of a list for each token row and kv head:
 * lists is tokens x kv_heads x count logical blocks, in any order, each at most
 * once; entries that are negative, holes or beyond what the row sees are left
 * out. */
int dance_kv_sparse_attention(const DanceKvCache *cache, const DanceKvBatch *batch, const DanceKvRows *queries,
                              const int32_t *lists, uint32_t count, float scale, void *out, float *lse, void *work,
                              size_t work_bytes, void *stream);
size_t dance_kv_sparse_attention_work(const DanceKvCache *cache, const DanceKvBatch *batch, uint32_t heads,
                                      uint32_t count);

#ifdef __cplusplus
}
#endif

#endif
