/* The blocks of dance_kv.h's cache: who owns them, for sequences that fork, grow
 * and shrink; copies of blocks; and the compaction of chosen tokens. Arrays are
 * device pointers, structs lie on the host; calls behave as dance_kv.h's do: they check their
 * arguments, launch on `stream`, allocate nothing, wait for nothing and can be recorded
 * into a HIP graph; 0 on success, -1 on error with a message on stderr. */
#ifndef DANCE_KV_PAGES_H
#define DANCE_KV_PAGES_H

#include "dance_kv.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Owners of a pool's blocks. refs[p] counts the table entries that name block p
 * (and whatever else the caller counts there to keep the block); a block with 0 is
 * free. The three calls below keep it as they change tables of `seqs` rows of
 * `width` entries and the rows' lengths (not negative). Results do not depend on
 * the order of execution. Calls on one pool come one behind the other, on one stream
 * or with the waits that the caller puts between streams. */
typedef struct DanceKvPages {
    int32_t *refs;
    uint32_t blocks, block_tokens;
} DanceKvPages;

/* Row i of the new table and lengths (new_seqs of them) is row parents[i] of the old
 * ones; a parent outside [0, seqs) gives holes (-1) and length 0. The old rows
 * end: refs[p] changes by the difference of p's entries. The new arrays must not
 * overlap the old ones. */
int dance_kv_fork(const DanceKvPages *pages, const int32_t *table, const int32_t *lengths, uint32_t seqs, uint32_t width,
                  const int32_t *parents, uint32_t new_seqs, int32_t *new_table, int32_t *new_lengths, void *stream);

/* Makes room for the tokens lengths[b] .. upto[b] - 1 of each sequence, in blocks
 * that it alone owns. Of the places with such tokens, one that is a hole gets a
 * block; one whose block has refs > 1 gets another one in its stead. The first of
 * them, where tokens stand already (lengths[b] is no multiple of block_tokens), must
 * keep what it holds: where its block has refs > 1, src[b] is that block and dst[b]
 * the new one, for dance_kv_copy (else both are -1); but where all refs of the block
 * are such places of sequences that grow in this call, the last of these keeps it.
 * A hole there stays one.
 * Sequences in ascending order, and their places in ascending order, take the
 * free blocks (refs = 0 before the call) in ascending order. A sequence whose
 * places, with those of all sequences before it, are more than the free blocks gets
 * none, nor does one whose upto passes the table's width; one that needs no block is
 * served all the same (but for one that keeps a block as the last of several: the
 * others must have theirs).
 * Where served, lengths[b] becomes upto[b] and so does now[b]; where not, lengths[b]
 * stays and now[b] is 0, with which an append writes nothing and attention sees
 * nothing. Where upto[b] <= lengths[b] nothing happens and now[b] is lengths[b].
 * `work` holds at least dance_kv_reserve_work() bytes, aligned to 16 (null where
 * that is 0), and may be used again once the call's work on the stream has
 * completed. */
int dance_kv_reserve(const DanceKvPages *pages, int32_t *table, int32_t *lengths, uint32_t seqs, uint32_t width,
                     const int32_t *upto, int32_t *now, int32_t *src, int32_t *dst, void *work, size_t work_bytes,
                     void *stream);
size_t dance_kv_reserve_work(const DanceKvPages *pages, uint32_t seqs, uint32_t width);

/* Gives places back: with keep (may be null) lengths[b] becomes min(lengths[b],
 * max(keep[b], 0)) and all places behind the last token become holes; with start (may be
 * null) so do the places of which every token stands before start[b]. refs of
 * their blocks go down by one for each. */
int dance_kv_release(const DanceKvPages *pages, int32_t *table, int32_t *lengths, uint32_t seqs, uint32_t width,
                     const int32_t *keep, const int32_t *start, void *stream);

/* Copies block src[i] of from[c] to block dst[i] of to[c], for each of `caches`
 * caches (a model's layers) and `pairs` pairs. A pair with either outside its cache
 * is left out. All caches have one kv_heads, dim and block_tokens, all of `from` one
 * number of blocks and all of `to` one; scales need no more than 8 bytes' alignment
 * here (a layer's part of one array of many layers). `to` may be `from`; then no
 * block may be both a source and a destination. No block may be a destination
 * twice. */
int dance_kv_copy(const DanceKvCache *from, const DanceKvCache *to, uint32_t caches, const int32_t *src, const int32_t *dst,
                  uint32_t pairs, void *stream);

/* Writes chosen tokens of sequences densely into other blocks: token i < counts[b]
 * of the new sequence is, for kv head h, the token at position keep[b][h][i] of
 * sequence b in `from` (table and lengths as in a batch; keep is seqs x keep_heads x
 * keep_width, keep_heads is kv_heads, or 1: the same for all heads). It goes to place
 * i of into_table's row, into_width blocks of `to`. Its value x is the product of
 * its code and its scale in float32. A block's scale becomes the least that append
 * would choose for its values, the codes rint(x / scale), the bounds those of its
 * codes; behind the last token it holds zeros. As in append, a product that is not finite
 * (a code times a scale above 2^121 may pass float32's range) counts for no scale: infinities
 * take the code +-127, NaN the code 0. A position that the sequence does not
 * have, or that stands in a hole, gives a token of zeros. What falls beyond
 * into_table's row or into a hole of it is not written, counts beyond keep_width count as that. `to` has from's kv_heads, dim
 * and block_tokens; it may be `from`, but no block that is read may be written, and
 * none may be named twice in into_table. */
int dance_kv_compact(const DanceKvCache *from, const DanceKvCache *to, const int32_t *table, const int32_t *lengths,
                     uint32_t seqs, uint32_t width, const int32_t *keep, uint32_t keep_heads, uint32_t keep_width,
                     const int32_t *counts, const int32_t *into_table, uint32_t into_width, void *stream);

#ifdef __cplusplus
}
#endif

#endif
