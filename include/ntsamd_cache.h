/*
 * ntsamd_cache.h - C ABI of the gfx950 (MI355X) cache of keys and values: appending to it and attention
 * over it. Exported by the same library as ntsamd_gemm.h, under the same conventions: 0 or an error code, the
 * message in ntsamd_last_error(), work queued on `stream` without synchronising, the caller's current device
 * restored, nothing thrown, any host thread, recordable into a HIP graph.
 *
 * Beyond the reference, whose decoder keeps one dense tensor of keys and one of values per layer and copies both to
 * append one position (source/sample/transformer/submodel/Attention.cpp:143-160): here the positions of a sequence
 * stand on pages of a pool, so that a sequence grows without a copy, sequences of any length share the pool, and
 * sequences with a common beginning share its pages.
 *
 * The cache. `pages` pages of `pageSize` positions, `heads` key heads of `dh` columns:
 *   column c of position r of page g, head h, is k[g * strides[0] + r * strides[1] + h * strides[2] + c],
 *   and v with strides[3..5]; strides in elements, columns contiguous. Both [page][position][head][column] and
 *   [page][head][position][column] are such layouts. dataType is X_FLOAT (dh and the strides multiples of 4) or
 *   X_FLOAT16 (multiples of 8); dh is at most 128; k and v are 16-byte aligned; pageSize is any number from 1.
 *   Pools may exceed 4 GiB.
 *
 * The batch. `sequences` sequences, the last positions of which are new in this step:
 *   lengths[i]     positions of sequence i, the new ones included (device memory);
 *   starts[i]      the row of q, k, v, out where sequence i's new tokens begin; sequence i has
 *                  starts[i + 1] - starts[i] of them (device memory, sequences + 1 values, not decreasing, from 0 or more).
 *                  NULL: every sequence has maxNew new tokens, those of sequence i begin at row i * maxNew;
 *   pageTable      device [sequences][tablePages]: position p of sequence i stands on page
 *                  pageTable[i * tablePages + p / pageSize], row p % pageSize of it;
 *   tokens         rows of q, k, v and out. Rows from starts[sequences] on belong to nobody: they are neither read
 *                  nor written;
 *   maxNew         no sequence has more new tokens than this;
 *   maxLength      no sequence is longer than this (0: tablePages * pageSize, which it may not exceed).
 *   New token t of sequence i is position lengths[i] - (its number of new tokens) + t. A sequence may have no new
 *   tokens, or none at all. The three arrays are read by the kernels, not by the host: a recorded graph may be
 *   replayed with other values in them, within maxNew and maxLength. Values outside those bounds give wrong
 *   results for their sequence, but no access outside the buffers described here: a page number outside [0, pages)
 *   counts as an absent page, see each function.
 */
#ifndef NTSAMD_CACHE_H
#define NTSAMD_CACHE_H

#include "ntsamd_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ntsamd_cache {
    void * k;
    void * v;
    int dataType;
    int pages, pageSize;
    int heads, dh;
    long long strides[6];
} ntsamd_cache;

typedef struct ntsamd_cache_batch {
    const int * lengths;
    const int * starts;
    const int * pageTable;
    int sequences;
    int tablePages;
    int tokens;
    int maxNew;
    int maxLength;
} ntsamd_cache_batch;

/* which columns of a head the rotation turns together: j and j + rotated / 2, or 2 j and 2 j + 1 */
#define NTSAMD_ROTATE_HALVES 0
#define NTSAMD_ROTATE_PAIRS 1

/*
 * The new tokens' keys and values go to their places in the cache; keys, and queries on the same way, are turned
 * by the angle of their position:
 *   k, v      [tokens] rows of cache->heads heads; strides[0], strides[1] step from token to token and from head to
 *             head of k, strides[2], strides[3] of v (elements; any, also of views into a fused projection);
 *   q, qOut   NULL, or [tokens] rows of `heads` heads with strides[4..5] and [6..7]; qOut may be q itself (equal
 *             strides), otherwise the two must not overlap;
 *   rotation  NULL (nothing is turned), or device float [positions][rotated / 2][2]: cosine and sine for every position
 *             and pair of columns; `rotated` is even, at most dh, columns from there on are left as they are.
 *             (x, y) becomes (x cos - y sin, y cos + x sin), in fp32, rounded once.
 * All of them have the cache's data type. A token whose position is negative, beyond its table row or beyond
 * `positions` is left out: nothing of it is written. One whose page is absent is not stored; its q is written. Two
 * tokens of a call that go to the same place leave one of the two there, column by column; no other place changes.
 */
int ntsamd_cache_append(int devID, void * stream, const ntsamd_cache * cache, const ntsamd_cache_batch * batch,
                        const void * k, const void * v, const void * q, void * qOut, int heads,
                        const long long * strides,
                        const float * rotation, int positions, int rotated, int pairing);

/*
 * Attention of the new tokens over their sequences' positions in the cache:
 *   out[t][h] = sum_j softmax_j(scale * <q[t][h], k_j>) v_j,   over the positions j that token t sees,
 * with k and v of key head h / (heads / cache->heads); `heads` is a multiple of cache->heads. causal != 0: a token
 * sees its own position and those before it (append its key first); causal == 0: all positions of its sequence, as
 * the rows of a decoder see cached states of an encoder, of another length than their own. A token that sees nothing gets zeros.
 * Positions on absent pages are left out of the softmax. What stands in the cache beyond a sequence's length is
 * never used, whatever its bits. Inside a sequence, a value that is not finite reaches every token that sees it,
 * and may reach, as NaN, tokens of the same sequence and call that stand before it.
 *   strides[0], strides[1]: token and head of q; strides[2], strides[3]: of out. q and out are 16-byte aligned, their strides
 *   multiples of 4 (float) or 8 (half) elements; out overlaps nothing else. Products accumulate in fp32, and the softmax is in fp32.
 *   Half: probabilities enter the second product as the sum of two halves where no sequence has more than 32 rows (maxNew tokens times
 *   the query heads of a key head); otherwise, and over a shared prefix, they may be rounded to one.
 * Long sequences are cut into pieces whose partial results meet in the stream's workspace (ntsamd_gemm.h) and are
 * added up by a second kernel, always in the same order; without a workspace they run in one piece.
 */
int ntsamd_attention_cached(int devID, void * stream, const ntsamd_cache * cache, const ntsamd_cache_batch * batch,
                            const void * q, void * out, int heads, const long long * strides,
                            float scale, int causal);

/*
 * ntsamd_attention_cached for sequences that begin alike: the first `prefix` positions of every sequence hold the same
 * keys and values, and are found through the first row of the page table for all of them (what the other rows have
 * there is not looked at). They are read once for all sequences: the queries of all sequences are multiplied
 * with them as the rows of one matrix; what follows the prefix is read sequence by sequence, and the two partial
 * results are joined. The result is that of ntsamd_attention_cached but for the order of the additions and the
 * rounding of probabilities. A sequence shorter than the prefix sees the part of it that it has, and nothing of what stands behind its
 * end. The prefix is shared between sequences of up to 32 rows (maxNew tokens times the query heads of a key head)
 * where a workspace is there and the prefix long enough to gain by it; otherwise every sequence reads it for itself, in
 * batches of more new tokens also where sharing would save most of the reading.
 */
int ntsamd_attention_prefix(int devID, void * stream, const ntsamd_cache * cache, const ntsamd_cache_batch * batch,
                            const void * q, void * out, int heads, const long long * strides,
                            float scale, int causal, int prefix);

#ifdef __cplusplus
}
#endif
#endif
