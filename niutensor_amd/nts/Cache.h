/*
 * Keys and values of a decoder on pages, and attention over them, on a gfx950 GPU: what the decoder of the
 * reference's transformer sample does with its Cache (source/sample/transformer/submodel/Attention.cpp:143-160, one dense tensor of
 * keys and one of values per layer, both copied to append a position), for sequences that grow in place, of any lengths together.
 */
#ifndef NTSAMD_CACHE_LAYER_H
#define NTSAMD_CACHE_LAYER_H

#include "XTensor.h"

namespace nts {

/* Which sequences stand where, and which of their positions are new. All X_INT and on the GPU of the pools; read by the
   kernels, so they may change between calls without a copy to the host.
   lengths    (n): positions of every sequence, the new ones included
   starts     (n + 1): the rows where the sequences' new tokens begin, ascending; NULL: every sequence has maxNew of them
   pageTable  (n, width): position p of sequence i stands in row p % pageSize of page pageTable[i][p / pageSize]
   maxNew     no sequence has more new tokens; maxLength: none is longer (0: width * pageSize) */
struct AmdCacheBatch {
    const XTensor * lengths;
    const XTensor * starts;
    const XTensor * pageTable;
    int maxNew;
    int maxLength;
};

/* The new tokens' keys and values go to their places in the pools.
   keys, values: (pages, pageSize, kvHead, dh), X_FLOAT or X_FLOAT16; k, v: (tokens, kvHead * dh) of the same type.
   rotation: NULL, or X_FLOAT (positions, rotated / 2, 2), cosine and sine by which columns j and j + rotated / 2 of every key head
   (isPairs: 2 j and 2 j + 1) are turned at a position. q: NULL, or (tokens, hidden), turned likewise into qOut, which may be q. */
void _AmdCacheAppend(XTensor * keys, XTensor * values, const AmdCacheBatch & batch, const XTensor * k, const XTensor * v,
                     const XTensor * rotation = NULL, bool isPairs = false, const XTensor * q = NULL, XTensor * qOut = NULL);

/* out = attention of the new tokens to what the pools hold of their sequences; q, out: (tokens, hidden), hidden = nhead * dh with
   nhead a multiple of kvHead. isCausal: to the positions up to their own, otherwise to all. Rows of no sequence stay as they are. */
void _AmdAttentionCached(const XTensor * keys, const XTensor * values, const AmdCacheBatch & batch, const XTensor * q, XTensor * out,
                         DTYPE scale, bool isCausal = true);

/* the same for sequences whose first `prefix` positions are one and the same, on the pages of the first row of the table */
void _AmdAttentionPrefix(const XTensor * keys, const XTensor * values, const AmdCacheBatch & batch, const XTensor * q, XTensor * out,
                         DTYPE scale, int prefix, bool isCausal = true);

/* into a new tensor shaped like q, zeros in rows of no sequence */
XTensor AmdAttentionCached(const XTensor & keys, const XTensor & values, const AmdCacheBatch & batch, const XTensor & q, DTYPE scale,
                           bool isCausal = true);

}  // namespace nts
#endif
