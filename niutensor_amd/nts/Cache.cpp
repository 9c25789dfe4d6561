/*
 * The cache on pages over the C ABI of ntsamd_cache.h: shapes and types are checked here, the rest there.
 */
#include "Cache.h"
#include "../../include/ntsamd_cache.h"

namespace nts {

/* an optional tensor that is given has memory: below this layer an address of NULL stands for one that is not */
static bool HasMemory(const XTensor * t)
{
    return t == NULL || t->data != NULL || t->unitNum == 0;
}

/* what the entry points get of the pools and the batch; `tokens` rows of x, of `width` columns */
static void Describe(const XTensor * keys, const XTensor * values, const AmdCacheBatch & batch, const XTensor * x,
                     ntsamd_cache & cache, ntsamd_cache_batch & b)
{
    CheckNTErrors((keys && values && x && batch.lengths && batch.pageTable), "Empty input tensors!");
    CheckNTErrors((keys->dataType == X_FLOAT || keys->dataType == X_FLOAT16), "TODO!");
    CheckNTErrors((values->dataType == keys->dataType && x->dataType == keys->dataType),
                  "Input tensors should have the same data type!");
    CheckNTErrors((keys->order == 4 && _IsSameShaped(keys, values)), "Unmatched tensors in a cache!");
    CheckNTErrors((x->order == 2), "Unmatched tensors in a cache!");
    const XTensor * ints[3] = {batch.lengths, batch.pageTable, batch.starts};
    const int n = batch.lengths->unitNum;
    CheckNTErrors((keys->devID >= 0), "This code must be run on GPUs!");
    CheckNTErrors((values->devID == keys->devID && x->devID == keys->devID), "The tensors must be on the same GPU!");
    for (int i = 0; i < 3; i++) {
        if (ints[i] == NULL)
            continue;
        CheckNTErrors((ints[i]->dataType == X_INT), "Lengths, starts and page numbers must be integers!");
        CheckNTErrors((ints[i]->devID == keys->devID), "The tensors must be on the same GPU!");
    }
    CheckNTErrors((batch.pageTable->order == 2 && batch.pageTable->dimSize[0] == n), "Unmatched tensors in a cache!");
    CheckNTErrors((batch.starts == NULL || batch.starts->unitNum == n + 1), "Unmatched tensors in a cache!");

    cache.k = keys->data;
    cache.v = values->data;
    cache.dataType = keys->dataType;
    cache.pages = keys->dimSize[0];
    cache.pageSize = keys->dimSize[1];
    cache.heads = keys->dimSize[2];
    cache.dh = keys->dimSize[3];
    for (int i = 0; i < 6; i += 3) {
        cache.strides[i + 2] = cache.dh;
        cache.strides[i + 1] = (long long)cache.heads * cache.dh;
        cache.strides[i] = cache.pageSize * cache.strides[i + 1];
    }
    b.lengths = (const int *)batch.lengths->data;
    b.starts = batch.starts != NULL ? (const int *)batch.starts->data : NULL;
    b.pageTable = (const int *)batch.pageTable->data;
    b.sequences = n;
    b.tablePages = batch.pageTable->dimSize[1];
    b.tokens = x->dimSize[0];
    b.maxNew = batch.maxNew;
    b.maxLength = batch.maxLength;
}

/* query heads of q, which has the type, the place and the rows of a call */
static int QueryHeads(const XTensor * q, const XTensor * out, const ntsamd_cache & cache, const ntsamd_cache_batch & b, int devID)
{
    CheckNTErrors((q->order == 2 && _IsSameShaped(q, out) && q->dimSize[0] == b.tokens), "Unmatched tensors in a cache!");
    CheckNTErrors((q->dataType == cache.dataType && out->dataType == cache.dataType),
                  "Input tensors should have the same data type!");
    CheckNTErrors((q->devID == devID && out->devID == devID), "The tensors must be on the same GPU!");
    CheckNTErrors((cache.dh > 0 && q->dimSize[1] % cache.dh == 0),
                  "The hidden size must be a multiple of the size of a head!");
    return q->dimSize[1] / cache.dh;
}

void _AmdCacheAppend(XTensor * keys, XTensor * values, const AmdCacheBatch & batch, const XTensor * k, const XTensor * v,
                     const XTensor * rotation, bool isPairs, const XTensor * q, XTensor * qOut)
{
    ntsamd_cache cache;
    ntsamd_cache_batch b;
    Describe(keys, values, batch, k, cache, b);
    CheckNTErrors((v != NULL && (q == NULL) == (qOut == NULL)), "Empty input tensors!");
    CheckNTErrors((_IsSameShaped(k, v) && k->dimSize[1] == cache.heads * cache.dh), "Unmatched tensors in a cache!");
    CheckNTErrors((v->dataType == cache.dataType), "Input tensors should have the same data type!");
    CheckNTErrors((v->devID == keys->devID), "The tensors must be on the same GPU!");
    const int nhead = q != NULL ? QueryHeads(q, qOut, cache, b, keys->devID) : 0;
    int positions = 0, rotated = 0;
    if (rotation != NULL) {
        CheckNTErrors((rotation->dataType == X_FLOAT && rotation->devID == keys->devID && rotation->order == 3 &&
                       rotation->dimSize[2] == 2), "Unmatched tensors in a cache!");
        positions = rotation->dimSize[0];
        rotated = 2 * rotation->dimSize[1];
    }
    CheckNTErrors((HasMemory(batch.starts) && HasMemory(rotation) && HasMemory(q) && HasMemory(qOut)), "Empty input tensors!");
    /* nothing of a table without elements is read */
    const float * turns = rotation == NULL ? NULL : (const float *)(rotation->data != NULL ? rotation->data : keys->data);
    const long long row = (long long)cache.heads * cache.dh, wide = (long long)nhead * cache.dh;
    const long long strides[8] = {row, cache.dh, row, cache.dh, wide, cache.dh, wide, cache.dh};
    int rc = ntsamd_cache_append(keys->devID, NULL, &cache, &b, k->data, v->data, q != NULL ? q->data : NULL,
                                 qOut != NULL ? qOut->data : NULL, nhead, strides,
                                 turns, positions, rotated,
                                 isPairs ? NTSAMD_ROTATE_PAIRS : NTSAMD_ROTATE_HALVES);
    if (rc != NTSAMD_OK) {
        ShowNTErrors(ntsamd_last_error());
    }
}

static void Attend(const XTensor * keys, const XTensor * values, const AmdCacheBatch & batch, const XTensor * q, XTensor * out,
                   DTYPE scale, int prefix, bool isCausal)
{
    ntsamd_cache cache;
    ntsamd_cache_batch b;
    Describe(keys, values, batch, q, cache, b);
    CheckNTErrors((out != NULL), "Empty input tensors!");
    const int nhead = QueryHeads(q, out, cache, b, keys->devID);
    CheckNTErrors((HasMemory(batch.starts)), "Empty input tensors!");
    const long long wide = (long long)nhead * cache.dh;
    const long long strides[4] = {wide, cache.dh, wide, cache.dh};
    int rc = prefix < 0 ? ntsamd_attention_cached(keys->devID, NULL, &cache, &b, q->data, out->data, nhead, strides, scale, isCausal)
                        : ntsamd_attention_prefix(keys->devID, NULL, &cache, &b, q->data, out->data, nhead, strides, scale, isCausal, prefix);
    if (rc != NTSAMD_OK) {
        ShowNTErrors(ntsamd_last_error());
    }
}

void _AmdAttentionCached(const XTensor * keys, const XTensor * values, const AmdCacheBatch & batch, const XTensor * q, XTensor * out,
                         DTYPE scale, bool isCausal)
{
    Attend(keys, values, batch, q, out, scale, -1, isCausal);
}

void _AmdAttentionPrefix(const XTensor * keys, const XTensor * values, const AmdCacheBatch & batch, const XTensor * q, XTensor * out,
                         DTYPE scale, int prefix, bool isCausal)
{
    CheckNTErrors((prefix >= 0), "A negative prefix!");
    Attend(keys, values, batch, q, out, scale, prefix, isCausal);
}

XTensor AmdAttentionCached(const XTensor & keys, const XTensor & values, const AmdCacheBatch & batch, const XTensor & q, DTYPE scale,
                           bool isCausal)
{
    XTensor out(q.order, q.dimSize, q.dataType, 1.0F, q.devID, q.mem);
    out.SetTMPFlag();
    /* without starts the first maxNew rows of every sequence are written: no fill where these are all */
    if (batch.starts != NULL || batch.lengths == NULL || (long long)batch.lengths->unitNum * batch.maxNew < q.dimSize[0])
        out.SetZeroAll();
    _AmdAttentionCached(&keys, &values, batch, &q, &out, scale, isCausal);
    return out;
}

}  // namespace nts
