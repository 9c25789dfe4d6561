/*
 * The cache of keys and values on pages: problem descriptor of its kernels (cache_append.hip,
 * attention_cached.hip), shared with the C ABI (ntsamd_capi.hip).
 */
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ntsamd {

/* n / d for 0 <= n < 2^31 by a multiplication: with 2^(l-1) < d <= 2^l and mul = ceil(2^(31+l) / d) < 2^32, mul * d exceeds
   2^(31+l) by less than 2^l, so n * mul / 2^(31+l) exceeds n / d by less than 1 / d. */
struct FastDiv {
    unsigned mul;
    int shift;
    unsigned d;
};

inline FastDiv fast_div(int d)
{
    FastDiv f;
    int l = 0;
    while ((1LL << l) < d)
        l++;
    f.mul = (unsigned)(((1ULL << (31 + l)) + (unsigned)d - 1) / (unsigned)d);
    f.shift = 31 + l;
    f.d = (unsigned)d;
    return f;
}

__device__ __forceinline__ int divided(int n, const FastDiv & f)
{
    return (int)(((unsigned long long)(unsigned)n * f.mul) >> f.shift);
}

/* Workgroups of a launch: its threads are counted in 32 bits, and of one with more, workgroups are left out without an error. */
constexpr long long most_workgroups(int threads) { return 0xffffffffLL / threads; }

struct CacheParams {
    void * k;                           /* the pools */
    void * v;
    long long kP, kR, kH, vP, vR, vH;   /* element strides: page, position in the page, head */
    int pages, kvHeads, dh;
    FastDiv pageSize;
    const int * lengths;                /* the batch */
    const int * starts;                 /* NULL: maxNew tokens each */
    const int * table;
    int sequences, tablePages, tokens, maxNew, maxLength;
};

/* what the batch says about one sequence, held to the bounds that the host was given: whatever the arrays hold, no
   row outside [0, tokens) and no position outside [0, maxLength) is touched */
struct CacheSequence {
    int start, fresh, length;           /* row of the first new token, new tokens, positions */
};

__device__ __forceinline__ CacheSequence cache_sequence(const CacheParams & c, int i)
{
    CacheSequence s;
    if (c.starts) {
        const int a = c.starts[i], b = c.starts[i + 1];
        s.start = min(max(a, 0), c.tokens);
        s.fresh = min(max(min(b, c.tokens) - s.start, 0), c.maxNew);
    }
    else {
        s.start = i * c.maxNew;
        s.fresh = c.maxNew;
    }
    s.length = min(max(c.lengths[i], 0), c.maxLength);
    return s;
}

struct AppendParams {
    CacheParams c;
    const void * nk;                    /* the new rows */
    const void * nv;
    const void * q;                     /* NULL: no queries */
    void * qOut;
    int heads;
    long long kT, kH, vT, vH, qT, qH, oT, oH;
    const float * rotation;             /* NULL: nothing is turned */
    int positions, rotated, pairing;
    bool whole;                         /* from here on filled in by plan_cache_append: items of 16 bytes, not of single columns */
    int items, perWave, waves;          /* pieces of work per token, of them per wave, waves per token */
    int token0;                         /* the first token of this launch */
};

struct CachedParams {
    CacheParams c;
    const void * q;
    void * out;
    long long qT, qH, oT, oH;
    int per;                            /* query heads per key head */
    FastDiv perDiv;
    float scale;
    int causal;
    int seq0, seqs;                     /* the sequences of this launch: seq0 .. seq0 + seqs - 1 */
    int first;                          /* positions before this one are another launch's (the shared prefix), see first_of */
    int common;                         /* positions before this one are found through the first row of the table */
    int prefix;                         /* > 0: this launch is the shared prefix of that many positions */
    int mode;                           /* CachedMode */
    int groups;                         /* CACHED_PIECES: pieces aimed at; CACHED_TILES: pieces of a tile's keys */
    int tiles;                          /* CACHED_TILES: tiles launched (at least those that the batch can have) */
    int sorted;                         /* CACHED_WHOLE, and CACHED_TILES without partial results, up to 64 sequences: the longest first */
    int runs;                           /* CACHED_TILES: so many keys (16, or 8, 4, 2) from a multiple of it on are on one page, within 2 GiB */
    int rows;                           /* rows of a slot */
    /* partial results: acc[slot][row][dh] and stat[slot][row][2] (maximum and sum, base 2); NULL: results go to out */
    float * acc;
    float * stat;
    int * slots;                        /* CACHED_PIECES: first slot and number of pieces of every pair, for the join */
    FastDiv part;                       /* with a shared prefix: keys of its pieces but the last */
};

/* CACHED_WHOLE: a workgroup takes all keys of one (sequence, key head).
   CACHED_PIECES: the keys of every pair cut into pieces of about the same length, one workgroup each.
   CACHED_TILES: rows cut into tiles (several to a sequence), the keys of a tile into `groups` pieces. */
enum CachedMode { CACHED_WHOLE = 0, CACHED_PIECES = 1, CACHED_TILES = 2 };

/* false: a token has more items than the kernel counts */
bool plan_cache_append(AppendParams & p, bool half);
int launch_cache_append(AppendParams p, bool half, hipStream_t stream);

}  // namespace ntsamd
