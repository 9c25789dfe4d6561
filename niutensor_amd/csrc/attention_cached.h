/*
 * What the kernels of the cached attention share (attention_cached.hip, attention_cached_join.hip): how the keys of a
 * batch are dealt out to workgroups, found again by the kernel that joins partial results.
 */
#pragma once
#include "cache.h"

namespace ntsamd {

struct CachedScan {
    long long sums[8];
    long long before;
    int found;
    int order[64];
};

/* Keys that the kernels take at a time: a wave of the few-rows kernel, a workgroup of tiles of 64 rows and more */
constexpr int CACHED_TILE_KEYS = 64;
constexpr int cached_block_keys(bool half, int columns, int rows)
{
    return rows < 64 ? (half ? 32 : 16) : (!half && columns > 64 ? 32 : CACHED_TILE_KEYS);
}

/* The first position that a sequence's own launch takes. A sequence that ends inside the shared prefix has no use for the partial
   result of the piece in which it ends: what stands behind its end is multiplied there too, by probabilities of zero, which is NaN
   where it is not finite. It takes the pieces that it has whole, and reads the rest, less than a piece, for itself. */
__device__ __forceinline__ int first_of(const CachedParams & p, const CacheSequence & s)
{
    return s.length >= p.first ? p.first : divided(s.length, p.part) * (int)p.part.d;
}

/* units of keys of one (sequence, key head) pair: at least one where there are tokens to answer */
template <int UK>
__device__ __forceinline__ int units_of(const CachedParams & p, const CacheSequence & s)
{
    return s.fresh > 0 ? max((s.length - first_of(p, s) + UK - 1) / UK, 1) : 0;
}

/* Sums over the sequences of a launch, weight(i) each: every thread of the 64 NW takes a run of sequences. */
struct SequenceScan {
    long long before, sum, total;       /* of the sequences before this thread's, of this thread's, of all */
    int from, to;                       /* this thread's sequences */
};

template <int NW = 4, typename W>
__device__ __forceinline__ SequenceScan scan_sequences(int count, CachedScan & sh, W weight)
{
    SequenceScan r;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int run = (count + 64 * NW - 1) / (64 * NW);
    r.from = min(tid * run, count);
    r.to = min(r.from + run, count);
    r.sum = 0;
    for (int i = r.from; i < r.to; i++)
        r.sum += weight(i);
    long long upTo = r.sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const long long x = __shfl_up(upTo, d);
        if (lane >= d)
            upTo += x;
    }
    if (lane == 63)
        sh.sums[wave] = upTo;
    __syncthreads();
    r.before = upTo - r.sum;
    r.total = 0;
#pragma unroll
    for (int w = 0; w < NW; w++) {
        if (w < wave)
            r.before += sh.sums[w];
        r.total += sh.sums[w];
    }
    return r;
}

/* the sequence of a launch in which place `at` of the sum (of its low half) falls, and the sum before it; -1 past the end */
template <typename W>
__device__ __forceinline__ int find_sequence(const SequenceScan & r, int at, long long & before, CachedScan & sh, W weight)
{
    if (at >= (int)r.total)
        return -1;
    if (at >= (int)r.before && at < (int)r.before + (int)r.sum) {
        long long b = r.before;
        int i = r.from;
        for (long long w = weight(i); i + 1 < r.to && at >= (int)b + (int)w; w = weight(i)) {
            b += w;
            i++;
        }
        sh.before = b;
        sh.found = i;
    }
    __syncthreads();
    const int i = __builtin_amdgcn_readfirstlane(sh.found);
    before = sh.before;
    return i;
}

/* CACHED_PIECES: every (sequence, key head) pair is cut into pieces of at most `most` units, `most` such that all units
   together make about p.groups pieces: at most p.groups + the number of pairs, and at most 2 p.groups of pairs that have more
   than one. Both sums over the sequences travel in one: pieces in the low half, pieces of cut pairs in the high one. */
struct PiecePlan {
    int most;
    SequenceScan scan;
};

template <int UK>
__device__ __forceinline__ long long pieces_of(const CachedParams & p, int i, int most)
{
    const unsigned n = ((unsigned)units_of<UK>(p, cache_sequence(p.c, p.seq0 + i)) + most - 1) / (unsigned)most;
    const long long all = (long long)n * p.c.kvHeads;
    return all + (n > 1 ? all << 32 : 0);
}

template <int UK>
__device__ __forceinline__ PiecePlan piece_plan(const CachedParams & p, CachedScan & sh)
{
    PiecePlan f;
    const SequenceScan units = scan_sequences(p.seqs, sh, [&](int i) { return (long long)units_of<UK>(p, cache_sequence(p.c, p.seq0 + i)); });
    /* whole rounds of the four waves, which take a unit each at a time; one where no sequence has new tokens, nor units */
    const long long total = units.total * p.c.kvHeads;
    const long long each = total >> 31 ? (total + p.groups - 1) / p.groups : ((unsigned)total + p.groups - 1) / (unsigned)p.groups;
    f.most = (int)min(max((each + 3) & ~3ll, 4ll), 0x7ffffffcll);
    __syncthreads();
    f.scan = scan_sequences(p.seqs, sh, [&](int i) { return pieces_of<UK>(p, i, f.most); });
    return f;
}

/* a range of the keys of one tile of rows */
struct Segment {
    CacheSequence s;
    int seq, head;                      /* table row, key head */
    int row0, rows;                     /* first row of the tile, rows the sequence has (0: nothing to do) */
    int keys;                           /* positions that any row of the tile sees */
    int first;                          /* position at which the units begin */
    int u0, u1;                         /* units */
    int slot;                           /* where the partial result goes, -1: the result goes to out */
};

/* The same for all lanes: in scalar registers. (Loaded by lanes, kept by lanes: the table's address alone would be
   spilled, and a reload inside the loop waits for every row in flight.) */
__device__ __forceinline__ Segment uniform(Segment sg)
{
    sg.s.start = __builtin_amdgcn_readfirstlane(sg.s.start);
    sg.s.fresh = __builtin_amdgcn_readfirstlane(sg.s.fresh);
    sg.s.length = __builtin_amdgcn_readfirstlane(sg.s.length);
    sg.seq = __builtin_amdgcn_readfirstlane(sg.seq);
    sg.head = __builtin_amdgcn_readfirstlane(sg.head);
    sg.row0 = __builtin_amdgcn_readfirstlane(sg.row0);
    sg.rows = __builtin_amdgcn_readfirstlane(sg.rows);
    sg.keys = __builtin_amdgcn_readfirstlane(sg.keys);
    sg.first = __builtin_amdgcn_readfirstlane(sg.first);
    sg.u0 = __builtin_amdgcn_readfirstlane(sg.u0);
    sg.u1 = __builtin_amdgcn_readfirstlane(sg.u1);
    sg.slot = __builtin_amdgcn_readfirstlane(sg.slot);
    return sg;
}

/* tokens of the sequences of a launch, which begin at row `start` */
__device__ __forceinline__ int prefix_tokens(const CachedParams & p, int start)
{
    const int most = p.seqs * p.c.maxNew;
    if (!p.c.starts)
        return most;
    return min(max(min(p.c.starts[p.seq0 + p.seqs], p.c.tokens) - start, 0), most);
}

/* sh.order: the sequences of a launch (64 at most), the one with the fewest positions first */
__device__ __forceinline__ void sort_sequences(const CachedParams & p, CachedScan & sh)
{
    const int lane = threadIdx.x & 63;
    const int length = lane < p.seqs ? cache_sequence(p.c, p.seq0 + lane).length : 0;
    const int key = min(length, 0x1ffffff) << 6 | lane;             /* no two alike */
    int rank = 0;
    for (int i = 0; i < p.seqs; i++)
        rank += __builtin_amdgcn_readlane(key, i) < key ? 1 : 0;
    if (threadIdx.x < p.seqs)
        sh.order[rank] = lane;
    __syncthreads();
}

/* CACHED_TILES: the segment of workgroup `id` of NW waves, tiles of TR rows, units of UK keys; without rows where it has none */
template <int TR, int UK, int NW = 4>
__device__ __forceinline__ Segment tile_segment(const CachedParams & p, CachedScan & sh, int id)
{
    /* the last tiles of a sequence see the most keys: first. Where there are more workgroups than run at once, those of the longest
       sequence too, so that the last ones to start are short (4 pieces of text of 257 to 1024 tokens in sequences of 1500 to 4096,
       32 heads on 8 of 128, half: 142 us in the order of the batch, 134 so, both with an address per row) */
    const int perTile = p.c.kvHeads * p.groups;
    const int tile = p.tiles - 1 - id / perTile, rest = id % perTile, piece = rest / p.c.kvHeads;
    int start, fresh, length, keys, seq = 0, row0 = tile * TR;
    if (p.prefix > 0) {
        start = cache_sequence(p.c, p.seq0).start;
        fresh = prefix_tokens(p, start);
        length = keys = p.prefix;
    }
    else {
        if (p.sorted)
            sort_sequences(p, sh);
        const auto sequence = [&](int n) { return p.seq0 + (p.sorted ? sh.order[n] : n); };
        const auto tiles = [&](int n) { return (long long)((cache_sequence(p.c, sequence(n)).fresh * p.per + TR - 1) / TR); };
        const SequenceScan scan = scan_sequences<NW>(p.seqs, sh, tiles);
        long long before = 0;
        const int i = find_sequence(scan, tile, before, sh, tiles);
        seq = sequence(max(i, 0));
        const CacheSequence s = cache_sequence(p.c, seq);
        start = s.start;
        fresh = i < 0 ? 0 : s.fresh;
        length = keys = s.length;
        row0 -= (int)before * TR;
        if (p.causal)
            keys -= fresh - 1 - divided(max(min(row0 + TR, fresh * p.per) - 1, 0), p.perDiv);
    }
    const int units = (max(keys, 0) + UK - 1) / UK;
    int each = units;
    if (p.prefix > 0)
        each = (int)p.part.d / UK;
    else if (p.groups > 1)
        each = (units + p.groups - 1) / p.groups;
    Segment sg;
    sg.s.start = start;
    sg.s.fresh = fresh;
    sg.s.length = length;
    sg.seq = seq;
    sg.head = rest - piece * p.c.kvHeads;
    sg.row0 = row0;
    sg.rows = row0 < fresh * p.per ? fresh * p.per : 0;
    sg.keys = keys;
    sg.first = 0;
    sg.u0 = min(each * piece, units);
    sg.u1 = min(sg.u0 + each, units);
    sg.slot = p.acc ? (tile * p.c.kvHeads + sg.head) * p.groups + piece : -1;
    return sg;
}

/* The sequences of this lane's rows (row0 + 16 q) in a launch over the shared prefix, whose rows are the tokens of all
   sequences: the last one that starts at or before the row's token, searched for in LDS (`from`, N of them at a time). */
template <int QR, int N>
__device__ __forceinline__ void row_sequences(const CachedParams & p, const Segment & sg, int row0, int * from, int (&seq)[QR])
{
    int tok[QR], count[QR];
#pragma unroll
    for (int q = 0; q < QR; q++) {
        const int row = row0 + 16 * q;
        tok[q] = sg.s.start + (row < sg.rows ? divided(row, p.perDiv) : 0);
        count[q] = 0;
    }
    for (int i0 = 0; i0 < p.seqs; i0 += N) {
        const int n = min(N, p.seqs - i0);
        for (int i = threadIdx.x; i < n; i += 256)
            from[i] = p.c.starts[p.seq0 + i0 + i];
        __syncthreads();
#pragma unroll
        for (int q = 0; q < QR; q++) {
            int lo = 0, hi = n;
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (from[mid] <= tok[q])
                    lo = mid + 1;
                else
                    hi = mid;
            }
            count[q] += lo;
        }
        __syncthreads();
    }
#pragma unroll
    for (int q = 0; q < QR; q++)
        seq[q] = p.seq0 + max(count[q] - 1, 0);
}

/* How many positions this lane's rows (row0 + 16 q) see, and the least of the 16 lanes' rows. Rows that a tile does not
   have see everything: they are computed with, never stored. */
template <int QR, int N>
__device__ __forceinline__ int rows_seen(const CachedParams & p, const Segment & sg, int row0, int * from, int (&seen)[QR])
{
    int seq[QR] = {};
    if (p.prefix > 0 && p.c.starts)
        row_sequences<QR, N>(p, sg, row0, from, seq);
    int least = 0x7fffffff;
#pragma unroll
    for (int q = 0; q < QR; q++) {
        const int row = row0 + 16 * q, t = divided(row, p.perDiv);
        int n = 0x7fffffff;
        if (row < sg.rows) {
            n = p.causal ? sg.s.length - sg.s.fresh + t + 1 : sg.s.length;
            if (p.prefix > 0) {
                const CacheSequence s = cache_sequence(p.c, p.c.starts ? seq[q] : p.seq0 + t / p.c.maxNew);
                n = min(p.causal ? s.length - s.fresh + (sg.s.start + t - s.start) + 1 : s.length, p.prefix);
            }
        }
        seen[q] = n;
        least = min(least, n);
    }
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1)
        least = min(least, __shfl_xor(least, d));
    return __builtin_amdgcn_readfirstlane(least);
}

/* The softmax of a row runs on raw scores s and the base-2 scale of p: 2^(s scale2 - shift). Scores are multiplied by |scale|
   (queries take its sign), at least by what leaves hidden scores at minus infinity. `shift` follows the row's maximum only
   where that has grown by more than 2^RISE: until then probabilities are up to 2^RISE, which half holds with the same relative
   precision, and sums and results need no rescaling (at most one block in a few has a row that does). */
constexpr float CACHED_RISE = 8.f;
__device__ __forceinline__ float score_scale(const CachedParams & p)
{
    const float s = fabsf(p.scale) * 1.4426950408889634f;
    return s < 1e-37f ? 1e-37f : s;     /* no fmaxf, which would make 1e-37 of a scale that is no number */
}

/* What the positions that do not exist read: a row of the widest head. */
static __device__ __align__(16) const float zero_row[128] = {};

/* Where a lane's key stands: the address of its row of k and of v, or of a row of zeros. Addresses and not pointers, so that
   they can be handed from lane to lane and loaded from as what they are, global memory. */
struct KeyPlace {
    long long k, v;
    bool there;
};

template <typename T>
__device__ __forceinline__ KeyPlace key_place(const CacheParams & c, int head, int key, int page)
{
    KeyPlace x;
    x.there = page >= 0 && page < c.pages;
    const int r = key - divided(key, c.pageSize) * (int)c.pageSize.d;
    const long long zero = (long long)reinterpret_cast<uintptr_t>(zero_row);
    x.k = x.there ? (long long)reinterpret_cast<uintptr_t>(static_cast<const T *>(c.k) + page * c.kP + r * c.kR + head * c.kH) : zero;
    x.v = x.there ? (long long)reinterpret_cast<uintptr_t>(static_cast<const T *>(c.v) + page * c.vP + r * c.vR + head * c.vH) : zero;
    return x;
}

__device__ __forceinline__ long long lane_of(long long x, int source)
{
    const int lo = __shfl((int)x, source), hi = __shfl((int)(x >> 32), source);
    return ((long long)hi << 32) | (unsigned)lo;
}

/* lane `source`'s x, for a `source` in a scalar register, into scalar registers */
__device__ __forceinline__ long long lane_of_all(long long x, int source)
{
    const int lo = __builtin_amdgcn_readlane((int)x, source), hi = __builtin_amdgcn_readlane((int)(x >> 32), source);
    return ((long long)hi << 32) | (unsigned)lo;
}

/* entry i of a row of the page table (rows are below 4 GiB) */
__device__ __forceinline__ int page_entry(const int * row, int i)
{
    return *(const __attribute__((address_space(1))) int *)((const __attribute__((address_space(1))) char *)row + (unsigned)i * 4u);
}

template <typename V>
__device__ __forceinline__ V load_global(long long address)
{
    return *(const __attribute__((address_space(1))) V *)address;
}

/* CACHED_WHOLE, CACHED_PIECES: `tile` (16 or 32) rows to a pair at most. wide: CACHED_WHOLE without partial results, up to 16 rows,
   as many waves to a workgroup as a CU runs */
int launch_attention_pairs(const CachedParams & p, bool half, int tile, bool wide, int blocks, hipStream_t stream);
/* CACHED_TILES: tiles of 64 or 128 (half) rows; tiles of 16 (half, float) or 32 (float) rows whose
   waves share out the keys */
int launch_attention_tiles(const CachedParams & p, bool half, int tile, int blocks, hipStream_t stream);
int launch_attention_tile_rows(const CachedParams & p, bool half, int tile, int blocks, hipStream_t stream);
/* both launches of a shared prefix in one: `pre` over it in tiles of `tile` rows (64 or 128 half, 16, 32 or 64 float), `own` over each
   sequence's own keys, 16 qr rows */
int launch_attention_prefix(const CachedParams & pre, const CachedParams & own, bool half, int tile, int qr, int preBlocks,
                            int ownBlocks, hipStream_t stream);

/* the partial results of a launch (p.acc, p.stat), and of the launch over the shared prefix before it, to p.out */
struct JoinParams {
    CachedParams p;
    const float * preAcc;               /* NULL: no prefix */
    const float * preStat;
    int prePieces, preRows;             /* pieces of its keys, rows of its tiles */
};
int launch_attention_join(const JoinParams & j, bool half, long long rows, hipStream_t stream);

}  // namespace ntsamd
