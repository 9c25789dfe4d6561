/*
 * What the kernels of the cached attention share (attention_cached.hip, attention_cached_join.hip): how the keys of a
 * batch are dealt out to workgroups, found again by the kernel that joins partial results.
 */
#pragma once
#include "cache.h"

namespace ntsamd {

struct CachedShared {
    float acc[4][16][132];
    float stat[4][16][2];
    long long sums[4];
    long long before;
    int found;
};

/* units of keys of one (sequence, key head) pair of a CACHED_FLAT launch: at least one where there are tokens to answer */
template <int UK>
__device__ __forceinline__ int units_of(const CachedParams & p, const CacheSequence & s)
{
    return s.fresh > 0 ? max((max(s.length - p.first, 0) + UK - 1) / UK, 1) : 0;
}

/* Sums over the sequences of a launch, weight(i) each: every thread of the 256 takes a run of sequences. */
struct SequenceScan {
    long long before, sum, total;       /* of the sequences before this thread's, of this thread's, of all */
    int from, to;                       /* this thread's sequences */
};

template <typename W>
__device__ __forceinline__ SequenceScan scan_sequences(int count, CachedShared & sh, W weight)
{
    SequenceScan r;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int run = (count + 255) / 256;
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
    for (int w = 0; w < 4; w++) {
        if (w < wave)
            r.before += sh.sums[w];
        r.total += sh.sums[w];
    }
    return r;
}

/* the sequence of a launch in which place `at` of the sum falls, and the sum before it; -1 past the end */
template <typename W>
__device__ __forceinline__ int find_sequence(const SequenceScan & r, long long at, long long & before, CachedShared & sh, W weight)
{
    if (at >= r.total)
        return -1;
    if (at >= r.before && at < r.before + r.sum) {
        long long b = r.before;
        int i = r.from;
        for (long long w = weight(i); at >= b + w; w = weight(i)) {
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

/* CACHED_FLAT: unit x of the whole launch belongs to workgroup owner(x), whose units are start(w) .. start(w + 1) - 1 */
struct FlatPlan {
    SequenceScan scan;
    int groups;
    __device__ __forceinline__ long long start(int w) const { return scan.total * w / groups; }
    __device__ __forceinline__ int owner(long long x) const { return (int)(((x + 1) * groups - 1) / scan.total); }
};

/* a workgroup's four waves take a unit each at a time: no more workgroups than whole rounds */
template <int UK>
__device__ __forceinline__ FlatPlan flat_plan(const CachedParams & p, CachedShared & sh)
{
    FlatPlan f;
    f.scan = scan_sequences(p.seqs, sh, [&](int i) { return (long long)units_of<UK>(p, cache_sequence(p.c, p.seq0 + i)) * p.c.kvHeads; });
    f.groups = (int)min((long long)p.groups, (f.scan.total + 3) / 4);
    return f;
}

/* tokens of the sequences of a launch, which begin at row `start` */
__device__ __forceinline__ int prefix_tokens(const CachedParams & p, int start)
{
    const int most = p.seqs * p.c.maxNew;
    if (!p.c.starts)
        return most;
    return min(max(min(p.c.starts[p.seq0 + p.seqs], p.c.tokens) - start, 0), most);
}

int launch_attention_cached(const CachedParams & p, bool half, int qr, int blocks, hipStream_t stream);

/* the partial results of a launch (p.acc, p.stat), and of the launch over the shared prefix before it, to p.out */
struct JoinParams {
    CachedParams p;
    const float * preAcc;               /* NULL: no prefix */
    const float * preStat;
    int prePieces, preRows;             /* pieces of its keys, rows of its tiles */
};
int launch_attention_join(const JoinParams & j, bool half, int blocks, hipStream_t stream);

}  // namespace ntsamd
