/*
 * The partial results of the cached attention (attention_cached.hip) joined: a row's pieces i, each an unnormalised row
 * a_i with the maximum m_i and the sum l_i of its softmax (base 2), give
 *   out = sum_i 2^(m_i - M) a_i / sum_i 2^(m_i - M) l_i,   M = max_i m_i.
 * A lane takes 4 columns of the pieces of a row, in the order of the keys; where a row may have many pieces eight groups of
 * lanes take them in turn and meet in LDS, in a fixed order, so results are the same bits on every run.
 * 2048 rows of 128 columns in up to four pieces, or 32 rows in 65: 5 us, most of it the start of a kernel and two dependent loads.
 */
#include "gemm_common.h"
#include "gemm_f16.h"       /* half_t */
#include "attention_cached.h"

namespace ntsamd {

namespace {

/* TILES: the rows of a CACHED_TILES launch. MANY: eight rows to a workgroup, a group of lanes each, otherwise a row to a
   workgroup. */
template <typename T, bool TILES, bool MANY>
__global__ void __launch_bounds__(256)
attention_join_kernel(const JoinParams j)
{
    __shared__ CachedScan sh;
    __shared__ float partAcc[MANY ? 1 : 8][128], partStat[8][2];
    const CachedParams & p = j.p;
    const int lane = threadIdx.x & 31, group = threadIdx.x >> 5, col = 4 * lane;
    const int kv = p.c.kvHeads, dh = p.c.dh;
    const int id = MANY ? (int)blockIdx.x * 8 + group : (int)blockIdx.x;
    const int unit = id / p.rows, row = id - unit * p.rows;     /* a pair or a tile, and a row of it */
    int head, inSeq;                    /* key head; the row among its sequence's */
    CacheSequence s;
    int pieces = 1, slot0 = unit;
    if constexpr (TILES) {
        const int tile = unit / kv;
        head = unit - tile * kv;
        const auto tiles = [&](int n) { return (long long)((cache_sequence(p.c, p.seq0 + n).fresh * p.per + p.rows - 1) / p.rows); };
        const SequenceScan scan = scan_sequences(p.seqs, sh, tiles);
        long long before;
        const int i = find_sequence(scan, tile, before, sh, tiles);
        if (i < 0)
            return;
        s = cache_sequence(p.c, p.seq0 + i);
        inSeq = (tile - (int)before) * p.rows + row;
        pieces = p.groups;
        slot0 = unit * p.groups;
    }
    else {
        const int i = unit / kv;
        if (MANY && i >= p.seqs)
            return;
        head = unit - i * kv;
        s = cache_sequence(p.c, p.seq0 + i);
        inSeq = row;
        if (p.mode == CACHED_PIECES && s.fresh > 0) {
            slot0 = p.slots[2 * unit];
            pieces = p.slots[2 * unit + 1];
            if (pieces == 0)
                return;                 /* one workgroup had all keys: the result stands in out */
        }
    }
    if (inSeq >= s.fresh * p.per)
        return;
    const int t = divided(inSeq, p.perDiv);

    /* the prefix's launch counts rows from the first token of the first sequence */
    int preSlot = 0, preRow = 0, pre = 0;
    if (!TILES && j.preAcc) {
        const int start0 = cache_sequence(p.c, p.seq0).start;
        const int fromStart = s.start - start0 + t;
        if (fromStart >= 0 && fromStart < prefix_tokens(p, start0)) {
            const int r = fromStart * p.per + (inSeq - t * p.per);
            const int tile = r / j.preRows;
            preRow = r - tile * j.preRows;
            preSlot = (tile * kv + head) * j.prePieces;
            pre = s.length >= p.first ? j.prePieces : divided(s.length, p.part);        /* see first_of */
        }
    }

    float mx = -INFINITY, sum = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    constexpr int AHEAD = MANY ? 8 : 4; /* pieces of a group in flight (42 pieces of 80 rows: 20.5 us the call with 4, 18.0 with 8) */
    constexpr int STEP = MANY ? 1 : 8;
    for (int i0 = MANY ? 0 : group; i0 < pre + pieces; i0 += STEP * AHEAD) {
        float m[AHEAD], l[AHEAD];
        f32x4 x[AHEAD];
        float newMax = mx;
#pragma unroll
        for (int e = 0; e < AHEAD; e++) {
            const int i = min(i0 + STEP * e, pre + pieces - 1);
            const bool own = i >= pre;
            const long long at = own ? (long long)(slot0 + i - pre) * p.rows + row : (long long)(preSlot + i) * j.preRows + preRow;
            const float * st = (own ? p.stat : j.preStat) + 2 * at;
            const bool there = i0 + STEP * e < pre + pieces;
            m[e] = there ? st[0] : -INFINITY;
            l[e] = there ? st[1] : 0.f;
            x[e] = there && col < dh ? *reinterpret_cast<const f32x4 *>((own ? p.acc : j.preAcc) + at * dh + col) : f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int e = 0; e < AHEAD; e++)
            newMax = fmaxf(newMax, m[e]);
        const float shift = newMax == -INFINITY ? 0.f : newMax;
        const float f0 = __builtin_amdgcn_exp2f(mx - shift);
        sum *= f0;
        acc *= f0;
#pragma unroll
        for (int e = 0; e < AHEAD; e++) {
            const float f = __builtin_amdgcn_exp2f(m[e] - shift);
            sum += l[e] * f;
            acc += x[e] * f;
        }
        mx = newMax;
    }
    if constexpr (!MANY) {
        if (lane == 0) {
            partStat[group][0] = mx;
            partStat[group][1] = sum;
        }
        *reinterpret_cast<f32x4 *>(&partAcc[group][col]) = acc;
        __syncthreads();
        if (threadIdx.x >= 32)
            return;
        float top = partStat[0][0];
#pragma unroll
        for (int g = 1; g < 8; g++)
            top = fmaxf(top, partStat[g][0]);
        const float shift = top == -INFINITY ? 0.f : top;
        sum = 0.f;
        acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < 8; g++) {
            const float f = __builtin_amdgcn_exp2f(partStat[g][0] - shift);
            sum += f * partStat[g][1];
            acc += *reinterpret_cast<const f32x4 *>(&partAcc[g][col]) * f;
        }
    }
    if (col < dh) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        typedef T vec __attribute__((ext_vector_type(4)));
        vec v;
#pragma unroll
        for (int e = 0; e < 4; e++)
            v[e] = (T)(acc[e] * inv);
        T * out = static_cast<T *>(p.out) + (long long)(s.start + t) * p.oT + (head * p.per + inSeq - t * p.per) * p.oH;
        *reinterpret_cast<vec *>(out + col) = v;
    }
}

template <typename T>
int launch_type(const JoinParams & j, long long rows, hipStream_t stream)
{
    /* Tiles have whole eights of rows, each in the same few pieces. Pairs whose keys are whole, behind a prefix: a row to a workgroup has
       eight pieces at a time, eight rows to a workgroup are an eighth of the workgroups, which is faster where rows are many for the
       pieces. The call with eight rows against one, 16 to 256 sequences, 8 to 32 heads, both types: 512 rows in 2 pieces the same,
       in 8 8 to 10 % slower; 1024 in 4 2 to 6 % faster, in 8 2 to 11 % slower; 2048 in 4 4 to 7 % faster, in 8 0 to 3 % faster, in 15
       the same; 4096 in 4 10 to 19 % faster, in 8 3 to 12 %. */
    const dim3 one((unsigned)rows), eight((unsigned)((rows + 7) / 8)), block(256);
    if (j.p.mode == CACHED_TILES)
        hipLaunchKernelGGL((attention_join_kernel<T, true, true>), eight, block, 0, stream, j);
    else if (j.p.mode == CACHED_WHOLE && 256LL * j.prePieces <= rows)
        hipLaunchKernelGGL((attention_join_kernel<T, false, true>), eight, block, 0, stream, j);
    else
        hipLaunchKernelGGL((attention_join_kernel<T, false, false>), one, block, 0, stream, j);
    return (int)hipGetLastError();
}

}  // namespace

int launch_attention_join(const JoinParams & j, bool half, long long rows, hipStream_t stream)
{
    return half ? launch_type<half_t>(j, rows, stream) : launch_type<float>(j, rows, stream);
}

}  // namespace ntsamd
