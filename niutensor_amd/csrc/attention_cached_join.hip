/*
 * The partial results of the cached attention (attention_cached.hip) joined: a row's pieces i, each an unnormalised row
 * a_i with the maximum m_i and the sum l_i of its softmax (base 2), give
 *   out = sum_i 2^(m_i - M) a_i / sum_i 2^(m_i - M) l_i,   M = max_i m_i.
 * One workgroup per row: lanes of 4 columns, eight groups of them, which take the pieces in turn, in the order of the
 * keys, and meet in LDS in a fixed order, so results are the same bits on every run. Which pieces a row has is
 * worked out from the lengths as the first kernel did it: nothing about them is stored.
 */
#include "gemm_common.h"
#include "gemm_f16.h"       /* half_t */
#include "attention_cached.h"

namespace ntsamd {

namespace {

template <typename T, int UK>
__global__ void __launch_bounds__(256)
attention_join_kernel(const JoinParams j)
{
    __shared__ CachedScan sh;
    __shared__ float partAcc[8][128], partStat[8][2];
    const CachedParams & p = j.p;
    const int id = (int)blockIdx.x, kv = p.c.kvHeads;
    const int unit = id / p.rows, row = id - unit * p.rows;     /* a pair or a tile, and a row of it */
    int head, inSeq;                    /* key head; the row among its sequence's */
    CacheSequence s;
    /* the pieces: slot0, then step apart from slot1 on */
    int pieces = 1, slot0, slot1 = 0, step = 0;
    if (p.mode == CACHED_TILES) {
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
        slot1 = slot0 + 1;
        step = 1;
    }
    else {
        const int i = unit / kv;
        head = unit - i * kv;
        s = cache_sequence(p.c, p.seq0 + i);
        inSeq = row;
        slot0 = unit;
        if (p.mode == CACHED_FLAT) {
            const FlatPlan f = flat_plan<UK>(p, sh);
            if (i >= f.scan.from && i < f.scan.to) {
                long long b = f.scan.before;
                for (int n = f.scan.from; n < i; n++)
                    b += (long long)units_of<UK>(p, cache_sequence(p.c, p.seq0 + n)) * kv;
                sh.before = b;
            }
            __syncthreads();
            const int units = units_of<UK>(p, s);
            if (units == 0)
                return;
            const long long begin = sh.before + (long long)head * units;
            const int first = f.owner(begin), last = f.owner(begin + units - 1);
            pieces = last - first + 1;
            if (pieces == 1) {
                if (p.first == 0)
                    return;             /* one workgroup had them all: the result stands in out */
                slot0 = 2 * p.groups + unit;
            }
            else {
                slot0 = 2 * first + (f.start(first) == begin ? 0 : 1);
                slot1 = 2 * (first + 1);
                step = 2;
            }
        }
    }
    if (inSeq >= s.fresh * p.per)
        return;
    const int t = divided(inSeq, p.perDiv), dh = p.c.dh;

    /* the prefix's launch counts rows from the first token of the first sequence */
    int preSlot = 0, preRow = 0, pre = 0;
    if (j.preAcc) {
        const int start0 = cache_sequence(p.c, p.seq0).start;
        const int fromStart = s.start - start0 + t;
        if (fromStart >= 0 && fromStart < prefix_tokens(p, start0)) {
            const int r = fromStart * p.per + (inSeq - t * p.per);
            const int tile = r / j.preRows;
            preRow = r - tile * j.preRows;
            preSlot = (tile * kv + head) * j.prePieces;
            pre = j.prePieces;
        }
    }

    const int lane = threadIdx.x & 31, group = threadIdx.x >> 5, col = 4 * lane;
    float mx = -INFINITY, sum = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int i = group; i < pre + pieces; i += 8) {
        const float * a;
        const float * st;
        if (i < pre) {
            const long long at = (long long)(preSlot + i) * j.preRows + preRow;
            a = j.preAcc + at * dh;
            st = j.preStat + 2 * at;
        }
        else {
            const long long at = (long long)(i == pre ? slot0 : slot1 + (i - pre - 1) * step) * p.rows + row;
            a = p.acc + at * dh;
            st = p.stat + 2 * at;
        }
        const float m = st[0], l = st[1];
        const f32x4 x = col < dh ? *reinterpret_cast<const f32x4 *>(a + col) : f32x4{0.f, 0.f, 0.f, 0.f};
        const float newMax = fmaxf(mx, m);
        const float shift = newMax == -INFINITY ? 0.f : newMax;
        const float f0 = __builtin_amdgcn_exp2f(mx - shift), f1 = __builtin_amdgcn_exp2f(m - shift);
        sum = sum * f0 + l * f1;
        acc = acc * f0 + x * f1;
        mx = newMax;
    }
    if (lane == 0) {
        partStat[group][0] = mx;
        partStat[group][1] = sum;
    }
    *reinterpret_cast<f32x4 *>(&partAcc[group][col]) = acc;
    __syncthreads();
    if (threadIdx.x < 32 && col < dh) {
        float top = partStat[0][0];
#pragma unroll
        for (int g = 1; g < 8; g++)
            top = fmaxf(top, partStat[g][0]);
        const float shift = top == -INFINITY ? 0.f : top;
        float total = 0.f;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < 8; g++) {
            const float f = __builtin_amdgcn_exp2f(partStat[g][0] - shift);
            total += f * partStat[g][1];
            o += *reinterpret_cast<const f32x4 *>(&partAcc[g][col]) * f;
        }
        const float inv = total == 0.f ? 0.f : 1.f / total;
        typedef T vec __attribute__((ext_vector_type(4)));
        vec v;
#pragma unroll
        for (int e = 0; e < 4; e++)
            v[e] = (T)(o[e] * inv);
        T * out = static_cast<T *>(p.out) + (long long)(s.start + t) * p.oT + (head * p.per + inSeq - t * p.per) * p.oH;
        *reinterpret_cast<vec *>(out + col) = v;
    }
}

}  // namespace

int launch_attention_join(const JoinParams & j, bool half, int blocks, hipStream_t stream)
{
    /* UK: the unit of attention_cached_kernel for the type */
    if (half)
        hipLaunchKernelGGL((attention_join_kernel<half_t, 32>), dim3((unsigned)blocks), dim3(256), 0, stream, j);
    else
        hipLaunchKernelGGL((attention_join_kernel<float, 16>), dim3((unsigned)blocks), dim3(256), 0, stream, j);
    return (int)hipGetLastError();
}

}  // namespace ntsamd
