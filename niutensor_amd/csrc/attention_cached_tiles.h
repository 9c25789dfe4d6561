/*
 * Attention over a cache on pages for many query rows in half: pieces of text against what is in the cache, and the
 * queries of a whole batch against a prefix they share (ntsamd_attention_cached, ntsamd_attention_prefix; the few rows of a
 * decoding step and float go to attention_cached.hip).
 *
 * Bound by the matrix instructions and what feeds them, so keys and values go through LDS once for all rows of a
 * workgroup, on the plan of attention_f16.hip: 64 QR rows (tokens x the query heads that share a key head) of a tile, 16 QR
 * per wave; blocks of 64 keys; both products transposed, so that probabilities pass from accumulator to operand inside
 * a lane; values read back by transposing LDS reads. What is different is where the keys stand: lane l of every wave looks
 * up the page of key l of a block, one block ahead, and hands its address to the lanes that fetch the row. Rows of a
 * tile see different numbers of keys; only the blocks in which some row's last key falls, or which have an absent page, take the
 * comparisons. Fetches of keys that a tile does not have read a row of zeros.
 */
#pragma once
#include "gemm_common.h"
#include "gemm_f16.h"       /* half_t, lds_read_tr16 */
#include "attention.h"
#include "attention_cached.h"

namespace ntsamd {

template <int DHM> struct CachedTilesShared {
    static constexpr int PITCH = DHM * 2 + 16;      /* bytes per LDS row: 16 mod 128, so 16-byte reads of consecutive rows
                                                       walk through the banks */
    __attribute__((aligned(16))) char k[CACHED_TILE_KEYS * PITCH];
    __attribute__((aligned(16))) char v[CACHED_TILE_KEYS * PITCH];
    CachedScan scan;
};

/* workgroup `id` of a CACHED_TILES launch over half tensors, tiles of 64 QR rows */
template <int DHM, int QR>
__device__ __forceinline__ void attend_tile(const CachedParams & p, int id, CachedTilesShared<DHM> & sh)
{
    constexpr int KB = CACHED_TILE_KEYS, TR = 64 * QR;
    constexpr int PITCH = CachedTilesShared<DHM>::PITCH;
    constexpr int NT = DHM / 32, ND = DHM / 16, NJ = KB / 16;
    constexpr int TPR = DHM / 8;             /* threads per row when staging */
    constexpr int RSTEP = 256 / TPR, LOADS = KB / RSTEP;

    char * const Ks = sh.k;
    char * const Vs = sh.v;
    const CacheParams & c = p.c;
    const int tid = threadIdx.x;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m = lane & 15, g = lane >> 4;
    const int dh = c.dh;

    const Segment sg = uniform(tile_segment<TR, KB>(p, sh.scan, id));
    if (sg.rows == 0)
        return;
    const int row0 = sg.row0 + wave * (16 * QR) + m;
    int seen[QR];
    const int seenMin = rows_seen<QR, KB * PITCH / 4>(p, sg, row0, reinterpret_cast<int *>(Ks), seen);

    /* ---- where the keys of a block stand: lane l looks after key l ---- */
    const int * table = c.table + (long long)sg.seq * c.tablePages;
    auto page_of = [&](int u) {
        const int key = p.first + u * KB + lane;
        return u < sg.u1 && key < sg.keys ? page_entry(table, divided(key, c.pageSize)) : -1;
    };
    const int sr0 = tid / TPR, sc = (tid % TPR) * 8;
    const int sLds = sr0 * PITCH + sc * 2;
    f16x8 kreg[LOADS], vreg[LOADS];
    unsigned long long there = 0;            /* which keys of the block being fetched exist */
    long long vRow = 0;
    const int col = sc < dh ? 2 * sc : 0;    /* columns past dh: the row's first, which meet zeros of q or are not stored */
    auto load_k = [&](int u, int page) {
        const KeyPlace at = key_place<half_t>(c, sg.head, p.first + u * KB + lane, page);
        vRow = at.v;
        there = __ballot(at.there);
#pragma unroll
        for (int s = 0; s < LOADS; s++)
            kreg[s] = load_global<f16x8>(lane_of(at.k, sr0 + s * RSTEP) + col);
    };
    auto load_v = [&]() {
#pragma unroll
        for (int s = 0; s < LOADS; s++)
            vreg[s] = load_global<f16x8>(lane_of(vRow, sr0 + s * RSTEP) + col);
    };
    int page = page_of(sg.u0);
    load_k(sg.u0, page);
    load_v();
    page = page_of(sg.u0 + 1);

    /* ---- Q fragments ---- */
    f16x8 qf[QR][NT];
#pragma unroll
    for (int q = 0; q < QR; q++) {
        const int row = row0 + 16 * q;
        const bool has = row < sg.rows;
        const int t = has ? divided(row, p.perDiv) : 0;
        const int h = sg.head * p.per + (has ? row - t * p.per : 0);
        const half_t * qr = static_cast<const half_t *>(p.q) + (long long)(sg.s.start + t) * p.qT + h * p.qH;
#pragma unroll
        for (int t4 = 0; t4 < NT; t4++) {
            const int col = 32 * t4 + 8 * g;
            const f16x8 z = {0, 0, 0, 0, 0, 0, 0, 0};
            qf[q][t4] = has && col < dh ? *reinterpret_cast<const f16x8 *>(qr + col) : z;
            if (p.scale < 0.f)
                qf[q][t4] = -qf[q][t4];
        }
    }

    f32x4 accO[QR][ND];
    float rowMax[QR], rowSum[QR];
#pragma unroll
    for (int q = 0; q < QR; q++) {
#pragma unroll
        for (int d = 0; d < ND; d++)
            accO[q][d] = f32x4{0.f, 0.f, 0.f, 0.f};
        rowMax[q] = -INFINITY;
        rowSum[q] = 0.f;
    }
    const float scale2 = score_scale(p);
    /* where this lane points for the transposing reads: row 4 g + (m / 4) of a 16-key block, columns 4 (m % 4) .. + 3 */
    const int trOff = (4 * g + (m >> 2)) * PITCH + (m & 3) * 8;

    for (int u = sg.u0; u < sg.u1; u++) {
        const int key0 = p.first + u * KB;
        const unsigned long long exist = there;
#pragma unroll
        for (int s = 0; s < LOADS; s++)
            *reinterpret_cast<f16x8 *>(&Ks[sLds + s * RSTEP * PITCH]) = kreg[s];
        __syncthreads();
        load_k(u + 1, page);                 /* past the end: rows of zeros */
        page = page_of(u + 2);

        /* ---- S^T = K Q^T ---- */
        f32x4 accS[QR][NJ];
#pragma unroll
        for (int q = 0; q < QR; q++)
#pragma unroll
            for (int j = 0; j < NJ; j++)
                accS[q][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                const f16x8 kf = *reinterpret_cast<const f16x8 *>(&Ks[(16 * j + m) * PITCH + 64 * t + 16 * g]);
#pragma unroll
                for (int q = 0; q < QR; q++)
                    accS[q][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[q][t], accS[q][j], 0, 0, 0);
            }

        /* ---- running softmax of the lane's rows ---- */
        f16x4 pf[QR][NJ];
        float top[QR];
        bool risen = false;
        const bool cut = exist != ~0ull || key0 + KB > seenMin;
#pragma unroll
        for (int q = 0; q < QR; q++) {
            if (cut) {
#pragma unroll
                for (int j = 0; j < NJ; j++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int at = 16 * j + 4 * g + r;
                        if (!((exist >> at) & 1) || key0 + at >= seen[q])
                            accS[q][j][r] = -INFINITY;
                    }
            }
            float mx = accS[q][0][0];
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    mx = fmaxf(mx, accS[q][j][r]);
            top[q] = lane_groups_max(mx) * scale2;
            risen = risen || top[q] > rowMax[q] + CACHED_RISE;
        }
        if (__any(risen)) {
#pragma unroll
            for (int q = 0; q < QR; q++) {
                const float newMax = fmaxf(rowMax[q], top[q]);
                const float corr = __builtin_amdgcn_exp2f(rowMax[q] - (newMax == -INFINITY ? 0.f : newMax));
                rowSum[q] *= corr;
                rowMax[q] = newMax;
#pragma unroll
                for (int d = 0; d < ND; d++)
                    accO[q][d] *= corr;
            }
        }
#pragma unroll
        for (int q = 0; q < QR; q++) {
            const float shift = rowMax[q] == -INFINITY ? 0.f : rowMax[q];
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float e = __builtin_amdgcn_exp2f(fmaf(accS[q][j][r], scale2, -shift));
                    rowSum[q] += e;                      /* this lane's keys only: the four lanes of a row meet at the end */
                    pf[q][j][r] = (half_t)e;
                }
        }

#pragma unroll
        for (int s = 0; s < LOADS; s++)
            *reinterpret_cast<f16x8 *>(&Vs[sLds + s * RSTEP * PITCH]) = vreg[s];
        __syncthreads();
        load_v();

        /* ---- O^T += V^T P^T, 32 keys per MFMA: its k index 8 g + e stands for key 4 g + e of the first 16-key block of a
           pair for e < 4 and for key 4 g + e - 4 of the second for e >= 4 ---- */
#pragma unroll
        for (int j = 0; j < NJ; j += 2)
#pragma unroll
            for (int d = 0; d < ND; d++) {
                const f16x4 lo = lds_read_tr16(reinterpret_cast<const half_t *>(&Vs[16 * j * PITCH + trOff + 32 * d]));
                const f16x4 hi = lds_read_tr16(reinterpret_cast<const half_t *>(&Vs[16 * (j + 1) * PITCH + trOff + 32 * d]));
                const f16x8 vf = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                for (int q = 0; q < QR; q++) {
                    const f16x8 pp = __builtin_shufflevector(pf[q][j], pf[q][j + 1], 0, 1, 2, 3, 4, 5, 6, 7);
                    accO[q][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pp, accO[q][d], 0, 0, 0);
                }
            }
    }

    /* ---- register r of block d is column 16 d + 4 g + r of the lane's row ---- */
#pragma unroll
    for (int q = 0; q < QR; q++) {
        const float total = lane_groups_sum(rowSum[q]);
        const int row = row0 + 16 * q;
        if (row >= sg.rows)
            continue;
        if (sg.slot < 0) {
            const int t = divided(row, p.perDiv);
            half_t * out = static_cast<half_t *>(p.out) + (long long)(sg.s.start + t) * p.oT + (sg.head * p.per + row - t * p.per) * p.oH;
            const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
            for (int d = 0; d < ND; d++) {
                const int col = 16 * d + 4 * g;
                if (col < dh) {
                    f16x4 o;
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        o[r] = (half_t)(accO[q][d][r] * inv);
                    *reinterpret_cast<f16x4 *>(out + col) = o;
                }
            }
        }
        else {
            const long long at = (long long)sg.slot * TR + (row - sg.row0);
#pragma unroll
            for (int d = 0; d < ND; d++) {
                const int col = 16 * d + 4 * g;
                if (col < dh)
                    *reinterpret_cast<f32x4 *>(p.acc + at * dh + col) = accO[q][d];
            }
            if (g == 0) {
                p.stat[2 * at] = rowMax[q];
                p.stat[2 * at + 1] = total;
            }
        }
    }
}

}  // namespace ntsamd
