/*
 * Float tiles of many rows of a sequence: the plan of attention_cached_tiles.h on the float matrix instruction, which takes
 * 32 cycles for 16 rows x 16 keys x 4 columns: bound by it, and softmax, LDS and the fetches hide behind it. (Tiles of 16 or 32
 * rows whose waves share the keys, attention_cached_rows.h, read a key row for each of them: 8 or 16 operations a byte, bound by
 * the caches when many run.) 512 tokens of 8 sequences of 2048 positions, not causal, 8 heads of 128, in one piece: 295 us, 117 TFLOP/s
 * (tiles of 32 rows 103, of 16 82; a large product 146); of 96 columns 109 (85, 69), of 64 112 (93, 79), of 32 96 (79, 67); 8 times 1024
 * on 4096, 32 heads on 8 of 128: 122. (The plan's estimate takes the lengths of a batch for uneven: in these calls it takes tiles of 32
 * rows with 128 columns, 329 us, and two pieces with fewer.) The matrix unit is busy 81 % of a wave's life there; the rest is the softmax
 * and the barrier, which its one neighbour on the SIMD covers in part.
 *
 * S^T = K Q^T: lane (m, g) = (l % 16, l / 16) feeds columns 16 t + 4 g + e, e = 0..3, of key m and of query m, one 16-byte read for four
 * MFMAs. O^T = V^T P^T: it holds the probabilities of keys 4 g + r, feeds them as they are, and of V reads VC neighbouring columns,
 * VC (16 h + m) .., of key 4 g + r for VC MFMAs, whose rows i stand for columns VC (16 h + i) + c. Everything is float: no rounding
 * but the products' own.
 */
#pragma once
#include "attention_cached_tiles.h"

namespace ntsamd {

/* workgroup `id` of a CACHED_TILES launch over float tensors, tiles of 64 rows (128 were 2 % faster at
   their best, and fewer). DHC: columns computed with, at least dh */
template <int DHM, int DHC>
__device__ __forceinline__ void attend_tile_f32(const CachedParams & p, int id, CachedTilesShared<float, DHM> & sh)
{
    typedef CachedTilesShared<float, DHM> Shared;
    constexpr int QR = 1, KB = Shared::KB, TR = 64 * QR, ROW = Shared::ROW;
    constexpr int NT = DHC / 16, NJ = KB / 16;
    constexpr int VC = DHC % 64 == 0 ? 4 : 2, NH = DHC / (16 * VC);
    constexpr unsigned long long ALL = KB == 64 ? ~0ull : 0xffffffffull;
    typedef float VPiece __attribute__((ext_vector_type(VC)));

    const int tid = threadIdx.x;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m = lane & 15, g = lane >> 4;
    const int dh = p.c.dh;

    const Segment sg = uniform(tile_segment<TR, KB>(p, sh.scan, id));
    if (sg.rows == 0)
        return;
    TileFetch<float, DHM> from(p, sg, sh, wave, lane);
    /* the first block is on its way before anything is asked about the rows */
    if (sg.u0 < sg.u1)
        from.block(sg.u0, from.page_of(sg.u0));
    int page = from.page_of(sg.u0 + 1);

    const int row0 = sg.row0 + wave * (16 * QR) + m;
    int seen[QR];
    const int seenMin = rows_seen<QR, Shared::BLOCK / 4>(p, sg, row0, reinterpret_cast<int *>(sh.k[1]), seen);

    f32x4 qf[QR][NT];
#pragma unroll
    for (int q = 0; q < QR; q++) {
        const int row = row0 + 16 * q;
        const bool has = row < sg.rows;
        const int t = has ? divided(row, p.perDiv) : 0;
        const int h = sg.head * p.per + (has ? row - t * p.per : 0);
        const float * qr = static_cast<const float *>(p.q) + (long long)(sg.s.start + t) * p.qT + h * p.qH;
#pragma unroll
        for (int t4 = 0; t4 < NT; t4++) {
            const int col = 16 * t4 + 4 * g;
            qf[q][t4] = has && col < dh ? *reinterpret_cast<const f32x4 *>(qr + col) : f32x4{0.f, 0.f, 0.f, 0.f};
            if (p.scale < 0.f)
                qf[q][t4] = -qf[q][t4];
        }
    }

    f32x4 accO[QR][NH][VC];
    float rowMax[QR], rowSum[QR];
#pragma unroll
    for (int q = 0; q < QR; q++) {
#pragma unroll
        for (int h = 0; h < NH; h++)
#pragma unroll
            for (int c = 0; c < VC; c++)
                accO[q][h][c] = f32x4{0.f, 0.f, 0.f, 0.f};
        rowMax[q] = -INFINITY;
        rowSum[q] = 0.f;
    }
    const float scale2 = score_scale(p);
    /* where this lane reads keys (row m of a 16-key block, piece 4 t + g) and values (row 4 g + r, columns VC (16 h + m) ..) */
    int kAt[NT], vAt[4][NH];
#pragma unroll
    for (int t = 0; t < NT; t++)
        kAt[t] = m * ROW + 16 * ((4 * t + g) ^ Shared::swizzle(m));
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
        for (int h = 0; h < NH; h++) {
            const int byte = 4 * VC * (16 * h + m), row = 4 * g + r;
            vAt[r][h] = row * ROW + 16 * ((byte >> 4) ^ Shared::swizzle(row)) + (byte & 15);
        }

    for (int u = sg.u0; u < sg.u1; u++) {
        const int key0 = u * KB;
        const unsigned long long exist = from.there;
        const char * const Ks = sh.k[(u - sg.u0) & 1];
        const char * const Vs = sh.v[(u - sg.u0) & 1];
        from.landed();
        if (u + 1 < sg.u1)
            from.block(u + 1, page);
        page = from.page_of(u + 2);

        /* ---- S^T = K Q^T ---- */
        f32x4 s[QR][NJ];
#pragma unroll
        for (int q = 0; q < QR; q++)
#pragma unroll
            for (int j = 0; j < NJ; j++)
                s[q][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        f32x4 kf[2][NJ];
#pragma unroll
        for (int j = 0; j < NJ; j++)
            kf[0][j] = *reinterpret_cast<const f32x4 *>(&Ks[kAt[0] + 16 * j * ROW]);
#pragma unroll
        for (int t = 0; t < NT; t++) {
            /* a step's operands are read while the one before is multiplied: left to itself the compiler reads them right before */
            if (t + 1 < NT) {
#pragma unroll
                for (int j = 0; j < NJ; j++)
                    kf[(t + 1) & 1][j] = *reinterpret_cast<const f32x4 *>(&Ks[kAt[t + 1] + 16 * j * ROW]);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int j = 0; j < NJ; j++)
#pragma unroll
                    for (int q = 0; q < QR; q++)
                        s[q][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[t & 1][j][e], qf[q][t][e], s[q][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        VPiece vf[2][NH];
#pragma unroll
        for (int h = 0; h < NH; h++)
            vf[0][h] = *reinterpret_cast<const VPiece *>(&Vs[vAt[0][h]]);
        __builtin_amdgcn_sched_barrier(0);

        /* ---- running softmax of the lane's rows ---- */
        const bool cut = exist != ALL || key0 + KB > seenMin;
#pragma unroll
        for (int q = 0; q < QR; q++) {
            if (cut)
                hide_scores(s[q], exist, seen[q] - key0, g);
            float mx = s[q][0][0];
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    mx = fmaxf(mx, s[q][j][r]);
            mx = lane_groups_max(mx) * scale2;
            if (__any(mx > rowMax[q] + CACHED_RISE)) {
                const float newMax = fmaxf(rowMax[q], mx);
                const float corr = __builtin_amdgcn_exp2f(rowMax[q] - (newMax == -INFINITY ? 0.f : newMax));
                rowSum[q] *= corr;
                rowMax[q] = newMax;
#pragma unroll
                for (int h = 0; h < NH; h++)
#pragma unroll
                    for (int c = 0; c < VC; c++)
                        accO[q][h][c] *= corr;
            }
            const float shift = rowMax[q] == -INFINITY ? 0.f : rowMax[q];
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    s[q][j][r] = __builtin_amdgcn_exp2f(fmaf(s[q][j][r], scale2, -shift));
                    rowSum[q] += s[q][j][r];            /* this lane's keys only: the lanes of a row meet at the end */
                }
        }

        /* ---- O^T += V^T P^T ---- */
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int at = 0; at < 4 * NJ; at++) {
            const int j = at >> 2, r = at & 3, n = at + 1;
            if (n < 4 * NJ) {
#pragma unroll
                for (int h = 0; h < NH; h++)
                    vf[n & 1][h] = *reinterpret_cast<const VPiece *>(&Vs[vAt[n & 3][h] + 16 * (n >> 2) * ROW]);
                __builtin_amdgcn_sched_group_barrier(0x100, NH, 0);
            }
#pragma unroll
            for (int h = 0; h < NH; h++)
#pragma unroll
                for (int c = 0; c < VC; c++)
#pragma unroll
                    for (int q = 0; q < QR; q++)
                        accO[q][h][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[at & 1][h][c], s[q][j][r], accO[q][h][c], 0, 0, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, NH * VC * QR, 0);
        }
    }

    /* ---- register r of MFMA c of set h is column VC (16 h + 4 g + r) + c of the lane's row ---- */
#pragma unroll
    for (int q = 0; q < QR; q++) {
        const float total = lane_groups_sum(rowSum[q]);
        const int row = row0 + 16 * q;
        if (row >= sg.rows)
            continue;
        float * to;
        float f = 1.f;
        if (sg.slot < 0) {
            const int t = divided(row, p.perDiv);
            to = static_cast<float *>(p.out) + (long long)(sg.s.start + t) * p.oT + (sg.head * p.per + row - t * p.per) * p.oH;
            f = total == 0.f ? 0.f : 1.f / total;
        }
        else {
            const long long at = (long long)sg.slot * TR + (row - sg.row0);
            to = p.acc + at * dh;
            if (g == 0) {
                p.stat[2 * at] = rowMax[q];
                p.stat[2 * at + 1] = total;
            }
        }
#pragma unroll
        for (int h = 0; h < NH; h++)
#pragma unroll
            for (int r = 0; r < 4; r += 4 / VC) {
                const int col = VC * (16 * h + 4 * g + r);
                if (col < dh) {
                    f32x4 o;
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        o[e] = accO[q][h][e % VC][r + e / VC] * f;
                    *reinterpret_cast<f32x4 *>(to + col) = o;
                }
            }
    }
}

}  // namespace ntsamd
