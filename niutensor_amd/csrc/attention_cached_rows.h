/*
 * Attention of new tokens over a cache on pages (ntsamd_attention_cached, ntsamd_attention_prefix;
 * include/ntsamd_cache.h):  out[t][h] = sum_j p_j v_j,  p = softmax_j(scale <q[t][h], k_j>),  j over the positions that t sees.
 *
 * A step of one token per sequence reads every key and value once and computes 4 R operations per element (R query
 * heads share a key head): bound by memory by far, so the plan is to keep loads in flight and to spread the keys evenly.
 *
 * A workgroup takes up to 16 QR query rows (tokens x the query heads of one key head) of one sequence and a range of
 * its keys; its four waves take units of UK keys (32 half, 16 float: 8 KB of k and 8 KB of v at 128 columns) in turn, each
 * with a running softmax of its own, and nothing is shared until the range is done. Both products run on MFMAs, transposed
 * (as in attention_f32.hip), so that the probabilities pass from accumulator to operand inside a lane:
 *   S^T = K Q^T   lane (m, g) = (l % 16, l / 16) feeds columns of key m and of query m, and receives the scores of query m
 *                 against keys 16 j + 4 g + r, r = 0..3;
 *   O^T = V^T P^T lane (m, g) feeds the probabilities it holds, and of V its keys in VC neighbouring columns, VC m ...: the
 *                 rows of V^T may stand for any columns, so MFMA c of a set takes column VC m + c, and a lane's
 *                 16-byte loads of VC columns of its keys are what the set needs. In half, where a lane feeds eight keys
 *                 of one column, the 8 x VC piece it loaded is transposed by byte permutes within the lane.
 * So k and v go from memory to registers, each element once, without LDS; the next unit is in flight while one is
 * computed, the page numbers of the one after it are looked up by the lanes, one key each, and handed round.
 * Addresses of positions that a range does not have, and of columns past dh, point at a row of zeros: nothing behind a
 * sequence's end is ever read, let alone multiplied.
 *
 * The four waves' results meet in LDS. Where a range is not all of a sequence's keys, the result is a partial one
 * (unnormalised row, maximum, sum), and a second kernel joins them in the order of the keys.
 *
 * 64 sequences of up to 8191 positions, 32 heads on 8 of 128 columns, half: 202 us and 5 for the join, 5.3 TB/s; one of 131072: 95 and 5,
 * 5.6 TB/s. One of 128, 8 heads of 64: 4.2 us replayed from a graph (a call through the host 5.3), of which the launch and four loads that
 * each need the one before are nearly all.
 */
#pragma once
#include "gemm_common.h"
#include "gemm_f16.h"       /* half_t */
#include "attention.h"
#include "attention_cached.h"

namespace ntsamd {

template <typename T, int DHM> struct Unit;
template <int DHM> struct Unit<half_t, DHM> {
    static constexpr int UK = cached_block_keys(true, DHM, 16), NJ = UK / 16;   /* keys, blocks of 16 of them */
    static constexpr int NT = DHM / 32;                 /* 16-byte pieces of a key row per lane */
    static constexpr int NV = 8;                        /* keys whose values a lane loads */
    static constexpr int VC = DHM / 16, NH = 1;         /* neighbouring columns of them, sets of such columns */
    typedef f16x8 KPiece;
    typedef half_t VPiece __attribute__((ext_vector_type(VC)));
};
template <int DHM> struct Unit<float, DHM> {
    static constexpr int UK = cached_block_keys(false, DHM, 16), NJ = UK / 16;
    static constexpr int NT = DHM / 16;
    static constexpr int NV = 4;
    static constexpr int VC = DHM % 64 == 0 ? 4 : 2, NH = DHM / 16 / VC;
    typedef f32x4 KPiece;
    typedef float VPiece __attribute__((ext_vector_type(VC)));
};

template <typename T, int DHM> struct UnitData {
    typename Unit<T, DHM>::KPiece k[Unit<T, DHM>::NJ][Unit<T, DHM>::NT];
    typename Unit<T, DHM>::VPiece v[Unit<T, DHM>::NV][Unit<T, DHM>::NH];
    unsigned there;                                     /* which of its keys exist */
};

/* NW: waves of a workgroup */
template <int DHM, int NW> struct CachedShared {
    float acc[NW][16][DHM + 4];
    float stat[NW][16][2];
    CachedScan scan;
};

/* ND columns from `col` on, those below dh, times f */
template <typename T, int ND>
__device__ __forceinline__ void store_columns(T * row, int col, int dh, const float (&x)[ND], float f)
{
    constexpr int MOST = 16 / (int)sizeof(T);                           /* dh is a multiple of it */
    constexpr int W = ND < MOST ? ND : (ND % MOST == 0 ? MOST : 2);
    typedef T vec __attribute__((ext_vector_type(W)));
#pragma unroll
    for (int at = 0; at < ND; at += W)
        if (col + at < dh) {
            vec v;
#pragma unroll
            for (int e = 0; e < W; e++)
                v[e] = (T)(x[at + e] * f);
            *reinterpret_cast<vec *>(row + col + at) = v;
        }
}

template <typename T, int DHM, int QR, int NW>
__device__ __forceinline__ void attend(const CachedParams & p, const Segment & sg, CachedShared<DHM, NW> & sh)
{
    typedef Unit<T, DHM> U;
    constexpr int ND = DHM / 16;
    constexpr unsigned ALL = U::UK == 32 ? 0xffffffffu : 0xffffu;
    const CacheParams & c = p.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m = lane & 15, g = lane >> 4;
    const int dh = c.dh;

    /* ---- loading a unit ---- */
    const int * table = c.table + (long long)sg.seq * c.tablePages;
    const int myKey = lane & (U::UK - 1);
    auto page_of = [&](int u) {
        const int key = sg.first + u * U::UK + myKey;
        return u < sg.u1 && key < sg.keys ? page_entry(key < p.common ? c.table : table, divided(key, c.pageSize)) : -1;
    };
    /* byte offsets of a lane's columns in a row. Columns past dh read the row's first: a key's meet zeros of q, a value's
       end in columns of the result that are not stored */
    int kCol[U::NT], vCol[U::NH];
#pragma unroll
    for (int t = 0; t < U::NT; t++)
        kCol[t] = 64 * t + 16 * g < dh * (int)sizeof(T) ? 64 * t + 16 * g : 0;
#pragma unroll
    for (int h = 0; h < U::NH; h++)
        vCol[h] = U::VC * (16 * h + m) < dh ? U::VC * (16 * h + m) * (int)sizeof(T) : 0;
    auto load = [&](int u, int page, UnitData<T, DHM> & d) {
        const KeyPlace at = key_place<T>(c, sg.head, sg.first + u * U::UK + myKey, page);
        d.there = (unsigned)__ballot(at.there) & ALL;
#pragma unroll
        for (int j = 0; j < U::NJ; j++) {
            const long long row = lane_of(at.k, 16 * j + m);
#pragma unroll
            for (int t = 0; t < U::NT; t++)
                d.k[j][t] = load_global<typename U::KPiece>(row + kCol[t]);
        }
#pragma unroll
        for (int e = 0; e < U::NV; e++) {
            const long long row = lane_of(at.v, 16 * (e >> 2) + 4 * g + (e & 3));
#pragma unroll
            for (int h = 0; h < U::NH; h++)
                d.v[e][h] = load_global<typename U::VPiece>(row + vCol[h]);
        }
    };

    /* One unit ahead, but for the widest tiles of the widest heads: their next unit would take the registers of a second
       workgroup on the CU, which hides more */
    constexpr bool AHEAD = QR == 1 || DHM < 128;
    UnitData<T, DHM> next;
    int u = sg.u0 + wave;
    int page = page_of(u);
    if (AHEAD) {
        if (u < sg.u1)
            load(u, page, next);
        page = page_of(u + NW);
    }

    /* ---- this lane's query rows: positions each sees, fragments ---- */
    int seen[QR];
    const int seenMin = rows_seen<QR, sizeof(sh.acc) / 4>(p, sg, sg.row0 + m, reinterpret_cast<int *>(&sh.acc[0][0][0]), seen);
    typename U::KPiece qf[QR][U::NT];
#pragma unroll
    for (int q = 0; q < QR; q++) {
        const int row = sg.row0 + 16 * q + m;
        const bool there = row < sg.rows;
        const int t = there ? divided(row, p.perDiv) : 0;
        const int h = sg.head * p.per + (there ? row - t * p.per : 0);
        const T * qr = static_cast<const T *>(p.q) + (long long)(sg.s.start + t) * p.qT + h * p.qH;
#pragma unroll
        for (int t4 = 0; t4 < U::NT; t4++) {
            constexpr int W = sizeof(typename U::KPiece) / sizeof(T);
            const int col = 4 * W * t4 + W * g;
            typename U::KPiece z = {};
            qf[q][t4] = there && col < dh ? *reinterpret_cast<const typename U::KPiece *>(qr + col) : z;
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

    for (; u < sg.u1; u += NW) {
        UnitData<T, DHM> d;
        if (AHEAD) {
            d = next;
            if (u + NW < sg.u1)
                load(u + NW, page, next);
            page = page_of(u + 2 * NW);
        }
        else {
            load(u, page, d);
            page = page_of(u + NW);
        }

        /* ---- S^T = K Q^T ---- */
        f32x4 s[QR][U::NJ];
#pragma unroll
        for (int q = 0; q < QR; q++)
#pragma unroll
            for (int j = 0; j < U::NJ; j++)
                s[q][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < U::NT; t++)
#pragma unroll
            for (int j = 0; j < U::NJ; j++)
#pragma unroll
                for (int q = 0; q < QR; q++) {
                    if constexpr (sizeof(T) == 2)
                        s[q][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(d.k[j][t], qf[q][t], s[q][j], 0, 0, 0);
                    else {
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            s[q][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(d.k[j][t][e], qf[q][t][e], s[q][j], 0, 0, 0);
                    }
                }

        const int key0 = sg.first + u * U::UK;
        const bool cut = d.there != ALL || key0 + U::UK > seenMin;
        /* The probabilities as the second product's operand. In half the sum of two: rounded to one alone they leave up to 2^-11 of each,
           as much again as the rounding of the result, and what the second costs is hidden where memory is waited for (64 sequences of
           up to 8191 positions, one of 131072: no change; one of 128 positions 4.1 -> 4.2 us; 32 rows of 32 sequences, heads of 64:
           51.3 -> 54.0) */
        T pr[QR][U::NJ][4], rest[QR][U::NJ][4];
#pragma unroll
        for (int q = 0; q < QR; q++) {
            if (cut) {
#pragma unroll
                for (int j = 0; j < U::NJ; j++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int at = 16 * j + 4 * g + r;
                        if (!((d.there >> at) & 1) || key0 + at >= seen[q])
                            s[q][j][r] = -INFINITY;
                    }
            }
            float mx = s[q][0][0];
#pragma unroll
            for (int j = 0; j < U::NJ; j++)
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
                for (int e = 0; e < ND; e++)
                    accO[q][e] *= corr;
            }
            const float shift = rowMax[q] == -INFINITY ? 0.f : rowMax[q];
#pragma unroll
            for (int j = 0; j < U::NJ; j++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float e = __builtin_amdgcn_exp2f(fmaf(s[q][j][r], scale2, -shift));
                    rowSum[q] += e;                     /* this lane's keys only: the lanes of a row meet at the end */
                    pr[q][j][r] = (T)e;
                    if constexpr (sizeof(T) == 2)
                        rest[q][j][r] = (T)(e - (float)pr[q][j][r]);
                }
        }

        /* ---- O^T += V^T P^T ---- */
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int v = 0; v < U::VC; v++) {
                f16x8 a;
#pragma unroll
                for (int e = 0; e < 8; e++)
                    a[e] = d.v[e][0][v];
#pragma unroll
                for (int q = 0; q < QR; q++) {
                    const f16x8 b = {pr[q][0][0], pr[q][0][1], pr[q][0][2], pr[q][0][3],
                                     pr[q][1][0], pr[q][1][1], pr[q][1][2], pr[q][1][3]};
                    const f16x8 r = {rest[q][0][0], rest[q][0][1], rest[q][0][2], rest[q][0][3],
                                     rest[q][1][0], rest[q][1][1], rest[q][1][2], rest[q][1][3]};
                    accO[q][v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, accO[q][v], 0, 0, 0);
                    accO[q][v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, r, accO[q][v], 0, 0, 0);
                }
            }
        }
        else {
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int h = 0; h < U::NH; h++)
#pragma unroll
                    for (int v = 0; v < U::VC; v++)
#pragma unroll
                        for (int q = 0; q < QR; q++)
                            accO[q][h * U::VC + v] =
                                __builtin_amdgcn_mfma_f32_16x16x4f32(d.v[e][h][v], pr[q][0][e], accO[q][h * U::VC + v], 0, 0, 0);
        }
    }

    /* ---- the waves' results, 16 rows at a time. Register r of MFMA v of set h holds column VC (16 h + 4 g + r) + v of
       the lane's row ---- */
#pragma unroll
    for (int q = 0; q < QR; q++) {
        const float sum = lane_groups_sum(rowSum[q]);
        if (g == 0) {
            sh.stat[wave][m][0] = rowMax[q];
            sh.stat[wave][m][1] = sum;
        }
#pragma unroll
        for (int h = 0; h < U::NH; h++)
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int v = 0; v < U::VC; v++)
                    sh.acc[wave][m][U::VC * (16 * h + 4 * g + r) + v] = accO[q][h * U::VC + v][r];
        __syncthreads();
        const int mine = tid >> 4, col = (tid & 15) * ND, row = sg.row0 + 16 * q + mine;
        if ((NW == 4 || tid < 256) && row < sg.rows) {
            float mx = sh.stat[0][mine][0];
#pragma unroll
            for (int w = 1; w < NW; w++)
                mx = fmaxf(mx, sh.stat[w][mine][0]);
            const float shift = mx == -INFINITY ? 0.f : mx;
            float total = 0.f, o[ND];
#pragma unroll
            for (int e = 0; e < ND; e++)
                o[e] = 0.f;
#pragma unroll
            for (int w = 0; w < NW; w++) {
                const float f = __builtin_amdgcn_exp2f(sh.stat[w][mine][0] - shift);
                total += f * sh.stat[w][mine][1];
#pragma unroll
                for (int e = 0; e < ND; e++)
                    o[e] += f * sh.acc[w][mine][col + e];
            }
            if (sg.slot < 0) {
                const int t = divided(row, p.perDiv);
                T * out = static_cast<T *>(p.out) + (long long)(sg.s.start + t) * p.oT + (sg.head * p.per + row - t * p.per) * p.oH;
                store_columns<T, ND>(out, col, dh, o, total == 0.f ? 0.f : 1.f / total);
            }
            else {
                const long long at = (long long)sg.slot * p.rows + (row - sg.row0);
                store_columns<float, ND>(p.acc + at * dh, col, dh, o, 1.f);
                if ((tid & 15) == 0) {
                    p.stat[2 * at] = mx;
                    p.stat[2 * at + 1] = total;
                }
            }
        }
        __syncthreads();
    }
}

/* CACHED_WHOLE, CACHED_PIECES: the segment of workgroup `id`; without rows where it has none */
template <int UK>
__device__ __forceinline__ Segment pair_segment(const CachedParams & p, CachedScan & sh, int id)
{
    int i, head, u0 = 0, u1 = 0x7fffffff, slot;
    if (p.mode == CACHED_PIECES) {
        const PiecePlan f = piece_plan<UK>(p, sh);
        long long before = 0;
        const int found = find_sequence(f.scan, id, before, sh, [&](int n) { return pieces_of<UK>(p, n, f.most); });
        i = max(found, 0);
        const int units = found < 0 ? 0 : units_of<UK>(p, cache_sequence(p.c, p.seq0 + i));
        const int pieces = (int)(((unsigned)units + f.most - 1) / (unsigned)f.most);
        /* the key heads of a piece side by side: their rows may be neighbours in memory */
        const int in = id - (int)before, piece = in / p.c.kvHeads;
        head = in - piece * p.c.kvHeads;
        u0 = piece * f.most;
        u1 = found < 0 ? -1 : u0 + f.most;
        /* slots of cut pairs are numbered through; behind a prefix the others have one each after those */
        const int pair = i * p.c.kvHeads + head;
        const int slot0 = pieces > 1 ? (int)(before >> 32) + head * pieces : (p.first > 0 ? 2 * p.groups + pair : -1);
        slot = slot0 < 0 ? -1 : slot0 + piece;
        if (found >= 0 && piece == 0 && threadIdx.x == 0) {
            p.slots[2 * pair] = slot0;
            p.slots[2 * pair + 1] = slot0 < 0 ? 0 : pieces;
        }
    }
    else {
        i = id / p.c.kvHeads;
        head = id - i * p.c.kvHeads;
        if (p.sorted) {
            sort_sequences(p, sh);
            i = sh.order[p.seqs - 1 - i];
        }
        slot = p.acc ? i * p.c.kvHeads + head : -1;
    }
    Segment sg;
    sg.seq = p.seq0 + i;
    sg.s = cache_sequence(p.c, sg.seq);
    sg.head = head;
    sg.row0 = 0;
    sg.rows = u1 < 0 ? 0 : sg.s.fresh * p.per;
    sg.keys = sg.s.length;
    sg.u0 = u0;
    sg.first = first_of(p, sg.s);
    sg.u1 = min(u1, (sg.s.length - sg.first + UK - 1) / UK);
    sg.slot = slot;
    return sg;
}

/* workgroup `id` of a CACHED_TILES launch, tiles of 16 QR rows, NW waves */
template <typename T, int DHM, int QR, int NW>
__device__ __forceinline__ void attend_tile_rows(const CachedParams & p, int id, CachedShared<DHM, NW> & sh)
{
    const Segment sg = uniform(tile_segment<16 * QR, Unit<T, DHM>::UK, NW>(p, sh.scan, id));
    if (sg.rows > 0)
        attend<T, DHM, QR, NW>(p, sg, sh);
}

/* workgroup `id` of a CACHED_WHOLE or CACHED_PIECES launch, NW waves (more than 4: CACHED_WHOLE only, scans take 256 threads) */
template <typename T, int DHM, int QR, int NW>
__device__ __forceinline__ void attend_pair(const CachedParams & p, int id, CachedShared<DHM, NW> & sh)
{
    const Segment sg = uniform(pair_segment<Unit<T, DHM>::UK>(p, sh.scan, id));
    if (sg.rows > 0)
        attend<T, DHM, QR, NW>(p, sg, sh);
}

}  // namespace ntsamd
