/*
 * Attention over a cache on pages for many query rows in half: pieces of text against what is in the cache, and the
 * queries of a whole batch against a prefix they share (ntsamd_attention_cached, ntsamd_attention_prefix). The stages and the fetch are
 * shared with float tiles of 64 rows (attention_cached_tiles_f32.h); the few rows of a decoding step, and tiles of 16 or 32 rows, are
 * attention_cached_rows.h.
 *
 * Bound by the matrix instructions and what feeds them, so keys and values go through LDS once for all rows of a
 * workgroup, on the plan of attention_f16.hip: 64 QR rows (tokens x the query heads that share a key head) of a tile, 16 QR
 * per wave; blocks of 64 keys; both products transposed, so that probabilities pass from accumulator to operand inside
 * a lane; values read back by transposing LDS reads. What is different: lane l of every wave looks
 * up the page of key l of a block, one block ahead, and hands its address to the lanes that fetch the row; rows go from memory
 * to LDS without registers in between, a block ahead, two stages, one barrier a block; the sums of the probabilities are one
 * more product, with a row of ones (of the rounded probabilities then, as the results are), since the vector ALU's exponentials and
 * conversions are what a wave spends most of its time on. Rows of a
 * tile see different numbers of keys; only the blocks in which some row's last key falls, or which have an absent page, take the
 * comparisons. Fetches of keys that a tile does not have read a row of zeros.
 *
 * A wave's block of 64 keys, 32 rows and 128 columns is 1090 cycles of MFMAs and about as many of vector instructions, 512 of them
 * exponentials. 4 pieces of text of 257 to 1024 tokens in sequences of 1500 to 4096, 32 heads on 8 of 128: 121 us, 807 TFLOP/s with
 * the last round of workgroups half empty; 8 times 1024 on 4096, not causal: 592 us, 928 TFLOP/s (822, 753, 530 with heads of 96, 64, 32;
 * a large product reaches 1207); causal 538 us, 894.
 */
#pragma once
#include "gemm_common.h"
#include "gemm_f16_direct.h"        /* half_t, lds_read_tr16, wait_vmcnt, wait_lgkmcnt0 */
#include "attention.h"
#include "attention_cached.h"

namespace ntsamd {

/* Two stages of a block of keys and values: KB keys, 32 KB at most, so that two workgroups share a CU. Rows are those of DHM columns,
   without padding (they are written 16 bytes a lane, one lane after the other); which 16-byte piece of a row stands where is
   swizzled by the row instead, so that 16 rows read at one column, and in half the pairs of pieces that a transposing read takes of
   8 rows, stand on all banks once. That is so for lanes served in order; the counters still show conflicts, a third of the cycles
   in which half tiles read LDS. */
template <typename T, int DHM> struct CachedTilesShared {
    static constexpr int KB = cached_block_keys(sizeof(T) == 2, DHM, 64);
    static constexpr int PIECES = DHM * (int)sizeof(T) / 16, ROW = DHM * (int)sizeof(T), BLOCK = KB * ROW;
    __attribute__((aligned(1024))) char k[2][BLOCK];
    __attribute__((aligned(1024))) char v[2][BLOCK];
    CachedScan scan;
    static __device__ __forceinline__ int swizzle(int row)
    {
        /* rows that share the 256 bytes of a round of banks take the same */
        const int k = PIECES >= 16 ? row & 15 : (row & 15) * PIECES / 16;
        return sizeof(T) == 4 ? k : ((k & (PIECES / 2 - 1)) << 1) | (k / (PIECES / 2));
    }
};

/* global memory -> LDS, 16 bytes per lane: lane l's data lands at lds + 16 l (the same for the whole wave). Counted by vmcnt, which
   the caller waits for: the compiler does not see a load. An instruction that reads M0 for LDS must not follow its write at once. */
__device__ __forceinline__ void lds_from_global16(unsigned lds, long long address)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :
                 : "s"(lds), "v"(address)
                 : "memory");
}

/* the same from an address that the whole wave shares and an offset per lane. A memory instruction must not read a scalar register
   within five cycles of the vector ALU writing it, which the compiler sees to only for its own */
__device__ __forceinline__ void lds_from_global16(unsigned lds, long long address, unsigned offset)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(lds), "v"(offset), "s"(address)
                 : "memory");
}

/* What fetches a tile's blocks: lane l of every wave looks after key l of a block, and tells the lanes that fetch a piece of its row
   where it stands. Where all keys of a block are there, the rows that a wave fetches with one load stand behind one another on a
   page, if that has a multiple of their number: they share an address, and the lanes' offsets are the same for every block. With
   pages of a multiple of 16 positions all rows of a wave do (4 pieces of text of 257 to 1024 tokens in sequences of 1500 to 4096, 32
   heads on 8 of 128, half, pages of 64: 133 us with an address per row, 121 so). */
template <typename T, int DHM> struct TileFetch {
    typedef CachedTilesShared<T, DHM> Shared;
    static constexpr int KB = Shared::KB, PIECES = Shared::PIECES;
    static constexpr int ROWS = 64 / PIECES;            /* rows of a block that a wave fetches at a time */
    static constexpr int LOADS = KB / (4 * ROWS);
    const CachedParams & p;
    const Segment & sg;
    const int * table;
    int lane, first, fetch;                 /* the wave fetches rows from `first` on; this lane fetches a piece of each of the rows `fetch` + ROWS s */
    int col[LOADS];                         /* columns past dh: the row's first, which meet zeros of q or are not stored */
    unsigned kLds, vLds;
    unsigned kOff[LOADS], vOff[LOADS];      /* from the first of the wave's rows */
    unsigned long long there;               /* which keys of the block being fetched exist */

    __device__ __forceinline__ TileFetch(const CachedParams & params, const Segment & segment, Shared & sh, int wave, int l)
        : p(params), sg(segment), table(params.c.table + (long long)segment.seq * params.c.tablePages), lane(l),
          first(wave * (LOADS * ROWS)), fetch(first + l / PIECES), there(0)
    {
#pragma unroll
        for (int s = 0; s < LOADS; s++) {
            const int at = 16 * ((lane % PIECES) ^ Shared::swizzle(fetch + ROWS * s));
            col[s] = at < (int)sizeof(T) * p.c.dh ? at : 0;
            kOff[s] = (unsigned)(lane / PIECES + ROWS * s) * (unsigned)p.c.kR * (unsigned)sizeof(T) + col[s];
            vOff[s] = (unsigned)(lane / PIECES + ROWS * s) * (unsigned)p.c.vR * (unsigned)sizeof(T) + col[s];
        }
        kLds = (unsigned)(size_t)((__attribute__((address_space(3))) char *)sh.k[0]) + wave * (LOADS * 1024);
        vLds = (unsigned)(size_t)((__attribute__((address_space(3))) char *)sh.v[0]) + wave * (LOADS * 1024);
    }
    /* the page of the lane's key of block u */
    __device__ __forceinline__ int page_of(int u) const
    {
        const int key = u * KB + lane;
        return u < sg.u1 && key < sg.keys && (KB == 64 || lane < KB) ? page_entry(key < p.common ? p.c.table : table, divided(key, p.c.pageSize)) : -1;
    }
    __device__ __forceinline__ void block(int u, int page)
    {
        const KeyPlace at = key_place<T>(p.c, sg.head, u * KB + lane, page);
        const unsigned stage = ((u - sg.u0) & 1) * Shared::BLOCK;
        there = __ballot(at.there);
        if (p.runs >= ROWS && there == (KB == 64 ? ~0ull : (1ull << (KB & 63)) - 1)) {
            if (p.runs >= LOADS * ROWS) {
                const long long k = lane_of_all(at.k, first), v = lane_of_all(at.v, first);
#pragma unroll
                for (int s = 0; s < LOADS; s++)
                    lds_from_global16(kLds + stage + s * 1024, k, kOff[s]);
#pragma unroll
                for (int s = 0; s < LOADS; s++)
                    lds_from_global16(vLds + stage + s * 1024, v, vOff[s]);
                return;
            }
            const unsigned kStep = ROWS * (unsigned)p.c.kR * (unsigned)sizeof(T), vStep = ROWS * (unsigned)p.c.vR * (unsigned)sizeof(T);
#pragma unroll
            for (int s = 0; s < LOADS; s++)
                lds_from_global16(kLds + stage + s * 1024, lane_of_all(at.k, first + ROWS * s), kOff[s] - s * kStep);
#pragma unroll
            for (int s = 0; s < LOADS; s++)
                lds_from_global16(vLds + stage + s * 1024, lane_of_all(at.v, first + ROWS * s), vOff[s] - s * vStep);
            return;
        }
#pragma unroll
        for (int s = 0; s < LOADS; s++)
            lds_from_global16(kLds + stage + s * 1024, lane_of(at.k, fetch + ROWS * s) + col[s]);
#pragma unroll
        for (int s = 0; s < LOADS; s++)
            lds_from_global16(vLds + stage + s * 1024, lane_of(at.v, fetch + ROWS * s) + col[s]);
    }
    /* the block being fetched has landed, for every wave, and nobody reads the other stage any more */
    __device__ __forceinline__ void landed() const
    {
        __builtin_amdgcn_sched_barrier(0);
        wait_vmcnt<0>();
        wait_lgkmcnt0();
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    }
};

/* Hides from a row's scores of a block those of keys that do not exist and of keys past the `left` ones that the row sees. Register r
   of part j is key 16 j + 4 g + r. Nothing of it is to be computed where it is not called (the compiler would keep a mask for every
   register for the whole loop). */
template <int NJ>
__device__ __forceinline__ void hide_scores(f32x4 (&s)[NJ], unsigned long long exist, int left, int g)
{
    const unsigned long long mine = (exist & (left >= 64 ? ~0ull : (1ull << max(left, 0)) - 1)) >> (4 * g);
    unsigned part[2] = {(unsigned)mine, (unsigned)(mine >> 32)};
    asm volatile("" : "+v"(part[0]), "+v"(part[1]));
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (!((part[j >> 1] >> (16 * (j & 1) + r)) & 1))
                s[j][r] = -INFINITY;
}

/* workgroup `id` of a CACHED_TILES launch over half tensors, tiles of 64 QR rows. DHC: columns computed with, at least dh (rows of 80
   or 96 columns stand in LDS as rows of 128) */
template <int DHM, int DHC, int QR>
__device__ __forceinline__ void attend_tile(const CachedParams & p, int id, CachedTilesShared<half_t, DHM> & sh)
{
    typedef CachedTilesShared<half_t, DHM> Shared;
    constexpr int KB = CACHED_TILE_KEYS, TR = 64 * QR;
    constexpr int NT = DHC / 32, ND = DHC / 16, NJ = KB / 16;

    const int tid = threadIdx.x;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m = lane & 15, g = lane >> 4;
    const int dh = p.c.dh;

    const Segment sg = uniform(tile_segment<TR, KB>(p, sh.scan, id));
    if (sg.rows == 0)
        return;
    TileFetch<half_t, DHM> from(p, sg, sh, wave, lane);
    /* the first block is on its way before anything is asked about the rows */
    if (sg.u0 < sg.u1)
        from.block(sg.u0, from.page_of(sg.u0));
    int page = from.page_of(sg.u0 + 1);

    const int row0 = sg.row0 + wave * (16 * QR) + m;
    int seen[QR];
    const int seenMin = rows_seen<QR, Shared::BLOCK / 4>(p, sg, row0, reinterpret_cast<int *>(sh.k[1]), seen);

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

    f32x4 accO[QR][ND], accL[QR];            /* accL: the sum of the row's probabilities, in every register */
    float rowMax[QR];
#pragma unroll
    for (int q = 0; q < QR; q++) {
#pragma unroll
        for (int d = 0; d < ND; d++)
            accO[q][d] = f32x4{0.f, 0.f, 0.f, 0.f};
        accL[q] = f32x4{0.f, 0.f, 0.f, 0.f};
        rowMax[q] = -INFINITY;
    }
    const float scale2 = score_scale(p);
    const half_t one = (half_t)1.f;
    const f16x8 ones = {one, one, one, one, one, one, one, one};
    /* where this lane reads keys (row m of a 16-key block, piece 4 t + g) and points for the transposing reads of values (row
       4 g + m / 4, columns 16 d + 4 (m % 4) .. + 3) */
    int kAt[NT], vAt[ND];
#pragma unroll
    for (int t = 0; t < NT; t++)
        kAt[t] = m * (2 * DHM) + 16 * ((4 * t + g) ^ Shared::swizzle(m));
    const int trRow = 4 * g + (m >> 2);
#pragma unroll
    for (int d = 0; d < ND; d++)
        vAt[d] = trRow * (2 * DHM) + 16 * ((2 * d + ((m & 3) >> 1)) ^ Shared::swizzle(trRow)) + 8 * (m & 1);

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
                const f16x8 kf = *reinterpret_cast<const f16x8 *>(&Ks[kAt[t] + 16 * j * (2 * DHM)]);
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
            if (cut)
                hide_scores(accS[q], exist, seen[q] - key0, g);
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
                accL[q] *= corr;
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
                for (int r = 0; r < 4; r++)
                    pf[q][j][r] = (half_t)__builtin_amdgcn_exp2f(fmaf(accS[q][j][r], scale2, -shift));
        }

        /* The probabilities are rounded to half, which leaves up to 2^-11 of each. The sum of two halves, as the few-rows kernel takes
           them, would double this product, which bounds the kernel: pieces of text 121 -> 160 us, 8 times 1024 on 4096 525 -> 681 (heads
           of 64: 329 -> 447). Their sum is that of the rounded ones, so that a probability's error is in numerator and denominator. */
        /* ---- O^T += V^T P^T, 32 keys per MFMA: its k index 8 g + e stands for key 4 g + e of the first 16-key block of a
           pair for e < 4 and for key 4 g + e - 4 of the second for e >= 4 ---- */
#pragma unroll
        for (int j = 0; j < NJ; j += 2) {
#pragma unroll
            for (int q = 0; q < QR; q++) {
                const f16x8 pp = __builtin_shufflevector(pf[q][j], pf[q][j + 1], 0, 1, 2, 3, 4, 5, 6, 7);
                accL[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pp, accL[q], 0, 0, 0);
            }
#pragma unroll
            for (int d = 0; d < ND; d++) {
                const f16x4 lo = lds_read_tr16(reinterpret_cast<const half_t *>(&Vs[vAt[d] + 16 * j * (2 * DHM)]));
                const f16x4 hi = lds_read_tr16(reinterpret_cast<const half_t *>(&Vs[vAt[d] + 16 * (j + 1) * (2 * DHM)]));
                const f16x8 vf = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                for (int q = 0; q < QR; q++) {
                    const f16x8 pp = __builtin_shufflevector(pf[q][j], pf[q][j + 1], 0, 1, 2, 3, 4, 5, 6, 7);
                    accO[q][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pp, accO[q][d], 0, 0, 0);
                }
            }
        }
    }

    /* ---- register r of block d is column 16 d + 4 g + r of the lane's row ---- */
#pragma unroll
    for (int q = 0; q < QR; q++) {
        const float total = accL[q][0];
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
