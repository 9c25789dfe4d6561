/*
 * Attention behind a shared prefix (ntsamd_attention_prefix): in one launch, workgroups that multiply the queries of all
 * sequences with the prefix, as tiles of one matrix, and workgroups that take each sequence's own keys. The first
 * wait on matrix instructions, the second on memory; taken in turn, eight of one kind and eight of the other (a workgroup
 * for each XCD), a CU has both. attention_join_kernel puts their partial results together.
 * 64 sequences of 8193 to 8704 positions behind a prefix of 8192, 8 key heads of 128, four query heads to each, half: 36 us and 6 us for
 * the join by the profiler, 41 us a call (28 us, 23 us and the join in launches of their own); the keys and values alone take 20 us at 5.1 TB/s.
 * What is left is the start of the workgroups, the blocks' first fetches, which nothing hides, and the partial results of the prefix's
 * pieces (17 MB written and read). Sequence by sequence, without the prefix read once, the same call takes 163 us.
 */
#include "attention_cached_rows.h"
#include "attention_cached_tiles.h"
#include "attention_cached_tiles_f32.h"

namespace ntsamd {

namespace {

/* TILE: rows of a tile of the prefix (16, 32 and 64 float, 64 and 128 half); QR: blocks of 16 rows of a sequence's own */
template <typename T, int DHM, int TILE, int QR>
__global__ void __launch_bounds__(256, 2)
attention_prefix_kernel(const CachedParams pre, const CachedParams own, int preBlocks, int ownBlocks)
{
    __shared__ union Shared {
        CachedShared<DHM, 4> rows;
        CachedTilesShared<T, DHM == 96 ? 128 : DHM> tiles;
        __device__ Shared() {}
    } sh;
    const int id = (int)blockIdx.x, both = 2 * (min(preBlocks, ownBlocks) & ~7);
    bool first;
    int at;
    if (id < both) {
        first = ((id >> 3) & 1) == 0;
        at = (id >> 4) * 8 + (id & 7);
    }
    else {
        at = id - both / 2;
        first = at < preBlocks;
        if (!first)
            at -= preBlocks - both / 2;
    }
    if (first) {
        if constexpr (sizeof(T) == 2)
            attend_tile<DHM, DHM, TILE / 64>(pre, at, sh.tiles);
        else if constexpr (TILE == 64)
            attend_tile_f32<DHM == 96 ? 128 : DHM, DHM>(pre, at, sh.tiles);
        else
            attend_tile_rows<T, DHM, TILE / 16, 4>(pre, at, sh.rows);
    }
    else
        attend_pair<T, DHM, QR, 4>(own, at, sh.rows);
}

template <typename T, int DHM, int TILE>
int launch_tile(const CachedParams & pre, const CachedParams & own, int qr, int preBlocks, int ownBlocks, hipStream_t stream)
{
    const dim3 grid((unsigned)(preBlocks + ownBlocks)), block(256);
    if (qr == 1)
        hipLaunchKernelGGL((attention_prefix_kernel<T, DHM, TILE, 1>), grid, block, 0, stream, pre, own, preBlocks, ownBlocks);
    else
        hipLaunchKernelGGL((attention_prefix_kernel<T, DHM, TILE, 2>), grid, block, 0, stream, pre, own, preBlocks, ownBlocks);
    return (int)hipGetLastError();
}

template <int DHM>
int launch_dhm(const CachedParams & pre, const CachedParams & own, bool half, int tile, int qr, int preBlocks, int ownBlocks,
               hipStream_t stream)
{
    if constexpr (DHM != 96)
        if (half)
            return tile <= 64 ? launch_tile<half_t, DHM, 64>(pre, own, qr, preBlocks, ownBlocks, stream)
                              : launch_tile<half_t, DHM, 128>(pre, own, qr, preBlocks, ownBlocks, stream);
    if (tile > 32)
        return launch_tile<float, DHM, 64>(pre, own, qr, preBlocks, ownBlocks, stream);
    return tile <= 16 ? launch_tile<float, DHM, 16>(pre, own, qr, preBlocks, ownBlocks, stream)
                      : launch_tile<float, DHM, 32>(pre, own, qr, preBlocks, ownBlocks, stream);
}

}  // namespace

int launch_attention_prefix(const CachedParams & pre, const CachedParams & own, bool half, int tile, int qr, int preBlocks,
                            int ownBlocks, hipStream_t stream)
{
    if (pre.c.dh <= 32)
        return launch_dhm<32>(pre, own, half, tile, qr, preBlocks, ownBlocks, stream);
    if (pre.c.dh <= 64)
        return launch_dhm<64>(pre, own, half, tile, qr, preBlocks, ownBlocks, stream);
    if (pre.c.dh <= 96 && !half)
        return launch_dhm<96>(pre, own, half, tile, qr, preBlocks, ownBlocks, stream);
    return launch_dhm<128>(pre, own, half, tile, qr, preBlocks, ownBlocks, stream);
}

}  // namespace ntsamd
