/*
 * Attention over a cache for few rows of a sequence, and float tiles: attention_cached_rows.h on its own.
 */
#include "attention_cached_rows.h"

namespace ntsamd {

namespace {

/* CACHED_WHOLE, CACHED_PIECES. NW: 4 waves, or, for CACHED_WHOLE of up to 16 rows, as many as a CU runs: 16, or 8 with heads of more
   than 64 columns, which need more than 128 registers */
template <int DHM> constexpr int WIDE = DHM > 64 ? 8 : 16;

template <typename T, int DHM, int QR, int NW>
__global__ void __launch_bounds__(64 * NW, NW == 16 ? 4 : 2)
attention_cached_kernel(const CachedParams p)
{
    __shared__ CachedShared<DHM, NW> sh;
    attend_pair<T, DHM, QR, NW>(p, (int)blockIdx.x, sh);
}

/* CACHED_TILES, float tiles of 16 or 32 rows (more rows, and half: attention_cached_tiles.hip) */
template <int DHM, int QR>
__global__ void __launch_bounds__(256, 2)
attention_cached_tile_kernel(const CachedParams p)
{
    __shared__ CachedShared<DHM, 4> sh;
    attend_tile_rows<float, DHM, QR>(p, (int)blockIdx.x, sh);
}

template <typename T, int DHM>
int launch_pairs(const CachedParams & p, int tile, bool wide, int blocks, hipStream_t stream)
{
    const dim3 grid((unsigned)blocks);
    if (wide)
        hipLaunchKernelGGL((attention_cached_kernel<T, DHM, 1, WIDE<DHM>>), grid, dim3(64 * WIDE<DHM>), 0, stream, p);
    else if (tile == 16)
        hipLaunchKernelGGL((attention_cached_kernel<T, DHM, 1, 4>), grid, dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL((attention_cached_kernel<T, DHM, 2, 4>), grid, dim3(256), 0, stream, p);
    return (int)hipGetLastError();
}

template <typename T>
int launch_type(const CachedParams & p, int tile, bool wide, int blocks, hipStream_t stream)
{
    if (p.c.dh <= 32)
        return launch_pairs<T, 32>(p, tile, wide, blocks, stream);
    if (p.c.dh <= 64)
        return launch_pairs<T, 64>(p, tile, wide, blocks, stream);
    if constexpr (sizeof(T) == 4)
        if (p.c.dh <= 96)
            return launch_pairs<T, 96>(p, tile, wide, blocks, stream);
    return launch_pairs<T, 128>(p, tile, wide, blocks, stream);
}

template <int DHM>
int launch_tile(const CachedParams & p, int tile, int blocks, hipStream_t stream)
{
    if (tile == 16)
        hipLaunchKernelGGL((attention_cached_tile_kernel<DHM, 1>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL((attention_cached_tile_kernel<DHM, 2>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
    return (int)hipGetLastError();
}

}  // namespace

int launch_attention_pairs(const CachedParams & p, bool half, int tile, bool wide, int blocks, hipStream_t stream)
{
    return half ? launch_type<half_t>(p, tile, wide, blocks, stream) : launch_type<float>(p, tile, wide, blocks, stream);
}

int launch_attention_tile_rows(const CachedParams & p, int tile, int blocks, hipStream_t stream)
{
    if (p.c.dh <= 32)
        return launch_tile<32>(p, tile, blocks, stream);
    if (p.c.dh <= 64)
        return launch_tile<64>(p, tile, blocks, stream);
    if (p.c.dh <= 96)
        return launch_tile<96>(p, tile, blocks, stream);
    return launch_tile<128>(p, tile, blocks, stream);
}

}  // namespace ntsamd
