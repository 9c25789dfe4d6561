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

/* CACHED_TILES, tiles of 16 or 32 rows (more rows: attention_cached_tiles.hip). NW: 4 waves; in half 8, for calls whose workgroups all
   run at once. Float has the form of 4 alone, which wide heads do better with (1024 keys of 128 columns: 31 us, 35 with 8) and narrow ones worse
   (of 32: 16.4 and 14.2). */
template <typename T, int DHM, int QR, int NW>
__global__ void __launch_bounds__(64 * NW, NW == 8 && DHM <= 64 ? 4 : 2)
attention_cached_tile_kernel(const CachedParams p)
{
    __shared__ CachedShared<DHM, NW> sh;
    attend_tile_rows<T, DHM, QR, NW>(p, (int)blockIdx.x, sh);
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

template <typename T, int DHM>
int launch_tile(const CachedParams & p, int tile, int blocks, hipStream_t stream)
{
    if constexpr (sizeof(T) == 2)
        hipLaunchKernelGGL((attention_cached_tile_kernel<T, DHM, 1, 8>), dim3((unsigned)blocks), dim3(512), 0, stream, p);
    else if (tile == 16)
        hipLaunchKernelGGL((attention_cached_tile_kernel<T, DHM, 1, 4>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL((attention_cached_tile_kernel<T, DHM, 2, 4>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
    return (int)hipGetLastError();
}

template <typename T>
int launch_tile_type(const CachedParams & p, int tile, int blocks, hipStream_t stream)
{
    if (p.c.dh <= 32)
        return launch_tile<T, 32>(p, tile, blocks, stream);
    if (p.c.dh <= 64)
        return launch_tile<T, 64>(p, tile, blocks, stream);
    if constexpr (sizeof(T) == 4)
        if (p.c.dh <= 96)
            return launch_tile<T, 96>(p, tile, blocks, stream);
    return launch_tile<T, 128>(p, tile, blocks, stream);
}

}  // namespace

int launch_attention_pairs(const CachedParams & p, bool half, int tile, bool wide, int blocks, hipStream_t stream)
{
    return half ? launch_type<half_t>(p, tile, wide, blocks, stream) : launch_type<float>(p, tile, wide, blocks, stream);
}

int launch_attention_tile_rows(const CachedParams & p, bool half, int tile, int blocks, hipStream_t stream)
{
    return half ? launch_tile_type<half_t>(p, tile, blocks, stream) : launch_tile_type<float>(p, tile, blocks, stream);
}

}  // namespace ntsamd
