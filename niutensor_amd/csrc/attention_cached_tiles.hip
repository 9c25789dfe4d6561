/*
 * Attention over a cache for many rows of a sequence: the tiles of attention_cached_tiles.h and attention_cached_tiles_f32.h on
 * their own.
 */
#include "attention_cached_tiles.h"
#include "attention_cached_tiles_f32.h"

namespace ntsamd {

namespace {

template <typename T, int DHM, int DHC, int QR>
__global__ void __launch_bounds__(256, 2)
attention_cached_tiles_kernel(const CachedParams p)
{
    __shared__ CachedTilesShared<T, DHM> sh;
    if constexpr (sizeof(T) == 2)
        attend_tile<DHM, DHC, QR>(p, (int)blockIdx.x, sh);
    else
        attend_tile_f32<DHM, DHC>(p, (int)blockIdx.x, sh);
}

template <typename T, int DHM, int DHC>
int launch_dhm(const CachedParams & p, int qr, int blocks, hipStream_t stream)
{
    if constexpr (sizeof(T) == 2)
        if (qr == 2) {
            hipLaunchKernelGGL((attention_cached_tiles_kernel<T, DHM, DHC, 2>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
            return (int)hipGetLastError();
        }
    hipLaunchKernelGGL((attention_cached_tiles_kernel<T, DHM, DHC, 1>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
    return (int)hipGetLastError();
}

template <typename T>
int launch_type(const CachedParams & p, int qr, int blocks, hipStream_t stream)
{
    if (p.c.dh <= 32)
        return launch_dhm<T, 32, 32>(p, qr, blocks, stream);
    if (p.c.dh <= 64)
        return launch_dhm<T, 64, 64>(p, qr, blocks, stream);
    if (p.c.dh <= 96)
        return launch_dhm<T, 128, 96>(p, qr, blocks, stream);
    return launch_dhm<T, 128, 128>(p, qr, blocks, stream);
}

}  // namespace

int launch_attention_tiles(const CachedParams & p, bool half, int tile, int blocks, hipStream_t stream)
{
    return half ? launch_type<half_t>(p, tile / 64, blocks, stream) : launch_type<float>(p, tile / 64, blocks, stream);
}

}  // namespace ntsamd
