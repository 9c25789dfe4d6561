/*
 * Attention over a cache for many rows of a sequence, half: the tiles of attention_cached_tiles.h on their own.
 */
#include "attention_cached_tiles.h"

namespace ntsamd {

namespace {

template <int DHM, int QR>
__global__ void __launch_bounds__(256, 2)
attention_cached_tiles_kernel(const CachedParams p)
{
    __shared__ CachedTilesShared<DHM> sh;
    attend_tile<DHM, QR>(p, (int)blockIdx.x, sh);
}

template <int DHM>
int launch_dhm(const CachedParams & p, int qr, int blocks, hipStream_t stream)
{
    if (qr == 1)
        hipLaunchKernelGGL((attention_cached_tiles_kernel<DHM, 1>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL((attention_cached_tiles_kernel<DHM, 2>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
    return (int)hipGetLastError();
}

}  // namespace

int launch_attention_tiles_f16(const CachedParams & p, int tile, int blocks, hipStream_t stream)
{
    if (p.c.dh <= 32)
        return launch_dhm<32>(p, tile / 64, blocks, stream);
    if (p.c.dh <= 64)
        return launch_dhm<64>(p, tile / 64, blocks, stream);
    return launch_dhm<128>(p, tile / 64, blocks, stream);
}

}  // namespace ntsamd
