/*
 * Attention over a cache for few rows of a sequence, and float tiles: the kernels of attention_cached_rows.h on their own.
 */
#include "attention_cached_rows.h"

namespace ntsamd {

namespace {

template <typename T, int DHM, int QR>
__global__ void __launch_bounds__(256, 2)
attention_cached_kernel(const CachedParams p)
{
    __shared__ CachedShared sh;
    const int id = (int)blockIdx.x;
    const Segment sg = uniform(p.mode == CACHED_TILES ? tile_segment<16 * QR, Unit<T, DHM>::UK>(p, sh.scan, id)
                                                      : pair_segment<Unit<T, DHM>::UK>(p, sh.scan, id));
    if (sg.rows > 0)
        attend<T, DHM, QR>(p, sg, sh);
}

template <typename T, int DHM>
int launch_dhm(const CachedParams & p, int qr, int blocks, hipStream_t stream)
{
    const dim3 grid((unsigned)blocks), block(256);
    if (qr == 1)
        hipLaunchKernelGGL((attention_cached_kernel<T, DHM, 1>), grid, block, 0, stream, p);
    else
        hipLaunchKernelGGL((attention_cached_kernel<T, DHM, 2>), grid, block, 0, stream, p);
    return (int)hipGetLastError();
}

template <typename T>
int launch_type(const CachedParams & p, int qr, int blocks, hipStream_t stream)
{
    if (p.c.dh <= 32)
        return launch_dhm<T, 32>(p, qr, blocks, stream);
    if (p.c.dh <= 64)
        return launch_dhm<T, 64>(p, qr, blocks, stream);
    return launch_dhm<T, 128>(p, qr, blocks, stream);
}

}  // namespace

int launch_attention_cached(const CachedParams & p, bool half, int qr, int blocks, hipStream_t stream)
{
    return half ? launch_type<half_t>(p, qr, blocks, stream) : launch_type<float>(p, qr, blocks, stream);
}

}  // namespace ntsamd
