/*
 * New keys and values to their places in a cache on pages, keys and queries turned by the angle of their position
 * on the way (ntsamd_cache_append, include/ntsamd_cache.h):
 *   (x, y) -> (x c - y s, y c + x s),  (c, s) = rotation[position][pair of columns],
 * in fp32, rounded once to the cache's type.
 *
 * Bound by memory: every new row is read once and written once, and one row of the rotation per token serves all
 * heads. A token's work is cut into items: 16 bytes of a row that is copied, twice 16 bytes where column j is turned
 * together with column j + rotated / 2 (both pieces by one lane, so that q may be turned in place). A wave takes 64, 128 or
 * 256 items of one token: it finds the token's sequence once, by counting the starts that are not behind the token,
 * 64 to a load (a binary search would chain a load per step in front of the two it cannot do without: the page number
 * and the row itself).
 * Rows that are not 16-byte aligned and numbers of turned columns that are no whole 16-byte pieces take items of one
 * column or pair instead.
 * 8 prompts of 513 to 2048 tokens, 32 heads on 8 of 128 columns, half: 45 us, 5.1 TB/s read and written. One token: 3.1 us, a launch and
 * the three loads; 64 sequences of one token: 3.4; both replayed from a graph, calls of them one after the other take the host 6.
 */
#include "gemm_common.h"
#include "gemm_f16.h"       /* half_t */
#include "cache.h"

namespace ntsamd {

namespace {

/* N consecutive columns as floats */
template <typename T, int N> struct Columns {
    typedef T vec __attribute__((ext_vector_type(N)));
    static __device__ __forceinline__ void load(const T * p, float (&x)[N])
    {
        const vec v = *reinterpret_cast<const vec *>(p);
#pragma unroll
        for (int e = 0; e < N; e++)
            x[e] = (float)v[e];
    }
    static __device__ __forceinline__ void store(T * p, const float (&x)[N])
    {
        vec v;
#pragma unroll
        for (int e = 0; e < N; e++)
            v[e] = (T)x[e];
        *reinterpret_cast<vec *>(p) = v;
    }
    static __device__ __forceinline__ void copy(const T * s, T * t) { *reinterpret_cast<vec *>(t) = *reinterpret_cast<const vec *>(s); }
};
template <typename T> struct Columns<T, 1> {
    static __device__ __forceinline__ void load(const T * p, float (&x)[1]) { x[0] = (float)p[0]; }
    static __device__ __forceinline__ void store(T * p, const float (&x)[1]) { p[0] = (T)x[0]; }
    static __device__ __forceinline__ void copy(const T * s, T * t) { t[0] = s[0]; }
};

/* one item of a row that is turned: pieces 0 .. turned - 1 are turned, the others copied. N = 1: pieces are single columns */
template <typename T, int N>
__device__ __forceinline__ void turned_item(const T * s, T * t, int piece, int turned, const AppendParams & p, const float * cs)
{
    const int half = p.rotated / 2;
    if (piece >= turned) {
        const int c = p.rotated + (piece - turned) * N;
        if (s != t)
            Columns<T, N>::copy(s + c, t + c);
    }
    else if (p.pairing == 0) {
        const int c = piece * N;
        float x[N], y[N], u[N], w[N];
        Columns<T, N>::load(s + c, x);
        Columns<T, N>::load(s + c + half, y);
#pragma unroll
        for (int e = 0; e < N; e++) {
            const float co = cs[2 * (c + e)], si = cs[2 * (c + e) + 1];
            u[e] = x[e] * co - y[e] * si;
            w[e] = y[e] * co + x[e] * si;
        }
        Columns<T, N>::store(t + c, u);
        Columns<T, N>::store(t + c + half, w);
    }
    else if constexpr (N == 1) {                        /* a piece is a pair of neighbours */
        const int c = 2 * piece;
        const float x = (float)s[c], y = (float)s[c + 1], co = cs[c], si = cs[c + 1];
        t[c] = (T)(x * co - y * si);
        t[c + 1] = (T)(y * co + x * si);
    }
    else {
        const int c = piece * N;
        float x[N], u[N];
        Columns<T, N>::load(s + c, x);
#pragma unroll
        for (int e = 0; e < N; e += 2) {
            const float co = cs[c + e], si = cs[c + e + 1];
            u[e] = x[e] * co - x[e + 1] * si;
            u[e + 1] = x[e + 1] * co + x[e] * si;
        }
        Columns<T, N>::store(t + c, u);
    }
}

/* pieces of a row that are turned (turned_item) */
template <int N>
__host__ __device__ __forceinline__ int turned_pieces(const AppendParams & p)
{
    if (!p.rotation)
        return 0;
    return p.pairing == 0 || N == 1 ? p.rotated / 2 / N : p.rotated / N;
}

template <typename T, int N>
__global__ void __launch_bounds__(256)
cache_append_kernel(const AppendParams p)
{
    const CacheParams & c = p.c;
    const int lane = threadIdx.x & 63;
    const int wave = (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int at = wave / p.waves, part = wave - at * p.waves;
    if (at >= c.tokens - p.token0)
        return;
    const int tok = p.token0 + at;
    /* the token's sequence: the last one that starts at or before it */
    int seq, place;
    if (c.starts) {
        int before = 0;
        for (int i = 0; i <= c.sequences; i += 64) {
            const int x = i + lane <= c.sequences ? c.starts[i + lane] : 0x7fffffff;
            before += __popcll(__ballot(x <= tok));
        }
        seq = before - 1;
        if (seq < 0 || seq >= c.sequences)
            return;
        place = tok - c.starts[seq];
    }
    else {
        seq = tok / c.maxNew;
        place = tok - seq * c.maxNew;
        if (seq >= c.sequences)
            return;
    }
    const int fresh = c.starts ? c.starts[seq + 1] - c.starts[seq] : c.maxNew;
    if (place < 0 || place >= fresh)
        return;
    const long long pos = (long long)c.lengths[seq] - fresh + place;
    if (pos < 0 || pos >= (long long)c.tablePages * c.pageSize.d || (p.rotation && pos >= p.positions))
        return;
    const int index = divided((int)pos, c.pageSize);
    const int page = c.table[(long long)seq * c.tablePages + index];
    const int row = (int)pos - index * (int)c.pageSize.d;
    const bool stored = page >= 0 && page < c.pages;

    const float * cs = p.rotation ? p.rotation + pos * p.rotated : nullptr;
    const int turned = turned_pieces<N>(p);
    const int copied = (c.dh - (p.rotation ? p.rotated : 0)) / N;
    const int perRow = turned + copied;                 /* items of a row of k or q; of v: dh / N */
    const int kItems = c.kvHeads * perRow, vItems = c.kvHeads * (c.dh / N);
    const int end = min(p.items, (part + 1) * p.perWave);
    for (int i = part * p.perWave + lane; i < end; i += 64) {
        if (i < kItems) {
            const int h = i / perRow;
            if (stored)
                turned_item<T, N>(static_cast<const T *>(p.nk) + tok * p.kT + h * p.kH,
                                  static_cast<T *>(c.k) + page * c.kP + row * c.kR + h * c.kH, i - h * perRow, turned, p, cs);
        }
        else if (i < kItems + vItems) {
            const int j = i - kItems, h = j / (c.dh / N), at = (j - h * (c.dh / N)) * N;
            if (stored)
                Columns<T, N>::copy(static_cast<const T *>(p.nv) + tok * p.vT + h * p.vH + at,
                                    static_cast<T *>(c.v) + page * c.vP + row * c.vR + h * c.vH + at);
        }
        else {
            const int j = i - kItems - vItems, h = j / perRow;
            turned_item<T, N>(static_cast<const T *>(p.q) + tok * p.qT + h * p.qH,
                              static_cast<T *>(p.qOut) + tok * p.oT + h * p.oH, j - h * perRow, turned, p, cs);
        }
    }
}

template <int N>
bool deal_items(AppendParams & p)
{
    const int turned = turned_pieces<N>(p), perRow = turned + (p.c.dh - (p.rotation ? p.rotated : 0)) / N;
    const long long items = (long long)p.c.kvHeads * (perRow + p.c.dh / N) + (p.q ? (long long)p.heads * perRow : 0);
    if (items > 0x7fffff00LL)                           /* ends of a wave's items are counted in 31 bits */
        return false;
    p.items = (int)items;
    /* A lane's items follow one another, each a load and a store that wait for memory: one each where the waves run at once (64 sequences
       of one token, 448 waves, replayed: 3.5 us; 4.6 with four). Beyond, what a wave does first counts, its look at the starts above all: two each
       (1 to 499 tokens of 7 sequences, float: 9.3, 7.7, 8.4 us with one, two and four; 8 prompts 48.5, 45.7, 47.5), four with more
       than 64 sequences (87 of up to 108 tokens: 13.9, 11.8, 9.9). */
    const int looks = p.c.starts ? p.c.sequences / 64 + 1 : 1;
    p.perWave = (long long)p.c.tokens * ((items + 63) / 64) * looks <= 1024 ? 64 : (looks == 1 ? 128 : 256);
    p.waves = (int)((items + p.perWave - 1) / p.perWave);
    return true;
}

template <typename T, int N>
int launch(AppendParams p, hipStream_t stream)
{
    const long long most = most_workgroups(256) * 4 / p.waves;      /* tokens of a launch */
    for (long long from = 0; from < p.c.tokens; from += most) {
        const long long n = p.c.tokens - from < most ? p.c.tokens - from : most;
        p.token0 = (int)from;
        hipLaunchKernelGGL((cache_append_kernel<T, N>), dim3((unsigned)((n * p.waves + 3) / 4)), dim3(256), 0, stream, p);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess)
            return (int)err;
    }
    return 0;
}

}  // namespace

/* 16-byte items need every row on a 16-byte boundary (the cache's are) and whole pieces of turned columns */
static bool whole_pieces(const AppendParams & p, bool half)
{
    const int n = half ? 8 : 4;
    const long long strides[8] = {p.kT, p.kH, p.vT, p.vH, p.q ? p.qT : 0, p.q ? p.qH : 0, p.q ? p.oT : 0, p.q ? p.oH : 0};
    for (int i = 0; i < 8; i++)
        if (strides[i] % n != 0)
            return false;
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.nk) | reinterpret_cast<uintptr_t>(p.nv) |
                         (p.q ? reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.qOut) : 0);
    if ((at & 15) != 0)
        return false;
    return !p.rotation || (p.pairing == 0 ? p.rotated / 2 : p.rotated) % n == 0;
}

bool plan_cache_append(AppendParams & p, bool half)
{
    p.whole = whole_pieces(p, half);
    return !p.whole ? deal_items<1>(p) : (half ? deal_items<8>(p) : deal_items<4>(p));
}

int launch_cache_append(AppendParams p, bool half, hipStream_t stream)
{
    if (half)
        return p.whole ? launch<half_t, 8>(p, stream) : launch<half_t, 1>(p, stream);
    return p.whole ? launch<float, 4>(p, stream) : launch<float, 1>(p, stream);
}

}  // namespace ntsamd
