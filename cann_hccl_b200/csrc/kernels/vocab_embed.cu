// Token embedding:  out[t] = scale * W[id_t - first], zeros for ids outside the table, and its gradient
// dW[v] = scale * sum over the tokens with id_t = first + v of dY[t].
//
// Lookup: a warp takes one stretch of one row (128 bytes per lane in flight), so that a decode batch spreads over the GPU and a
// prefill batch keeps every SM's loads in flight.  Bound: HBM (16384 tokens x 8192 bf16 in 60 us, 6.4 TB/s).
//
// Gradient: the tokens are sorted by id (stable, so that the sums have one order whatever ran before), then a CTA walks a tile of
// the sorted list, keeps the running row in fp32 registers and writes it when the id changes: every row of dY is read once and
// every row of the table written once, without atomics on sums.  A run of one id that crosses tiles leaves fp32 pieces, which a last
// launch adds in order, so that a token that makes up a large part of a text is summed by many CTAs.  The sort leaves a bit for each
// row that has a token; the launch that sums also zeroes the others (reads and writes together run at 7.0 TB/s; the table zeroed by
// the SMs that the sort leaves idle, and its rows written twice: 185 + 70 us instead of 188 for 32768 tokens, 128256 x 4096).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <algorithm>
#include <cstring>
#include "common/base.h"
#include "common/log.h"
#include "kernels/pdl.cuh"
#include "kernels/smem_grant.h"
#include "kernels/vocab_embed.h"

namespace hcclb {

namespace {

// ---------------------------------------------------------------------------------------------------- vectors of B bytes
template <int B> struct Bytes;
template <> struct Bytes<32> { uint32_t w[8]; };
template <> struct Bytes<16> { uint32_t w[4]; };
template <> struct Bytes<4> { uint32_t w[1]; };
template <> struct Bytes<2> { uint16_t h; };

__device__ __forceinline__ void ld(Bytes<32> &v, const void *p)
{
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]), "=r"(v.w[7]) : "l"(p) : "memory");
}
__device__ __forceinline__ void ld(Bytes<16> &v, const void *p)
{
    const uint4 u = *(const uint4 *)p;
    v.w[0] = u.x; v.w[1] = u.y; v.w[2] = u.z; v.w[3] = u.w;
}
__device__ __forceinline__ void ld(Bytes<4> &v, const void *p) { v.w[0] = *(const uint32_t *)p; }
__device__ __forceinline__ void ld(Bytes<2> &v, const void *p) { v.h = *(const uint16_t *)p; }
__device__ __forceinline__ void st(void *p, const Bytes<32> &v)
{
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"l"(p), "r"(v.w[0]), "r"(v.w[1]), "r"(v.w[2]), "r"(v.w[3]), "r"(v.w[4]), "r"(v.w[5]), "r"(v.w[6]), "r"(v.w[7]) : "memory");
}
__device__ __forceinline__ void st(void *p, const Bytes<16> &v) { *(uint4 *)p = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]); }
__device__ __forceinline__ void st(void *p, const Bytes<4> &v) { *(uint32_t *)p = v.w[0]; }
__device__ __forceinline__ void st(void *p, const Bytes<2> &v) { *(uint16_t *)p = v.h; }

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <class T, int B> __device__ __forceinline__ void unpack(const Bytes<B> &v, float (&f)[B / sizeof(T)])
{
    T e[B / sizeof(T)];
    memcpy(e, &v, B);
#pragma unroll
    for (int i = 0; i < (int)(B / sizeof(T)); ++i) f[i] = to_f(e[i]);
}
template <class T, int B> __device__ __forceinline__ Bytes<B> pack(const float (&f)[B / sizeof(T)], float scale)
{
    T e[B / sizeof(T)];
#pragma unroll
    for (int i = 0; i < (int)(B / sizeof(T)); ++i) e[i] = from_f<T>(f[i] * scale);
    Bytes<B> v;
    memcpy(&v, e, B);
    return v;
}

__device__ __forceinline__ int64_t id_at(const void *ids, int wide, int64_t t) { return wide ? ((const int64_t *)ids)[t] : (int64_t)((const int32_t *)ids)[t]; }
// Row of the table that id stands for, -1 outside it (no overflow for any id: the difference is taken unsigned).
__device__ __forceinline__ int64_t row_of(int64_t id, int64_t first, int64_t vocab)
{
    const uint64_t r = (uint64_t)id - (uint64_t)first;
    return r < (uint64_t)vocab ? (int64_t)r : -1;
}

// ---------------------------------------------------------------------------------------------------- lookup
struct LookupArgs {
    const void *ids;
    const uint8_t *w;
    uint8_t *out;
    int64_t tokens, units, vocab, first, stride;  // units: stretches of all rows; stride: bytes between rows of w
    int wide, nvec, nseg;
    float scale;
};
constexpr int kLookupThreads = 128;
template <int B> constexpr int kLookupVecs = B >= 16 ? 128 / B : 8;  // vectors of a lane

template <class T, int B, bool kScale>
__global__ void __launch_bounds__(kLookupThreads) embed_lookup_kernel(const __grid_constant__ LookupArgs a)
{
    constexpr int U = kLookupVecs<B>;
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int64_t unit = (int64_t)blockIdx.x * (kLookupThreads / 32) + threadIdx.x / 32;
    if (unit >= a.units) return;
    const int64_t t = a.nseg == 1 ? unit : unit / a.nseg;
    const int v0 = (int)(unit - t * a.nseg) * (32 * U) + lane;
    pdl_wait();
    const int64_t row = row_of(id_at(a.ids, a.wide, t), a.first, a.vocab);
    Bytes<B> x[U];
    memset(x, 0, sizeof(x));
    if (row >= 0) {
        const uint8_t *src = a.w + row * a.stride;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (v0 + 32 * u < a.nvec) ld(x[u], src + (int64_t)(v0 + 32 * u) * B);
    }
    uint8_t *dst = a.out + t * a.nvec * B;
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (v0 + 32 * u < a.nvec) {
            if (kScale) {
                float f[B / sizeof(T)];
                unpack<T, B>(x[u], f);
                x[u] = pack<T, B>(f, a.scale);
            }
            st(dst + (int64_t)(v0 + 32 * u) * B, x[u]);
        }
}

// ---------------------------------------------------------------------------------------------------- stable sort by id
// A pair is (row of the table, token); rows outside the table sort behind all others as `vocab`.  Few tokens: a token's place is the
// number of tokens that belong before it, counted by comparing with all of them.  More: radix sort from the least significant digit;
// a warp takes consecutive stretches of 32 pairs, __match_any_sync gives the lanes of one digit, the warp's counters in shared
// memory the earlier stretches, so equal digits keep their order.
// (1531 tokens by counting 6.0 us; one CTA of a radix sort 8.1 us, one cluster 13 us, both exchanging through shared memory; 32768
// tokens: a cluster 25 us, the tiles below 20 us.  The whole gradient of rows of 64: 4096 tokens by counting 22 us, 8192 47 us, by
// tiles 29 us.)
constexpr int kCountMost = 4096, kCountTokens = 32, kCountThreads = 256;  // tokens that are sorted by counting, tokens of a CTA
constexpr int kWindow = 1 << 18;                                          // rows whose bits a CTA makes
constexpr int kDigitBits = 9, kBins = 1 << kDigitBits;
constexpr int kSortItems = 8;
// CTAs of the radix sort: small ones for parallelism, large ones so that the histograms that each of them reads stay few
constexpr int kSmallTile = 256, kLargeTile = 1024;
constexpr int64_t kSmallMost = 256 << 10;  // tokens

struct SortArgs {
    const void *ids;                 // first pass
    int wide;
    int64_t vocab, first;
    const uint2 *in;                 // later passes
    uint2 *out;
    int32_t *hist;                   // [tile][bin]
    int64_t tokens;
    uint32_t *has;                   // a bit for each row with a token, cleared and set on the way (null: not wanted)
    int tiles, shift, passes, digit, last;
};

// Ranks of a warp's pairs within (warp, digit); counts[warp][bin] end up holding the warp's pairs of each digit.
__device__ __forceinline__ void warp_ranks(const uint32_t (&key)[kSortItems], int shift, uint32_t mask, int32_t *counts, int (&rank)[kSortItems])
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int32_t *mine = counts + warp * kBins;
#pragma unroll
    for (int i = 0; i < kSortItems; ++i) {
        const uint32_t d = (key[i] >> shift) & mask;
        const uint32_t peers = __match_any_sync(0xffffffffu, d);
        const int before = mine[d], below = __popc(peers & ((1u << lane) - 1));
        __syncwarp();
        if (below == 0) mine[d] = before + __popc(peers);
        __syncwarp();
        rank[i] = before + below;
    }
}

// counts[warp][bin] -> pairs of the bin in earlier warps; returns the bin's total for thread `bin`.
template <int WARPS> __device__ __forceinline__ int warp_prefix(int32_t *counts, int bin)
{
    int t = 0;
#pragma unroll 8
    for (int w = 0; w < WARPS; ++w) {
        const int n = counts[w * kBins + bin];
        counts[w * kBins + bin] = t;
        t += n;
    }
    return t;
}

// Exclusive prefix over the bins; thread i of the first kBins / N threads holds N consecutive bins' totals.
template <int N> __device__ __forceinline__ void bins_prefix(int (&t)[N], int32_t *s_warp)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int own = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) { const int n = t[i]; t[i] = own; own += n; }
    int v = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int w = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += w;
    }
    if (lane == 31) s_warp[warp] = v;
    __syncthreads();
    int base = v - own;
    for (int w = 0; w < warp; ++w) base += s_warp[w];
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] += base;
}

__device__ __forceinline__ void mark_row(const SortArgs &a, uint32_t row)
{
    if (!a.has || row >= (uint32_t)a.vocab) return;
    uint32_t *word = a.has + (row >> 5);
    const uint32_t bit = 1u << (row & 31);
    // where tokens are more than rows most find their bit set (2^20 tokens of 1000 rows: 370 us for their atomics alone); elsewhere the
    // look costs more than it saves (32768 tokens of 128256 rows: 3 us)
    if (a.tokens < a.vocab || !(__ldcg(word) & bit)) atomicOr(word, bit);
}

__device__ __forceinline__ uint32_t key_at(const SortArgs &a, int64_t t)
{
    const int64_t r = row_of(id_at(a.ids, a.wide, t), a.first, a.vocab);
    return r >= 0 ? (uint32_t)r : (uint32_t)a.vocab;
}

// Up to kCountMost tokens: grid of token groups, then of windows of the table's bits.  Dynamic shared memory: keys of all tokens (a
// multiple of 4, those behind the last one above every other), bits of a window.
__global__ void __launch_bounds__(kCountThreads) embed_sort_count_kernel(const __grid_constant__ SortArgs a)
{
    extern __shared__ uint4 sh4[];
    __shared__ int s_rank[kCountThreads / 32][kCountTokens];
    uint32_t *keys = (uint32_t *)sh4;
    const int n = (int)a.tokens, padded = (n + 3) / 4 * 4, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_trigger();
    pdl_wait();
    for (int t = threadIdx.x; t < padded; t += kCountThreads) keys[t] = t < n ? key_at(a, t) : 0xffffffffu;
    if ((int)blockIdx.x >= a.tiles) {
        uint32_t *bits = keys + padded;
        const uint32_t r0 = (uint32_t)(blockIdx.x - a.tiles) * kWindow, rows = (uint32_t)min((int64_t)kWindow, a.vocab - r0), words = (rows + 31) / 32;
        for (uint32_t i = threadIdx.x; i < words; i += kCountThreads) bits[i] = 0;
        __syncthreads();
        for (int t = threadIdx.x; t < n; t += kCountThreads) {
            const uint32_t r = keys[t] - r0;
            if (r < rows) atomicOr(bits + (r >> 5), 1u << (r & 31));
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < words; i += kCountThreads) a.has[(r0 >> 5) + i] = bits[i];
        return;
    }
    __syncthreads();
    const int t = (int)blockIdx.x * kCountTokens + lane;
    const uint32_t mine = t < n ? keys[t] : 0xffffffffu;
    int rank = 0;
    const uint4 *k4 = (const uint4 *)keys;
#pragma unroll 4
    for (int q = warp; q < padded / 4; q += kCountThreads / 32) {
        const uint4 k = k4[q];
        // earlier tokens come before equal ones, later ones do not
        rank += (k.x < mine + (q * 4 < t)) + (k.y < mine + (q * 4 + 1 < t)) + (k.z < mine + (q * 4 + 2 < t)) + (k.w < mine + (q * 4 + 3 < t));
    }
    s_rank[warp][lane] = rank;
    __syncthreads();
    if (warp || t >= n) return;
    rank = 0;
#pragma unroll
    for (int w = 0; w < kCountThreads / 32; ++w) rank += s_rank[w][lane];
    a.out[rank] = make_uint2(mine, (uint32_t)t);
}

template <int THREADS>
__device__ __forceinline__ void load_tile(const SortArgs &a, int64_t tile, uint32_t (&key)[kSortItems], uint32_t (&pos)[kSortItems])
{
    const int64_t t0 = tile * (THREADS * kSortItems) + (threadIdx.x >> 5) * (32 * kSortItems) + (threadIdx.x & 31);
#pragma unroll
    for (int i = 0; i < kSortItems; ++i) {
        const int64_t t = t0 + i * 32;
        key[i] = 0xffffffffu;
        pos[i] = 0;
        if (t < a.tokens) {
            if (a.in) {
                const uint2 p = a.in[t];
                key[i] = p.x; pos[i] = p.y;
            } else {
                key[i] = key_at(a, t);
                pos[i] = (uint32_t)t;
            }
        }
    }
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) embed_sort_hist_kernel(const __grid_constant__ SortArgs a)
{
    __shared__ int32_t bins[kBins];
    for (int i = threadIdx.x; i < kBins; i += THREADS) bins[i] = 0;
    __syncthreads();
    pdl_trigger();
    pdl_wait();
    if (a.has && !a.in)  // the first pass clears the bits, the last one sets them
        for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < (a.vocab + 31) / 32; i += (int64_t)gridDim.x * THREADS) a.has[i] = 0;
    uint32_t key[kSortItems], pos[kSortItems];
    load_tile<THREADS>(a, blockIdx.x, key, pos);
    const int64_t t0 = (int64_t)blockIdx.x * (THREADS * kSortItems) + (threadIdx.x >> 5) * (32 * kSortItems) + (threadIdx.x & 31);
#pragma unroll
    for (int i = 0; i < kSortItems; ++i)
        if (t0 + i * 32 < a.tokens) atomicAdd(&bins[(key[i] >> a.shift) & ((1u << a.digit) - 1)], 1);
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += THREADS) a.hist[(int64_t)blockIdx.x * kBins + i] = bins[i];
}

// Dynamic shared memory: [warp][bin] counters, first place of each bin.
template <int THREADS> constexpr size_t kScatterSmem = (size_t)(THREADS / 32 + 1) * kBins * 4;
template <int THREADS>
__global__ void __launch_bounds__(THREADS) embed_sort_scatter_kernel(const __grid_constant__ SortArgs a)
{
    constexpr int W = THREADS / 32, N = kBins > THREADS ? kBins / THREADS : 1;  // N bins of a thread
    extern __shared__ uint4 sh4[];
    __shared__ int32_t s_warp[W];
    int32_t *counts = (int32_t *)sh4, *base = counts + W * kBins;
    for (int i = threadIdx.x; i < W * kBins; i += THREADS) counts[i] = 0;
    __syncthreads();
    pdl_trigger();
    pdl_wait();
    uint32_t key[kSortItems], pos[kSortItems];
    load_tile<THREADS>(a, blockIdx.x, key, pos);
    const uint32_t mask = (1u << a.digit) - 1;
    const bool mine = (int)threadIdx.x * N < kBins;
    int rank[kSortItems];
    warp_ranks(key, a.shift, mask, counts, rank);
    // pairs of each bin in earlier tiles, and of all smaller bins in all tiles
    int before[N], total[N];
#pragma unroll
    for (int j = 0; j < N; ++j) before[j] = total[j] = 0;
    if (mine)
#pragma unroll 8
        for (int q = 0; q < a.tiles; ++q)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int h = a.hist[(int64_t)q * kBins + threadIdx.x * N + j];
                total[j] += h;
                before[j] += q < (int)blockIdx.x ? h : 0;
            }
    bins_prefix<N>(total, s_warp);  // its barrier puts all warps' counters before warp_prefix
    if (mine)
#pragma unroll
        for (int j = 0; j < N; ++j) {
            base[threadIdx.x * N + j] = total[j] + before[j];
            warp_prefix<W>(counts, threadIdx.x * N + j);
        }
    __syncthreads();
    const int64_t t0 = (int64_t)blockIdx.x * (THREADS * kSortItems) + (threadIdx.x >> 5) * (32 * kSortItems) + (threadIdx.x & 31);
#pragma unroll
    for (int i = 0; i < kSortItems; ++i)
        if (t0 + i * 32 < a.tokens) {  // pairs that pad the tile are last in it: they displace none of the others
            const uint32_t d = (key[i] >> a.shift) & mask;
            a.out[base[d] + counts[(threadIdx.x >> 5) * kBins + d] + rank[i]] = make_uint2(key[i], pos[i]);
            if (a.last) mark_row(a, key[i]);
        }
}

// ---------------------------------------------------------------------------------------------------- sums by row
struct SumArgs {
    const uint2 *pairs;              // sorted
    const uint8_t *dy;
    void *out;
    float *pieces;                   // [tile][2][nvec * per]: run from an earlier tile, run that goes on behind the tile
    int64_t tokens, vocab, stride;   // stride: bytes between rows of dy
    const uint32_t *has;             // bits of the rows with a token (null: none has one)
    int64_t tiles;
    int rows, nvec, nslice, add, wide, zero_rows;  // rows: tokens of a tile; wide: rows of an fp32 out that is added to are whole sectors
    float scale;
};
constexpr int kSumThreads = 256, kSumBatch = 4, kMostRows = 256;

template <class T, int B> __device__ __forceinline__ void put_row(const SumArgs &a, int64_t row, int v, const float (&acc)[B / sizeof(T)])
{
    constexpr int N = B / sizeof(T);
    const int64_t at = (row * a.nvec + v) * N;
    if (a.add) {
        float *p = (float *)a.out + at;
        if (N == 8 && a.wide) {  // one 32-byte sector of a lane
            Bytes<32> v;
            ld(v, p);
            float f[8];
            unpack<float, 32>(v, f);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = fmaf(acc[i < N ? i : 0], a.scale, f[i]);
            st(p, pack<float, 32>(f, 1.f));
        } else
#pragma unroll
            for (int i = 0; i < N; ++i) p[i] = fmaf(acc[i], a.scale, p[i]);
    } else
        st((T *)a.out + at, pack<T, B>(acc, a.scale));
}

// Zeros over `bytes` bytes from p, by the whole CTA: 32-byte stores whatever the rows' own alignment is.
template <int SIZE> __device__ __forceinline__ void zero_bytes(uint8_t *p, int64_t bytes)
{
    const int64_t head = min(bytes, (int64_t)(-(uintptr_t)p & 31)), body = (bytes - head) / 32, tail = bytes - head - body * 32;
    Bytes<32> zero;
    memset(&zero, 0, sizeof(zero));
    Bytes<SIZE> one;
    memset(&one, 0, sizeof(one));
    for (int64_t i = (int64_t)threadIdx.x * SIZE; i < head; i += blockDim.x * SIZE) st(p + i, one);
    for (int64_t i = threadIdx.x; i < body; i += blockDim.x) st(p + head + i * 32, zero);
    for (int64_t i = (int64_t)threadIdx.x * SIZE; i < tail; i += blockDim.x * SIZE) st(p + head + body * 32 + i, one);
}

// grid: tiles x slices of a row, then CTAs that zero zero_rows rows of the table each where they have no token
template <class T, int B>
__global__ void __launch_bounds__(kSumThreads) embed_sum_kernel(const __grid_constant__ SumArgs a)
{
    constexpr int N = B / sizeof(T);
    __shared__ uint2 s_pair[kMostRows];
    __shared__ uint32_t s_edge[2];
    pdl_trigger();
    pdl_wait();
    const int64_t sums = a.tiles * a.nslice;
    if ((int64_t)blockIdx.x >= sums) {
        const int64_t r0 = ((int64_t)blockIdx.x - sums) * a.zero_rows;
        const int n = (int)min((int64_t)a.zero_rows, a.vocab - r0);
        const uint32_t has = a.has ? a.has[r0 >> 5] >> (r0 & 31) : 0;
        for (int i = 0; i < n;) {
            if (has >> i & 1) { ++i; continue; }
            const int from = i;
            while (i < n && !(has >> i & 1)) ++i;
            zero_bytes<sizeof(T)>((uint8_t *)a.out + (r0 + from) * a.nvec * B, (int64_t)(i - from) * a.nvec * B);
        }
        return;
    }
    const int64_t tile = blockIdx.x / a.nslice, t0 = tile * a.rows;
    const int v = (int)(blockIdx.x - tile * a.nslice) * (int)blockDim.x + threadIdx.x, n = (int)min((int64_t)a.rows, a.tokens - t0);
    for (int i = threadIdx.x; i < n; i += blockDim.x) s_pair[i] = a.pairs[t0 + i];
    if (threadIdx.x == 0) {
        s_edge[0] = t0 > 0 ? a.pairs[t0 - 1].x : 0xffffffffu;
        s_edge[1] = t0 + n < a.tokens ? a.pairs[t0 + n].x : 0xffffffffu;
    }
    __syncthreads();
    if (v >= a.nvec) return;
    float acc[N];
    uint32_t cur = s_pair[0].x;
    bool head = cur == s_edge[0];  // the run in hand came in from an earlier tile
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
    const uint8_t *src = a.dy + (int64_t)v * B;
    for (int i0 = 0; i0 < n; i0 += kSumBatch) {
        Bytes<B> x[kSumBatch];
#pragma unroll
        for (int j = 0; j < kSumBatch; ++j)
            if (i0 + j < n && s_pair[i0 + j].x < (uint32_t)a.vocab) ld(x[j], src + (int64_t)s_pair[i0 + j].y * a.stride);
#pragma unroll
        for (int j = 0; j < kSumBatch; ++j) {
            if (i0 + j >= n) break;
            const uint32_t key = s_pair[i0 + j].x;
            if (key != cur) {
                if (head) {
                    float *p = a.pieces + ((tile * 2) * a.nvec + v) * N;
#pragma unroll
                    for (int i = 0; i < N; ++i) p[i] = acc[i];
                } else
                    put_row<T, B>(a, cur, v, acc);
                cur = key;
                head = false;
#pragma unroll
                for (int i = 0; i < N; ++i) acc[i] = 0.f;
            }
            if (key >= (uint32_t)a.vocab) return;  // outside the table: nothing but such tokens follows
            float f[N];
            unpack<T, B>(x[j], f);
#pragma unroll
            for (int i = 0; i < N; ++i) acc[i] += f[i];
        }
    }
    const bool tail = cur == s_edge[1];
    if (head || tail) {
        float *p = a.pieces + ((tile * 2 + (head ? 0 : 1)) * a.nvec + v) * N;
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = acc[i];
    } else
        put_row<T, B>(a, cur, v, acc);
}

// Up to M pieces, one after the other but loaded together.
template <int N, int M> __device__ __forceinline__ void add_pieces(const float *src, int64_t hidden, int n, float (&acc)[N])
{
    float h[M][N];
#pragma unroll
    for (int j = 0; j < M; ++j)
        if (j < n) {
            if (N == 4) *(float4 *)h[j] = *(const float4 *)(src + j * 2 * hidden);
            else h[j][0] = src[j * 2 * hidden];
        }
#pragma unroll
    for (int j = 0; j < M; ++j)
        if (j < n)
#pragma unroll
            for (int i = 0; i < N; ++i) acc[i] += h[j][i];
}

// The runs that begin in a tile and go on behind it: their pieces, in order.  N columns of a thread, sixteen pieces in flight (with one at
// a time, and 16 columns: 32768 tokens x 4096, the most frequent one 1900 times, 72 us).
template <class T, int N>
__global__ void __launch_bounds__(kSumThreads) embed_join_kernel(const __grid_constant__ SumArgs a)
{
    pdl_trigger();
    const int64_t tile = blockIdx.x / a.nslice, t1 = (tile + 1) * a.rows;  // not the last tile
    const int64_t c = ((int64_t)(blockIdx.x - tile * a.nslice) * blockDim.x + threadIdx.x) * N, hidden = a.nvec;
    pdl_wait();
    const uint32_t key = a.pairs[t1 - 1].x;
    if (key >= (uint32_t)a.vocab || a.pairs[t1].x != key || (tile > 0 && a.pairs[tile * a.rows - 1].x == key)) return;
    int64_t last = tile;  // tile in which the run ends: a warp looks at the first rows of 32 tiles at a time
    for (uint32_t same = ~0u; same == ~0u;) {
        const int64_t q = last + 1 + (threadIdx.x & 31);
        same = __ballot_sync(0xffffffffu, q < a.tiles && a.pairs[q * a.rows].x == key);
        last += same == ~0u ? 32 : __ffs(~same) - 1;
    }
    if (c >= hidden) return;
    float acc[N];
    const float *p = a.pieces + (tile * 2 + 1) * hidden + c;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = p[i];
    int64_t q0 = tile + 1;
    for (; q0 + 15 <= last; q0 += 16) add_pieces<N, 16>(a.pieces + q0 * 2 * hidden + c, hidden, 16, acc);
    for (; q0 <= last; q0 += 4) add_pieces<N, 4>(a.pieces + q0 * 2 * hidden + c, hidden, (int)min((int64_t)4, last - q0 + 1), acc);
    const int64_t at = (int64_t)key * hidden + c;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (a.add) ((float *)a.out)[at + i] = fmaf(acc[i], a.scale, ((float *)a.out)[at + i]);
        else ((T *)a.out)[at + i] = from_f<T>(acc[i] * a.scale);
    }
}

// ---------------------------------------------------------------------------------------------------- launches
template <class K> HcclResult grid_of(int64_t ctas, K *out, const char *what)
{
    CHK_RET_LOG(ctas > 0x7fffffff, HCCL_E_PARA, "%s: too many rows for one launch (%lld CTAs)", what, (long long)ctas);
    *out = (K)ctas;
    return HCCL_SUCCESS;
}

// Widest vector that every row starts on and is a whole number of; `lanes`: narrower ones where a row has fewer vectors than that.
int vector_bytes(int64_t row_bytes, uintptr_t bits, int size, int lanes)
{
    bits |= (uintptr_t)row_bytes;
    if (row_bytes < 32 * lanes) bits |= 16;
    if (row_bytes < 16 * lanes) bits |= 4;
    return bits % 32 == 0 ? 32 : bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : size;
}

template <class T, int B> HcclResult lookup(LookupArgs &a, int64_t row_bytes, void *stream)
{
    a.nvec = (int)(row_bytes / B);
    a.nseg = (a.nvec + 32 * kLookupVecs<B> - 1) / (32 * kLookupVecs<B>);
    a.units = a.tokens * a.nseg;
    unsigned ctas;
    CHK_RET(grid_of((a.units + kLookupThreads / 32 - 1) / (kLookupThreads / 32), &ctas, "embedding"));
    const void *fn = a.scale == 1.f ? (const void *)embed_lookup_kernel<T, B, false> : (const void *)embed_lookup_kernel<T, B, true>;
    return launch_pdl(fn, dim3(ctas), kLookupThreads, 0, &a, stream, "embedding");
}

template <class T> HcclResult lookup_typed(LookupArgs &a, int64_t hidden, void *stream)
{
    const int64_t row = hidden * (int64_t)sizeof(T);
    switch (vector_bytes(row, (uintptr_t)a.w | (uintptr_t)a.out | (uintptr_t)a.stride, sizeof(T), 1)) {
        case 32: return lookup<T, 32>(a, row, stream);
        case 16: return lookup<T, 16>(a, row, stream);
        case 4: return lookup<T, 4>(a, row, stream);
        default: return lookup<T, sizeof(T)>(a, row, stream);
    }
}

// Tokens of a tile: short tiles for parallelism, longer ones where there are many tokens, so that a run has few pieces.
int tile_rows(int64_t tokens) { return (int)std::min<int64_t>(kMostRows, std::max<int64_t>(32, (tokens / 592 + 31) / 32 * 32)); }

struct Scratch { int64_t pairs, spare, hist, has, pieces, bytes; };
Scratch scratch_of(int64_t tokens, int64_t vocab, int32_t hidden)
{
    auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
    Scratch s;
    const int64_t tiles = (tokens + tile_rows(tokens) - 1) / tile_rows(tokens);
    s.pairs = 0;
    s.spare = s.pairs + up(tokens * 8);
    s.hist = s.spare + (tokens > kCountMost ? up(tokens * 8) : 0);
    s.has = s.hist + (tokens > kCountMost ? up(std::max((std::min(tokens, kSmallMost) - 1) / (kSmallTile * kSortItems), (tokens - 1) / (kLargeTile * kSortItems)) * kBins * 4 + kBins * 4) : 0);
    s.pieces = s.has + (tokens ? up((vocab + 31) / 32 * 4) : 0);
    s.bytes = s.pieces + (tiles > 1 ? up(tiles * 2 * hidden * 4) : 0);
    return s;
}

template <class T, int B> HcclResult sum(SumArgs &a, int64_t row_bytes, void *stream)
{
    a.nvec = (int)(row_bytes / B);
    const int threads = std::min(kSumThreads, (a.nvec + 31) / 32 * 32);
    a.nslice = (a.nvec + threads - 1) / threads;
    unsigned ctas;
    a.zero_rows = 32;  // those of one word, fewer where they are long
    while (a.zero_rows > 1 && a.zero_rows * row_bytes > 65536) a.zero_rows /= 2;
    CHK_RET(grid_of(a.tiles * a.nslice + (a.add ? 0 : (a.vocab + a.zero_rows - 1) / a.zero_rows), &ctas, "embedding gradient"));
    if (ctas) CHK_RET(launch_pdl((const void *)embed_sum_kernel<T, B>, dim3(ctas), (unsigned)threads, 0, &a, stream, "embedding gradient"));
    if (a.tiles <= 1) return HCCL_SUCCESS;
    const int hidden = (int)(row_bytes / (int64_t)sizeof(T)), n = hidden % 4 ? 1 : 4, join = std::min(kSumThreads, (hidden / n + 31) / 32 * 32);
    a.nvec = hidden;
    a.nslice = (hidden / n + join - 1) / join;
    CHK_RET(grid_of((a.tiles - 1) * a.nslice, &ctas, "embedding gradient (join)"));
    return launch_pdl(n == 4 ? (const void *)embed_join_kernel<T, 4> : (const void *)embed_join_kernel<T, 1>, dim3(ctas), (unsigned)join, 0, &a, stream,
                      "embedding gradient (join)");
}

template <class T> HcclResult sum_typed(SumArgs &a, int64_t hidden, void *stream)
{
    const int64_t row = hidden * (int64_t)sizeof(T);
    a.wide = a.add && hidden % 8 == 0 && ((uintptr_t)a.out & 31) == 0;
    // where sums are added to an fp32 row a lane has eight columns, a sector of it, at most (with sixteen, one word at a time: 32768 tokens of
    // 128256 x 4096 954 us)
    const uintptr_t sector = a.add && sizeof(T) == 2 ? 16 : 0;
    switch (vector_bytes(row, (uintptr_t)a.dy | (uintptr_t)a.stride | sector | (a.add ? 0 : (uintptr_t)a.out), sizeof(T), 32)) {
        case 32: return sum<T, 32>(a, row, stream);
        case 16: return sum<T, 16>(a, row, stream);
        case 4: return sum<T, 4>(a, row, stream);
        default: return sum<T, sizeof(T)>(a, row, stream);
    }
}

template <int THREADS> HcclResult sort_tiles(SortArgs &a, uint2 *const (&buf)[2], void *stream, const uint2 **sorted)
{
    a.tiles = (int)((a.tokens + THREADS * kSortItems - 1) / (THREADS * kSortItems));
    const void *scatter = (const void *)embed_sort_scatter_kernel<THREADS>;
    if (kScatterSmem<THREADS> > 32 * 1024) CHK_RET(grant_smem(scatter, kScatterSmem<THREADS>, "embedding gradient"));
    for (int pass = 0; pass < a.passes; ++pass) {
        a.in = pass ? buf[(pass - 1) & 1] : nullptr;
        a.out = buf[pass & 1];
        a.shift = pass * a.digit;
        a.last = pass == a.passes - 1;
        CHK_RET(launch_pdl((const void *)embed_sort_hist_kernel<THREADS>, dim3((unsigned)a.tiles), THREADS, 0, &a, stream, "embedding gradient (histogram)"));
        CHK_RET(launch_pdl(scatter, dim3((unsigned)a.tiles), THREADS, kScatterSmem<THREADS>, &a, stream, "embedding gradient (scatter)"));
        *sorted = a.out;
    }
    return HCCL_SUCCESS;
}

HcclResult sort_tokens(const EmbedTable &t, const EmbedIds &ids, const Scratch &s, uint8_t *scratch, uint32_t *has, void *stream, const uint2 **sorted)
{
    SortArgs a;
    memset(&a, 0, sizeof(a));
    a.ids = ids.ids; a.wide = ids.wide; a.vocab = t.vocab; a.first = t.first; a.tokens = ids.tokens;
    a.has = has;
    int bits = 1;
    while ((t.vocab >> bits) != 0) ++bits;  // rows 0 .. vocab
    a.passes = (bits + kDigitBits - 1) / kDigitBits;
    a.digit = (bits + a.passes - 1) / a.passes;
    uint2 *buf[2] = {(uint2 *)(scratch + s.pairs), (uint2 *)(scratch + s.spare)};
    if (ids.tokens <= kCountMost) {
        a.out = buf[0];
        *sorted = buf[0];
        a.tiles = (int)((ids.tokens + kCountTokens - 1) / kCountTokens);
        const size_t smem = (size_t)(ids.tokens + 3) / 4 * 16 + (has ? kWindow / 8 : 0);
        if (smem > 32 * 1024) CHK_RET(grant_smem((const void *)embed_sort_count_kernel, kCountMost * 4 + kWindow / 8, "embedding gradient"));
        const int64_t windows = has ? (t.vocab + kWindow - 1) / kWindow : 0;
        return launch_pdl((const void *)embed_sort_count_kernel, dim3((unsigned)(a.tiles + windows)), kCountThreads, smem, &a, stream, "embedding gradient (sort)");
    }
    a.hist = (int32_t *)(scratch + s.hist);
    return ids.tokens <= kSmallMost ? sort_tiles<kSmallTile>(a, buf, stream, sorted) : sort_tiles<kLargeTile>(a, buf, stream, sorted);
}

}  // namespace

HcclResult embed_lookup(const EmbedTable &t, const EmbedIds &ids, const void *weights, int64_t stride, float scale, void *out, void *stream)
{
    if (!ids.tokens) return HCCL_SUCCESS;
    const int size = dtype_size(t.type);
    LookupArgs a;
    memset(&a, 0, sizeof(a));
    a.ids = ids.ids; a.wide = ids.wide; a.tokens = ids.tokens;
    a.w = (const uint8_t *)weights; a.out = (uint8_t *)out;
    a.vocab = t.vocab; a.first = t.first; a.stride = stride * size; a.scale = scale;
    switch (t.type) {
        case HCCL_DATA_TYPE_FP32: return lookup_typed<float>(a, t.hidden, stream);
        case HCCL_DATA_TYPE_FP16: return lookup_typed<__half>(a, t.hidden, stream);
        default: return lookup_typed<__nv_bfloat16>(a, t.hidden, stream);
    }
}

int64_t embed_grad_scratch_bytes(int64_t tokens, int64_t vocab, int32_t hidden) { return std::max<int64_t>(256, scratch_of(tokens, vocab, hidden).bytes); }

HcclResult embed_grad(const EmbedTable &t, const EmbedIds &ids, const void *grad, int64_t stride, float scale, void *out, bool add, void *scratch,
                      void *stream)
{
    const Scratch s = scratch_of(ids.tokens, t.vocab, t.hidden);
    SumArgs a;
    memset(&a, 0, sizeof(a));
    uint32_t *has = add ? nullptr : (uint32_t *)((uint8_t *)scratch + s.has);
    if (ids.tokens) {
        CHK_RET(sort_tokens(t, ids, s, (uint8_t *)scratch, has, stream, &a.pairs));
        a.has = has;
    }
    a.dy = (const uint8_t *)grad; a.stride = stride * dtype_size(t.type);
    a.out = out; a.add = add; a.scale = scale;
    a.tokens = ids.tokens; a.vocab = t.vocab;
    a.rows = tile_rows(ids.tokens);
    a.tiles = (ids.tokens + a.rows - 1) / a.rows;
    a.pieces = (float *)((uint8_t *)scratch + s.pieces);
    switch (t.type) {
        case HCCL_DATA_TYPE_FP32: return sum_typed<float>(a, t.hidden, stream);
        case HCCL_DATA_TYPE_FP16: return sum_typed<__half>(a, t.hidden, stream);
        default: return sum_typed<__nv_bfloat16>(a, t.hidden, stream);
    }
}

}  // namespace hcclb
