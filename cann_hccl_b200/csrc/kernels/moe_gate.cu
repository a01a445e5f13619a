// Router of a mixture-of-experts layer.  For each token: p = softmax(logits), the top-k experts by logit (equal logits: the lowest
// expert; -inf is never chosen, its slot gets expert -1 and gate 0), gates = p of the chosen ones, divided by their sum where they
// are normalised.  Over the tokens that are routed (n of them: not masked, not all -inf): counts[e] pairs of expert e,
// prob_sum[e] = sum of p[.,e], balance = E / (k n^2) * sum_e counts[e] * prob_sum[e], which is 1 for an even load.
// Gradient: counts are constants; dl = p (u - sum_e p_e u_e) with u_e = coef * E / (k n^2) * counts[e], and through the gates
// g_j (dg_j - sum_i g_i dg_i) at the chosen experts (normalised), or u raised by dg_j there (not normalised).
//
// A warp takes a token, a lane the experts lane, lane + 32, ... : one pass over the logits, as order-preserving integer keys.  The k-th
// largest of the lanes' maxima is a bound that at least k experts reach and few more do (about ten for top 8 of 256): these go to a
// list in shared memory, a lane takes one of them and counts the others before it.  More than 32 of them (many equal logits), or NaN: k
// rounds of a maximum over the lanes.  (65536 tokens x 256, top 8: rounds in which every lane searches its registers 167 us, rounds that the
// warp searches together 63 us, this 43 us.)  Sums of probabilities stay in registers, counts in shared memory; each CTA leaves one partial row,
// a second launch adds them in a fixed order (no floating-point atomics).  Up to kOneCta tokens one CTA does it all.
// Bound: launches and latency for decode batches (16 tokens x 64: 4.5 us), instruction issue for large ones (0.78 of a warp instruction
// per cycle; the gradient 35 us, 4.0 TB/s).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <algorithm>
#include <cstring>
#include "common/base.h"
#include "common/log.h"
#include "kernels/moe_gate.h"
#include "kernels/pdl.cuh"
#include "kernels/smem_grant.h"

namespace hcclb {

namespace {

constexpr uint32_t kAll = 0xffffffffu;
constexpr int kGateThreads = 512, kMaxBlocks = 296, kGradThreads = 256, kOneThreads = 512, kOneCta = 64;
constexpr int kEndExperts = 8, kEndSlices = 32, kEndThreads = kEndExperts * kEndSlices;

__device__ __forceinline__ float ld_f(const float *p) { return *p; }
__device__ __forceinline__ float ld_f(const __half *p) { return __half2float(*p); }
__device__ __forceinline__ float ld_f(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ void st_f(float *p, float x) { *p = x; }
__device__ __forceinline__ void st_f(__half *p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void st_f(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

// Order of the logits as unsigned integers: 0 is left for "not there", -inf is kInfKey, both zeros are one, NaN is above +inf.
__device__ __forceinline__ uint32_t key_of(float x)
{
    const uint32_t b = __float_as_uint(x + 0.f);
    return x != x ? kAll : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
constexpr uint32_t kInfKey = 0x007fffffu;  // ~bits(-inf)

// e^x from ex2, its smallest results cut to zero
__device__ __forceinline__ float exp_of(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
    return y;
}

// Maximum that is NaN where one of the two is.
__device__ __forceinline__ float max_nan(float x, float y)
{
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(x), "f"(y));
    return m;
}

__device__ __forceinline__ float warp_sum(float x)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(kAll, x, o);
    return x;
}

__device__ __forceinline__ float value_of(uint32_t key)
{
    return __uint_as_float(key == kAll ? 0x7fffffffu : key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

struct GateArgs {
    const void *logits;
    const uint8_t *mask;
    int32_t *idx;
    float *gates;
    float *part_p;                  // [cta][experts]
    int32_t *part_c, *part_n;       // [cta][experts], [cta]
    uint32_t *arrived;              // of the CTAs that add the parts
    float *prob_sum, *balance;
    int32_t *counts, *routed;
    const float *d_gates;
    void *d_logits;
    int64_t tokens, stride;
    int experts, topk, normalize, again;
    float coef;
};

__device__ __forceinline__ float balance_of(float sum, int n, int experts, int topk)
{
    return n ? sum / (float)n / (float)n * ((float)experts / (float)topk) : 0.f;
}

// V: experts of a lane.  Sums of probabilities: in registers up to 32 of them, else in the warp's row of shared memory.
template <int V> constexpr bool kInRegs = V <= 32;
template <int V> constexpr int kGateMost = V <= 32 ? 512 : 128;      // threads of a CTA
template <int V> constexpr int kGateCtas = V <= 8 ? 2 : 1;           // CTAs of that size on an SM
template <class T, int V> __device__ __forceinline__ void load_row(const GateArgs &a, int64_t t, int lane, float (&x)[V])
{
    const T *row = (const T *)a.logits + t * a.stride;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int e = j * 32 + lane;
        x[j] = e < a.experts ? ld_f(row + e) : -INFINITY;
    }
}
// Dynamic shared memory: [warps][32 V] keys, [warps][experts] sums, [experts] counts.
template <class T, int V>
__global__ void __launch_bounds__(kGateMost<V>, kGateCtas<V>) moe_gate_kernel(const __grid_constant__ GateArgs a)
{
    extern __shared__ uint32_t sh[];
    __shared__ int s_n;
    __shared__ float s_b[kOneThreads / 32];
    __shared__ alignas(16) uint2 s_list[kGateMost<V> / 32][36];
    __shared__ alignas(16) uint32_t s_head[kGateMost<V> / 32][32];
    const int E = a.experts, k = a.topk, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = blockDim.x >> 5;
    constexpr int S = V * 32;  // keys of a row: zeros behind the experts
    uint32_t *key = sh + warp * S;
    float *s_p = (float *)(sh + W * S);
    int32_t *s_c = (int32_t *)(sh + W * (S + E));
    if (!kInRegs<V>)
        for (int i = threadIdx.x; i < W * E; i += blockDim.x) s_p[i] = 0.f;
    for (int i = threadIdx.x; i < E; i += blockDim.x) s_c[i] = 0;
    if (threadIdx.x == 0) s_n = 0;
    __syncthreads();
    pdl_trigger();
    pdl_wait();
    if (blockIdx.x == 0 && threadIdx.x == 0 && a.arrived) *a.arrived = 0;
    int mine = 0;  // routed tokens
    float sums[kInRegs<V> ? V : 1] = {};
    for (int64_t t = (int64_t)blockIdx.x * W + warp; t < a.tokens; t += (int64_t)gridDim.x * W) {
        const bool on = !a.mask || a.mask[t];
        float x[V], high = -INFINITY;  // experts outside count as -inf
        load_row<T, V>(a, t, lane, x);
#pragma unroll
        for (int j = 0; j < V; ++j) high = max_nan(high, x[j]);
        uint32_t best = key_of(high);  // largest key of this lane
        const uint32_t top = __reduce_max_sync(kAll, best);
        const bool routed = on && top > kInfKey;
        const float m = value_of(top);
        int sel = -1, slot = lane;  // this lane's choice, if it has one, and its place
        uint32_t sel_key = 0;
        if (routed) {
            // the k-th largest of the lanes' maxima: the least one that fewer than k are above
            uint32_t *heads = s_head[warp];
            __syncwarp();                       // list and maxima of the token before are not read any more
            heads[lane] = best;
            __syncwarp();
            int above = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint4 h = ((const uint4 *)heads)[i];
                above += (h.x > best) + (h.y > best) + (h.z > best) + (h.w > best);
            }
            // as a value: comparisons with it see -0 and 0 as one, and no NaN is there where it is used
            const float least = value_of(max(__reduce_min_sync(kAll, above < k ? best : kAll), kInfKey + 1));
            int own = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) own += x[j] >= least;
            int at = own;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int before = __shfl_up_sync(kAll, at, o);
                if (lane >= o) at += before;
            }
            const int c = __shfl_sync(kAll, at, 31);
            at -= own;
            if (c <= 32 && top != kAll) {
                uint2 *raw = s_list[warp];      // logit and expert, then key and the expert so that lower ones are larger
                raw += at;
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (x[j] >= least) *raw++ = make_uint2(__float_as_uint(x[j]), (uint32_t)(j * 32 + lane));
                __syncwarp();
                uint64_t *list = (uint64_t *)s_list[warp];
                if (lane < c) {
                    const uint2 r = s_list[warp][lane];
                    list[lane] = (uint64_t)key_of(__uint_as_float(r.x)) << 32 | (uint32_t)~r.y;
                }
                if (lane < 4) list[c + lane] = 0;
                __syncwarp();
                if (lane < c) {
                    const uint64_t mine = list[lane];
                    int rank = 0;
                    for (int i = 0; i < c; i += 4)
#pragma unroll
                        for (int u = 0; u < 4; ++u) rank += list[i + u] > mine;
                    slot = rank;
                    sel = rank < k ? (int)~(uint32_t)mine : -1;
                    sel_key = (uint32_t)(mine >> 32);
                }
            } else {
                __syncwarp();
#pragma unroll
                for (int j = 0; j < V; ++j) key[j * 32 + lane] = j * 32 + lane < E ? key_of(x[j]) : 0;
                __syncwarp();
                for (int s = 0; s < k; ++s) {
                    const uint32_t now = __reduce_max_sync(kAll, best);
                    if (now <= kInfKey) break;
                    uint32_t first = kAll;  // the lowest expert with that key
                    if (best == now)
                        for (int e = lane; e < S; e += 32)
                            if (key[e] == now) { first = e; break; }
                    const uint32_t e = __reduce_min_sync(kAll, first);
                    if (first == e) {
                        key[e] = 0;
                        best = 0;
                        for (int i = lane; i < S; i += 32) best = max(best, key[i]);
                    }
                    __syncwarp();
                    if (lane == s) { sel = (int)e; sel_key = now; }
                }
            }
            float z = 0.f;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                x[j] = exp_of(x[j] - m);  // experts outside are -inf
                z += x[j];
            }
            z = warp_sum(z);
            const float inv = __fdividef(1.f, z);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (kInRegs<V>) sums[kInRegs<V> ? j : 0] += x[j] * inv;
                else if (j * 32 + lane < E) s_p[warp * E + j * 32 + lane] += x[j] * inv;
            }
            const float g = sel >= 0 ? exp_of(value_of(sel_key) - m) : 0.f;
            const float whole = a.normalize ? warp_sum(g) : z;
            if (slot < k) a.gates[t * k + slot] = __fdividef(g, whole);
            if (sel >= 0) atomicAdd(&s_c[sel], 1);
            ++mine;
        } else if (lane < k)
            a.gates[t * k + lane] = 0.f;
        if (slot < k) a.idx[t * k + slot] = sel;
    }
    if (kInRegs<V>)
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j * 32 + lane < E) s_p[warp * E + j * 32 + lane] = sums[kInRegs<V> ? j : 0];
    if (lane == 0) atomicAdd(&s_n, mine);
    __syncthreads();
    const bool alone = gridDim.x == 1;
    float sum = 0.f;
    for (int e = threadIdx.x; e < E; e += blockDim.x) {
        float p = 0.f;
        for (int w = 0; w < W; ++w) p += s_p[w * E + e];
        if (alone) {
            a.prob_sum[e] = p;
            a.counts[e] = s_c[e];
            sum += (float)s_c[e] * p;
        } else {
            a.part_p[(int64_t)blockIdx.x * E + e] = p;
            a.part_c[(int64_t)blockIdx.x * E + e] = s_c[e];
        }
    }
    if (!alone) {
        if (threadIdx.x == 0) a.part_n[blockIdx.x] = s_n;
        return;
    }
    sum = warp_sum(sum);
    if (lane == 0) s_b[warp] = sum;
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 1; w < W; ++w) sum += s_b[w];
    *a.routed = s_n;
    *a.balance = balance_of(sum, s_n, E, k);
}

struct EndArgs {
    const float *part_p;
    const int32_t *part_c, *part_n;
    float *prob_sum, *balance;      // prob_sum, counts, routed: null where the parts are the sums
    int32_t *counts, *routed;
    float *shares;                  // [cta] of sum_e counts * prob_sum
    uint32_t *arrived;              // 0 before the launch; null for one CTA
    int parts, experts, topk;
};

// A CTA adds the parts of kEndExperts experts at a time, kEndSlices threads for each; the one that arrives last adds the shares, in
// the order of the CTAs.
__global__ void __launch_bounds__(kEndThreads) moe_gate_end_kernel(const __grid_constant__ EndArgs a)
{
    __shared__ float s_p[kEndSlices][kEndExperts + 1], s_w[kEndThreads / 32];
    __shared__ int s_c[kEndSlices][kEndExperts + 1], s_n[kEndThreads / 32], s_last;
    const int x = threadIdx.x % kEndExperts, slice = threadIdx.x / kEndExperts, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, E = a.experts;
    pdl_trigger();
    pdl_wait();
    float sum = 0.f;
    for (int e0 = blockIdx.x * kEndExperts; e0 < E; e0 += gridDim.x * kEndExperts) {
        const int e = e0 + x;
        float p = 0.f;
        int c = 0;
        if (e < E)
#pragma unroll 8
            for (int i = slice; i < a.parts; i += kEndSlices) { p += a.part_p[(int64_t)i * E + e]; c += a.part_c[(int64_t)i * E + e]; }
        s_p[slice][x] = p;
        s_c[slice][x] = c;
        __syncthreads();
        if (threadIdx.x < kEndExperts && e < E) {
            p = 0.f; c = 0;
#pragma unroll
            for (int q = 0; q < kEndSlices; ++q) { p += s_p[q][x]; c += s_c[q][x]; }
            if (a.counts) { a.counts[e] = c; a.prob_sum[e] = p; }
            sum += (float)c * p;
        }
        __syncthreads();
    }
    if (warp == 0) sum = warp_sum(sum);  // lanes behind the experts hold 0
    if (threadIdx.x == 0) {
        s_last = 1;
        if (a.arrived) {
            a.shares[blockIdx.x] = sum;
            __threadfence();
            s_last = atomicAdd(a.arrived, 1u) == gridDim.x - 1;
            __threadfence();
        }
    }
    __syncthreads();
    if (!s_last) return;
    int n = 0;
    for (int i = threadIdx.x; i < a.parts; i += kEndThreads) n += a.part_n[i];
    n = __reduce_add_sync(kAll, n);
    float all = 0.f;
    if (a.arrived)
        for (int i = threadIdx.x; i < (int)gridDim.x; i += kEndThreads) all += __ldcg(a.shares + i);
    all = warp_sum(all);
    if (lane == 0) { s_n[warp] = n; s_w[warp] = all; }
    __syncthreads();
    if (threadIdx.x) return;
    n = 0; all = 0.f;
    for (int w = 0; w < kEndThreads / 32; ++w) { n += s_n[w]; all += s_w[w]; }
    if (a.routed) *a.routed = n;
    *a.balance = balance_of(a.arrived ? all : sum, n, E, a.topk);
}

// kAgain: slots of a token may name an expert again, as gate() never does.  The first of them stands for all then: how many they are, and
// the sum of their gradients, in the order of the slots.  (A variant of its own: the look for such slots alone costs the others 6 to 15 %.)
__device__ __forceinline__ void merge_slots(int lane, int k, int *sel, float *dg, float *times)
{
    const uint32_t peers = __match_any_sync(kAll, *sel);
    float sum = 0.f;
    for (int j = 0; j < k; ++j) {
        const float v = __shfl_sync(kAll, *dg, j);
        if (peers >> j & 1) sum += v;
    }
    const bool first = *sel >= 0 && __ffs(peers) - 1 == lane;
    *dg = first ? sum : 0.f;
    *times = (float)__popc(peers);
    *sel = first ? *sel : -1;
}

// Dynamic shared memory: [experts] u, [warps][experts] what the gates add at the chosen experts.
template <class T, int V, bool kAgain>
__global__ void __launch_bounds__(kGateMost<V>, kGateCtas<V>) moe_gate_grad_kernel(const __grid_constant__ GateArgs a)
{
    extern __shared__ uint32_t sh[];
    const int E = a.experts, k = a.topk, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = blockDim.x >> 5;
    float *s_u = (float *)sh, *extra = s_u + E + warp * E;
    for (int i = lane; i < E; i += 32) extra[i] = 0.f;
    pdl_trigger();
    pdl_wait();
    const int n = *a.routed;
    const float per = n ? a.coef * ((float)E / (float)k) / (float)n / (float)n : 0.f;
    for (int e = threadIdx.x; e < E; e += blockDim.x) s_u[e] = per * (float)a.counts[e];
    __syncthreads();
    for (int64_t t = (int64_t)blockIdx.x * W + warp; t < a.tokens; t += (int64_t)gridDim.x * W) {
        const T *row = (const T *)a.logits + t * a.stride;
        T *out = (T *)a.d_logits + t * E;
        int sel = lane < k ? a.idx[t * k + lane] : -1;
        if (sel >= E) sel = -1;
        float dg = a.d_gates && sel >= 0 ? a.d_gates[t * k + lane] : 0.f, times = 1.f;
        float x[V], m = -INFINITY;
        load_row<T, V>(a, t, lane, x);
        if (kAgain) merge_slots(lane, k, &sel, &dg, &times);
        const float sel_x = sel >= 0 ? ld_f(row + sel) : -INFINITY;
#pragma unroll
        for (int j = 0; j < V; ++j) m = max_nan(m, x[j]);
        m = value_of(__reduce_max_sync(kAll, key_of(m)));  // NaN where one is
        const bool on = (!a.mask || a.mask[t]) && !(m == -INFINITY);
        if (!on) {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j * 32 + lane < E) st_f(out + j * 32 + lane, 0.f);
            continue;
        }
        float z = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) { x[j] = exp_of(x[j] - m); z += x[j]; }
        z = warp_sum(z);
        const float inv = __fdividef(1.f, z);
        float g = exp_of(sel_x - m);   // 0 where the slot is empty
        const float whole = a.normalize ? warp_sum(kAgain ? g * times : g) : z;
        g = g > 0.f ? __fdividef(g, whole) : g;
        const float gd = warp_sum(g * dg);
        if (sel >= 0) extra[sel] = a.normalize ? g * (dg - (kAgain ? times * gd : gd)) : g * dg;
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int e = j * 32 + lane;
            x[j] *= inv;
            if (e < E) dot += x[j] * s_u[e];
        }
        dot = warp_sum(dot);  // its shuffles also put `extra` before the reads below
        __syncwarp();
        if (!a.normalize) dot += gd;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int e = j * 32 + lane;
            if (e < E) st_f(out + e, fmaf(x[j], s_u[e] - dot, extra[e]));
        }
        __syncwarp();
        if (sel >= 0) extra[sel] = 0.f;
        __syncwarp();
    }
}

// Threads and CTAs of a call.
struct GateGrid { int threads, ctas; };
GateGrid gate_grid(int64_t tokens, int experts, bool grad)
{
    const int most = experts > 1024 ? 128 : kOneThreads;
    if (!grad && tokens <= kOneCta) return {(int)std::min<int64_t>(most, std::max<int64_t>(1, tokens) * 32), 1};
    // a token for every warp, until the CTAs are as many as run at once
    const int threads = std::min(grad ? kGradThreads : tokens >= (int64_t)kMaxBlocks * 16 ? kGateThreads : 128, most), warps = threads / 32;
    return {threads, (int)std::min<int64_t>(grad ? 148 * 4 : kMaxBlocks, (tokens + warps - 1) / warps)};
}

// Dynamic shared memory of a CTA: a row of the experts for each warp and one more, `keys` words of a warp.
constexpr size_t gate_smem(int threads, int experts, int keys) { return ((size_t)(threads / 32) * (keys + experts) + experts) * 4; }
template <int V> constexpr int kGradMost = kGateMost<V> < kGradThreads ? kGateMost<V> : kGradThreads;
static_assert(gate_smem(kGateMost<128>, 4096, 4096) <= 220 * 1024 && gate_smem(kGateMost<32>, 1024, 1024) <= 220 * 1024, "beside what the kernel has of its own");

template <class T, int V> HcclResult run_gate(GateArgs &a, bool grad, void *stream)
{
    const GateGrid g = gate_grid(a.tokens, a.experts, grad);
    const size_t smem = gate_smem(g.threads, a.experts, grad ? 0 : V * 32);
    const void *fn = !grad ? (const void *)moe_gate_kernel<T, V> : a.again ? (const void *)moe_gate_grad_kernel<T, V, true> : (const void *)moe_gate_grad_kernel<T, V, false>;
    if (smem > 32 * 1024) CHK_RET(grant_smem(fn, grad ? gate_smem(kGradMost<V>, V * 32, 0) : gate_smem(kGateMost<V>, V * 32, V * 32), "router"));
    return launch_pdl(fn, dim3((unsigned)g.ctas), (unsigned)g.threads, smem, &a, stream, grad ? "router gradient" : "router");
}

template <class T> HcclResult gate_typed(GateArgs &a, bool grad, void *stream)
{
    const int E = a.experts;
    if (E <= 64) return run_gate<T, 2>(a, grad, stream);
    if (E <= 128) return run_gate<T, 4>(a, grad, stream);
    if (E <= 256) return run_gate<T, 8>(a, grad, stream);
    if (E <= 512) return run_gate<T, 16>(a, grad, stream);
    if (E <= 1024) return run_gate<T, 32>(a, grad, stream);
    if (E <= 2048) return run_gate<T, 64>(a, grad, stream);
    return run_gate<T, 128>(a, grad, stream);
}

HcclResult gate_any(const GateShape &s, GateArgs &a, bool grad, void *stream)
{
    a.tokens = s.tokens; a.stride = s.stride; a.experts = s.experts; a.topk = s.topk; a.normalize = s.normalize; a.again = s.again;
    switch (s.type) {
        case HCCL_DATA_TYPE_FP32: return gate_typed<float>(a, grad, stream);
        case HCCL_DATA_TYPE_FP16: return gate_typed<__half>(a, grad, stream);
        default: return gate_typed<__nv_bfloat16>(a, grad, stream);
    }
}

}  // namespace

// [cta][experts] sums and counts, [cta] tokens, shares of the CTAs that add them, arrivals
int64_t moe_gate_scratch_bytes(int64_t tokens, int32_t experts)
{
    const int ctas = gate_grid(tokens, experts, false).ctas;
    return ctas == 1 ? 0 : (int64_t)ctas * (experts * 8 + 4) + kGateMaxExperts / kEndExperts * 4 + 16;
}

HcclResult moe_gate(const GateShape &s, const void *logits, const uint8_t *mask, int32_t *idx, float *gates, int32_t *counts, float *prob_sum,
                    int32_t *routed, float *balance, void *scratch, void *stream)
{
    GateArgs a;
    memset(&a, 0, sizeof(a));
    a.logits = logits; a.mask = mask; a.idx = idx; a.gates = gates;
    a.prob_sum = prob_sum; a.balance = balance; a.counts = counts; a.routed = routed;
    const int ctas = gate_grid(s.tokens, s.experts, false).ctas;
    if (ctas == 1) return gate_any(s, a, false, stream);
    EndArgs e;
    memset(&e, 0, sizeof(e));
    a.part_p = (float *)scratch;
    a.part_c = (int32_t *)scratch + (int64_t)ctas * s.experts;
    a.part_n = a.part_c + (int64_t)ctas * s.experts;
    e.shares = (float *)(a.part_n + ctas);
    e.arrived = (uint32_t *)(e.shares + kGateMaxExperts / kEndExperts);
    a.arrived = e.arrived;
    CHK_RET(gate_any(s, a, false, stream));
    e.part_p = a.part_p; e.part_c = a.part_c; e.part_n = a.part_n;
    e.prob_sum = prob_sum; e.balance = balance; e.counts = counts; e.routed = routed;
    e.parts = ctas;
    e.experts = s.experts; e.topk = s.topk;
    return launch_pdl((const void *)moe_gate_end_kernel, dim3((unsigned)((s.experts + kEndExperts - 1) / kEndExperts)), kEndThreads, 0, &e, stream, "router (sums)");
}

HcclResult moe_balance(const int32_t *counts, const float *prob_sum, const int32_t *routed, int32_t experts, int32_t topk, float *balance, void *stream)
{
    EndArgs e;
    memset(&e, 0, sizeof(e));
    e.part_p = prob_sum; e.part_c = counts; e.part_n = routed; e.balance = balance;
    e.parts = 1; e.experts = experts; e.topk = topk;
    return launch_pdl((const void *)moe_gate_end_kernel, dim3(1), kEndThreads, 0, &e, stream, "router (balance)");
}

HcclResult moe_gate_grad(const GateShape &s, const void *logits, const int32_t *idx, const float *d_gates, const int32_t *counts, const int32_t *routed,
                         const uint8_t *mask, float coef, void *d_logits, void *stream)
{
    if (!s.tokens) return HCCL_SUCCESS;
    GateArgs a;
    memset(&a, 0, sizeof(a));
    a.logits = logits; a.mask = mask; a.idx = (int32_t *)idx; a.d_gates = d_gates; a.counts = (int32_t *)counts; a.routed = (int32_t *)routed;
    a.coef = coef; a.d_logits = d_logits;
    return gate_any(s, a, true, stream);
}

}  // namespace hcclb
