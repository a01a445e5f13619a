// Router of a mixture-of-experts layer.  For each token: p = softmax(logits), the top-k experts by logit (equal logits: the lowest
// expert; -inf is never chosen, its slot gets expert -1 and gate 0), gates = p of the chosen ones, divided by their sum where they
// are normalised.  Over the tokens that are routed (n of them: not masked, not all -inf): counts[e] pairs of expert e,
// prob_sum[e] = sum of p[.,e], balance = E / (k n^2) * sum_e counts[e] * prob_sum[e], which is 1 for an even load.
// Gradient: counts are constants; dl = p (u - sum_e p_e u_e) with u_e = coef * E / (k n^2) * counts[e], and through the gates
// g_j (dg_j - sum_i g_i dg_i) at the chosen experts (normalised), or u raised by dg_j there (not normalised).
//
// A warp takes a token, a lane the experts lane, lane + 32, ... in registers: one pass over the logits; a round of the top-k is a
// maximum over the lanes of an order-preserving integer key.  Sums of probabilities and counts stay in the warp and in shared
// memory, each CTA leaves one partial row, and one cluster adds them in a fixed order (no floating-point atomics).
// Bound: launches and latency for decode batches, instruction issue of the top-k rounds for large ones.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <algorithm>
#include <cstring>
#include "common/base.h"
#include "common/log.h"
#include "kernels/moe_gate.h"
#include "kernels/pdl.cuh"

namespace hcclb {

namespace {

constexpr uint32_t kAll = 0xffffffffu;
constexpr int kGateThreads = 256, kMaxBlocks = 296, kEndThreads = 1024, kEndCluster = 8;

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
    if (x != x) return kAll;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t kInfKey = 0x007fffffu;  // ~bits(-inf)

__device__ __forceinline__ float warp_sum(float x)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(kAll, x, o);
    return x;
}

struct GateArgs {
    const void *logits;
    const uint8_t *mask;
    int32_t *idx;
    float *gates;
    float *part_p;                  // [cta][experts]
    int32_t *part_c, *part_n;       // [cta][experts], [cta]
    const int32_t *counts, *routed;
    const float *d_gates;
    void *d_logits;
    int64_t tokens, stride;
    int experts, topk, normalize;
    float coef;
};

// V: experts of a lane; kWarps x experts floats and experts words of shared memory
template <int V> constexpr int kGateWarps = V > 32 ? 4 : kGateThreads / 32;

template <class T, int V>
__global__ void __launch_bounds__(kGateWarps<V> * 32) moe_gate_kernel(const __grid_constant__ GateArgs a)
{
    constexpr int W = kGateWarps<V>;
    extern __shared__ float sh[];
    __shared__ int s_n;
    const int E = a.experts, k = a.topk, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float *s_p = sh + warp * E;
    int32_t *s_c = (int32_t *)(sh + W * E);
    for (int i = threadIdx.x; i < W * E; i += W * 32) sh[i] = 0.f;
    for (int i = threadIdx.x; i < E; i += W * 32) s_c[i] = 0;
    if (threadIdx.x == 0) s_n = 0;
    __syncthreads();
    pdl_trigger();
    pdl_wait();
    int mine = 0;  // routed tokens
    for (int64_t t = (int64_t)blockIdx.x * W + warp; t < a.tokens; t += (int64_t)gridDim.x * W) {
        const T *row = (const T *)a.logits + t * a.stride;
        const bool on = !a.mask || a.mask[t];
        float x[V];
        uint32_t best = 0, where = 0;  // of this lane's experts: largest key, its place
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int e = j * 32 + lane;
            x[j] = e < E ? ld_f(row + e) : -INFINITY;
            const uint32_t q = e < E ? key_of(x[j]) : 0;
            if (q > best) { best = q; where = j; }
        }
        uint32_t top = __reduce_max_sync(kAll, best);
        const bool routed = on && top > kInfKey;
        float m = top == kAll ? __uint_as_float(0x7fffffffu) : 0.f;  // NaN in the row
        if (top != kAll) m = __uint_as_float(top & 0x80000000u ? top & 0x7fffffffu : ~top);
        int sel = -1;           // of slot `lane`
        float sel_x = -INFINITY;
        if (routed) {
            uint32_t taken[(V + 31) / 32];
#pragma unroll
            for (int j = 0; j < (V + 31) / 32; ++j) taken[j] = 0;
            for (int s = 0; s < k; ++s) {
                if (s) top = __reduce_max_sync(kAll, best);
                if (top <= kInfKey) break;
                const uint32_t e = __reduce_min_sync(kAll, best == top ? where * 32 + lane : kAll);
                if (lane == s) {
                    sel = (int)e;
                    sel_x = top == kAll ? __uint_as_float(0x7fffffffu) : __uint_as_float(top & 0x80000000u ? top & 0x7fffffffu : ~top);
                }
                if ((e & 31) == (uint32_t)lane) {
                    if (V > 32) taken[(e >> 5) >> 5] |= 1u << ((e >> 5) & 31);
                    else taken[0] |= 1u << (e >> 5);
                    best = 0;
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const uint32_t q = j * 32 + lane < E && !(taken[j / 32] >> (j & 31) & 1) ? key_of(x[j]) : 0;
                        if (q > best) { best = q; where = j; }
                    }
                }
            }
            float z = 0.f;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                x[j] = __expf(x[j] - m);  // experts outside are -inf
                z += x[j];
            }
            z = warp_sum(z);
            const float inv = 1.f / z;
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j * 32 + lane < E) s_p[j * 32 + lane] += x[j] * inv;
            const float g = sel >= 0 ? __expf(sel_x - m) : 0.f;
            const float whole = a.normalize ? warp_sum(g) : z;
            if (lane < k) a.gates[t * k + lane] = g / whole;
            if (sel >= 0) atomicAdd(&s_c[sel], 1);
            ++mine;
        } else if (lane < k)
            a.gates[t * k + lane] = 0.f;
        if (lane < k) a.idx[t * k + lane] = sel;
    }
    if (lane == 0) atomicAdd(&s_n, mine);
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += W * 32) {
        float p = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) p += sh[w * E + e];
        a.part_p[(int64_t)blockIdx.x * E + e] = p;
        a.part_c[(int64_t)blockIdx.x * E + e] = s_c[e];
    }
    if (threadIdx.x == 0) a.part_n[blockIdx.x] = s_n;
}

struct EndArgs {
    const float *part_p;
    const int32_t *part_c, *part_n;
    float *prob_sum, *balance;      // prob_sum, counts, routed: null where the parts are the sums
    int32_t *counts, *routed;
    int parts, experts, topk;
};

__device__ __forceinline__ float load_cluster_f(const float *own, int cta)
{
    uint32_t at;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(own)), "r"(cta));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

// One cluster: a warp's lanes hold 32 consecutive experts, the warps of such a group share the parts.
__global__ void __launch_bounds__(kEndThreads) moe_gate_end_kernel(const __grid_constant__ EndArgs a)
{
    __shared__ float s_p[32][33], s_b;
    __shared__ int s_c[32][33], s_n[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, E = a.experts, cta = blockIdx.x;
    pdl_trigger();
    pdl_wait();
    int n = 0;
    for (int i = threadIdx.x; i < a.parts; i += kEndThreads) n += a.part_n[i];
    n = __reduce_add_sync(kAll, n);
    if (lane == 0) s_n[warp] = n;
    float sum = 0.f;  // thread's share of sum_e counts * prob_sum
    for (int e0 = cta * 32; e0 < E; e0 += kEndCluster * 32) {
        const int e = e0 + lane;
        float p = 0.f;
        int c = 0;
        if (e < E)
#pragma unroll 4
            for (int i = warp; i < a.parts; i += kEndThreads / 32) { p += a.part_p[(int64_t)i * E + e]; c += a.part_c[(int64_t)i * E + e]; }
        s_p[warp][lane] = p;
        s_c[warp][lane] = c;
        __syncthreads();
        if (warp == 0) {
            p = 0.f; c = 0;
#pragma unroll
            for (int w = 0; w < kEndThreads / 32; ++w) { p += s_p[w][lane]; c += s_c[w][lane]; }
            if (e < E) {
                if (a.counts) { a.counts[e] = c; a.prob_sum[e] = p; }
                sum += (float)c * p;
            }
        }
        __syncthreads();
    }
    if (warp == 0) {
        sum = warp_sum(sum);
        if (lane == 0) s_b = sum;
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (cta == 0 && threadIdx.x == 0) {
        float b = 0.f;
        for (int q = 0; q < kEndCluster; ++q) b += load_cluster_f(&s_b, q);
        int all = 0;
        for (int w = 0; w < kEndThreads / 32; ++w) all += s_n[w];
        if (a.routed) *a.routed = all;
        // n^2 leaves 32 bits for a few thousand million tokens only, but counts * p / n / n keeps its digits either way
        *a.balance = all ? b / (float)all / (float)all * ((float)E / (float)a.topk) : 0.f;
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <class T, int V>
__global__ void __launch_bounds__(kGateWarps<V> * 32) moe_gate_grad_kernel(const __grid_constant__ GateArgs a)
{
    constexpr int W = kGateWarps<V>;
    extern __shared__ float s_u[];
    const int E = a.experts, k = a.topk, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_trigger();
    pdl_wait();
    const int n = *a.routed;
    const float per = n ? a.coef * ((float)E / (float)k) / (float)n / (float)n : 0.f;
    for (int e = threadIdx.x; e < E; e += W * 32) s_u[e] = per * (float)a.counts[e];
    __syncthreads();
    for (int64_t t = (int64_t)blockIdx.x * W + warp; t < a.tokens; t += (int64_t)gridDim.x * W) {
        const T *row = (const T *)a.logits + t * a.stride;
        T *out = (T *)a.d_logits + t * E;
        const int sel = lane < k ? a.idx[t * k + lane] : -1;
        const float dg = a.d_gates && sel >= 0 && sel < E ? a.d_gates[t * k + lane] : 0.f;
        float x[V], m = -INFINITY;
        bool nan = false;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int e = j * 32 + lane;
            x[j] = e < E ? ld_f(row + e) : -INFINITY;
            m = fmaxf(m, x[j]);
            nan = nan || x[j] != x[j];
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kAll, m, o));
        const bool on = (!a.mask || a.mask[t]) && (m > -INFINITY || __any_sync(kAll, nan));
        if (!on) {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j * 32 + lane < E) st_f(out + j * 32 + lane, 0.f);
            continue;
        }
        float sel_x = -INFINITY;
        if (sel >= 0 && sel < E) sel_x = ld_f(row + sel);
        float z = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) { x[j] = __expf(x[j] - m); z += x[j]; }
        z = warp_sum(z);
        const float inv = 1.f / z;
        float g = __expf(sel_x - m);   // 0 where the slot is empty
        const float whole = a.normalize ? warp_sum(g) : z;
        g = g > 0.f ? g / whole : g;
        const float gd = warp_sum(g * dg);
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int e = j * 32 + lane;
            x[j] *= inv;
            if (e < E) dot += x[j] * s_u[e];
        }
        dot = warp_sum(dot);
        if (!a.normalize) dot += gd;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int e = j * 32 + lane;
            if (e < E) x[j] *= s_u[e] - dot;
        }
        const float add = a.normalize ? g * (dg - gd) : g * dg;  // at the chosen expert
        for (int s = 0; s < k; ++s) {
            const int e = __shfl_sync(kAll, sel, s);
            const float v = __shfl_sync(kAll, add, s);
            if (e >= 0 && (e & 31) == lane)
#pragma unroll
                for (int j = 0; j < V; ++j) x[j] += j == e >> 5 ? v : 0.f;
        }
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j * 32 + lane < E) st_f(out + j * 32 + lane, x[j]);
    }
}

int gate_blocks(int64_t tokens, int warps) { return (int)std::min<int64_t>(kMaxBlocks, std::max<int64_t>(1, (tokens + warps - 1) / warps)); }

template <class T, int V> HcclResult run_gate(GateArgs &a, bool grad, void *stream)
{
    constexpr int W = kGateWarps<V>;
    const size_t smem = grad ? (size_t)a.experts * 4 : (size_t)(W + 1) * a.experts * 4;
    const void *fn = grad ? (const void *)moe_gate_grad_kernel<T, V> : (const void *)moe_gate_kernel<T, V>;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        CHK_RET_LOG(e != cudaSuccess, HCCL_E_RUNTIME, "router set-up failed: %s", cudaGetErrorString(e));
    }
    const unsigned blocks = grad ? (unsigned)std::min<int64_t>(148 * 8, (a.tokens + W - 1) / W) : (unsigned)gate_blocks(a.tokens, W);
    return launch_pdl(fn, dim3(blocks), W * 32, smem, &a, stream, grad ? "router gradient" : "router");
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
    a.tokens = s.tokens; a.stride = s.stride; a.experts = s.experts; a.topk = s.topk; a.normalize = s.normalize;
    switch (s.type) {
        case HCCL_DATA_TYPE_FP32: return gate_typed<float>(a, grad, stream);
        case HCCL_DATA_TYPE_FP16: return gate_typed<__half>(a, grad, stream);
        default: return gate_typed<__nv_bfloat16>(a, grad, stream);
    }
}

}  // namespace

int64_t moe_gate_scratch_bytes(int64_t, int32_t experts) { return (int64_t)kMaxBlocks * (experts * 8 + 4); }

HcclResult moe_gate(const GateShape &s, const void *logits, const uint8_t *mask, int32_t *idx, float *gates, int32_t *counts, float *prob_sum,
                    int32_t *routed, float *balance, void *scratch, void *stream)
{
    GateArgs a;
    memset(&a, 0, sizeof(a));
    a.logits = logits; a.mask = mask; a.idx = idx; a.gates = gates;
    a.part_p = (float *)scratch;
    a.part_c = (int32_t *)scratch + (int64_t)kMaxBlocks * s.experts;
    a.part_n = a.part_c + (int64_t)kMaxBlocks * s.experts;
    CHK_RET(gate_any(s, a, false, stream));
    EndArgs e;
    memset(&e, 0, sizeof(e));
    e.part_p = a.part_p; e.part_c = a.part_c; e.part_n = a.part_n;
    e.prob_sum = prob_sum; e.balance = balance; e.counts = counts; e.routed = routed;
    e.parts = gate_blocks(s.tokens, s.experts > 1024 ? 4 : kGateThreads / 32);
    e.experts = s.experts; e.topk = s.topk;
    return launch_pdl((const void *)moe_gate_end_kernel, dim3(kEndCluster), kEndThreads, 0, &e, stream, "router (sums)", kEndCluster);
}

HcclResult moe_balance(const int32_t *counts, const float *prob_sum, const int32_t *routed, int32_t experts, int32_t topk, float *balance, void *stream)
{
    EndArgs e;
    memset(&e, 0, sizeof(e));
    e.part_p = prob_sum; e.part_c = counts; e.part_n = routed; e.balance = balance;
    e.parts = 1; e.experts = experts; e.topk = topk;
    return launch_pdl((const void *)moe_gate_end_kernel, dim3(kEndCluster), kEndThreads, 0, &e, stream, "router (balance)", kEndCluster);
}

HcclResult moe_gate_grad(const GateShape &s, const void *logits, const int32_t *idx, const float *d_gates, const int32_t *counts, const int32_t *routed,
                         const uint8_t *mask, float coef, void *d_logits, void *stream)
{
    if (!s.tokens) return HCCL_SUCCESS;
    GateArgs a;
    memset(&a, 0, sizeof(a));
    a.logits = logits; a.mask = mask; a.idx = (int32_t *)idx; a.d_gates = d_gates; a.counts = counts; a.routed = routed; a.coef = coef; a.d_logits = d_logits;
    return gate_any(s, a, true, stream);
}

}  // namespace hcclb
