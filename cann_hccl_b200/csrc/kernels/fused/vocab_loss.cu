// Linear layer and softmax cross entropy over the vocabulary, with gradients, without keeping the logits:
//   s = x W^T;  lse_t = log sum_v exp s_tv;  loss_t = lse_t - s_t,y;  d_tv = q_t (exp(s_tv - lse_t) - [v = y]);  dx = a d W;  dW = a d^T x
// (q: weight of the token; a: scale, divided by the sum of the weights for a mean; applied to the fp32 sums, so that the d of a target
// far from sure is -q and not -q a: an ordinary weight of one is not rounded at all.  Other weights are, with d, by half a step of bf16: dx and dW
// are 2.4e-3 off in their 2-norm then, 1.9e-3 without.  d without q, with q in dx's epilogue and in the x that dW reads, would spare dx that
// rounding and round dW's operands twice)
//
// x        with gradients (or where rows do not start on 128-byte lines) the tokens' rows are copied, those of tokens that do not count as
//          zeros: 0 x inf is not 0.
//
// scores   tcgen05 product of a chunk of tokens with all tiles of the vocabulary.  The epilogue takes a row's half tile from TMEM,
//          leaves its maximum m and sum of exp(s - m) (fp32) and, for gradients, 2^15 exp(s - m) in fp16: relative to the half
//          tile's own maximum 11 bits hold every probability down to 2^-29 of it, so that the one rounding that counts
//          is the later one of d to bf16.  Logits are never stored, and nothing is computed twice (6 T V H operations in all;
//          a second product in place of the exponentials would make it 8).
// rows     lse and loss of a token from its half tiles.  The target's logit is summed once more in fp32 FMAs of short chains and put in the
//          place of the tensor cores' one in lse too: their running sum cuts digits off instead of rounding, and a loss near zero is
//          the difference of two logits that would carry that.  The other logits keep the cut: sums that grow evenly come out nearer
//          to zero by about 1e-9 of themselves for each element of the depth (2.6e-7, 1.05e-6, 4.1e-6 for 256, 1024, 4096), with one sign, so
//          that a mean does not average it out.  So the depth is taken in parts of 1024 to 2047 elements (512 to 1023 where a single CTA
//          has the rows), whose sums the epilogue adds in fp32: means of losses at H = 4096 are 1.3e-7 low around 10, 2.7e-6 around
//          0.1 (5.8e-7 and 7.3e-6 in one part).
// d        exponentials to d in place (bf16), rescaled by exp(m - lse); the target's column is q expm1(-loss), and the loss is formed of the
//          largest logit, the target's and log of the sum beside it, never of lse: rounded to fp32 that would be off by half a step of
//          a logit, more than a sure guess has (1e-6 at logits of 20).  Tokens that do not count become rows of zeros.
//          In a whole step with gradients rows and d are one launch, a CTA for each token.
// dx, dW   tcgen05 products that read W, d and x as they lie: an operand whose depth is not its contiguous side goes to the tensor
//          cores MN-major (boxes of 64 elements x 64 deep).  dx with few tiles is cut along the vocabulary into fp32 shares that a
//          last launch adds in order; dW over several chunks is summed in fp32.
//
// One persistent CTA per SM: warp 0 TMA producer (128-byte swizzle, never multicast), warp 1 MMA issuer into one of two TMEM
// accumulators, warps 2-9 epilogue of the other.  More than 128 rows: clusters of two CTAs on 256 rows (cta_group::2).
// Bound: tensor cores under the power cap (8192 x 128256 x 4096: scores 5.5, dx 5.4, dW 5.5 ms, 1.57 PFLOP/s alone; rows and d 0.69 ms, 6.5
// TB/s; a step 19.4 to 23 ms by box and by what ran before), HBM for few tokens (7 x 32000 x 4096: 47 us) and, with gradients, for small
// hidden sizes, since each logit moves ten bytes (1024 x 160000 x 256: scores 118, rows and d 123, dx 74, dW 73 us).
// A wait that runs out makes what it was for NaN.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <algorithm>
#include <cstring>
#include <mutex>
#include "common/log.h"
#include "kernels/fused/tc05.cuh"
#include "kernels/fused/tensor_map.h"
#include "kernels/fused/vocab_loss.h"
#include "kernels/pdl.cuh"

namespace hcclb {

namespace {
using namespace tc05;

enum Mode : int { SCORES = 0, DX = 1, DW = 2 };
constexpr int kThreads = 320, kEpiWarps = 8;
constexpr uint32_t kABytes = BM * BK * 2, kStageSpace = 7 * 32768;  // seven stages of a pair
constexpr uint32_t kTmemCols = 512;
// k_iters of a part of the scores' depth, the least.  Parts as short as these cost 0.7 % at most; of pairs, half as long ones cost the step up
// to 7 % (1024 x 128256 x 2048), since the epilogue has half of the time for its own work while the next parts are multiplied.
template <bool kPair> constexpr int kPartLeast = kPair ? 16 : 8;
constexpr int kMaxStages = 8, kMaxCols = BN;
constexpr uint32_t kChunkBytes = BK * 128;         // MN-major: 64 elements x 64 deep
constexpr float kExpBits = 15.f, kExpScale = 1.f / 32768.f, kLog2e = 1.4426950408889634f;

struct alignas(64) LossGemm {
    CUtensorMap tmA, tmB;
    int M, N;                        // rows and columns of the result
    int cols, um_tiles, n_tiles, panel;
    int k_iters, split;              // split: shares along the depth (DX)
    int part;                        // k_iters of a part of the depth (scores in parts)
    int units, stages;
    uint32_t stage_bytes, a_bytes, idesc;  // of a stage, of A in it
    // scores
    float2 *stats;                   // [row][2 * n_tiles]: maximum, sum of exp(s - maximum)
    float *target;                   // [row]
    __half *e;                       // [row][ld], of which `width` columns are written; may be null
    const void *y;
    int64_t first, ignore;
    int wide_y;
    // dx, dW
    __nv_bfloat16 *out;
    float *sum;                      // shares of dx: [share][row][N]
    int kind;                        // VocabLossOut
    int64_t ld, width;
    const float *total;              // the sums are multiplied by scale / *total (null: scale; a total of 0: 0)
    float scale;
};

struct LossShared {
    alignas(1024) uint8_t tiles[kStageSpace];
    alignas(8) uint64_t full_bar[kMaxStages];
    uint64_t empty_bar[kMaxStages];
    uint64_t tmem_full[2], tmem_empty[2];
    uint32_t tmem_base, fail;
};
constexpr size_t kSmemBytes = sizeof(LossShared) + 1024;
static_assert(kSmemBytes <= 227 * 1024, "one CTA per SM");

// Pairs turn dW around in the end of the stages' space, 32 rows x 128 bytes of a warp at a time, so that a store covers whole 128-byte
// lines: a lane's own row in 32-byte stores moves 16 bytes per cycle and SM (1 token, 128256 x 4096: 252 us, 214 this way; as boxes
// stored by the TMA 335 us).  The exponentials leave in 32-byte stores all the same: beside their 128 values a lane has no
// registers left for it (1024 tokens, 160000 x 256: 218 against 117 us).
constexpr uint32_t kTurnWarp = 32 * 128, kTurnSpace = kEpiWarps * kTurnWarp;
template <int MODE, bool kPair> constexpr bool kTurn = kPair && MODE == DW;

// MN-major operand, 128-byte swizzle: 64 elements side by side, 8 deep in 1024 bytes, the next 64 elements kChunkBytes on.
__device__ __forceinline__ uint64_t make_desc_mn(const void *ptr)
{
    uint64_t d = 0;
    d |= (uint64_t)((smem_u32(ptr) & 0x3FFFF) >> 4);
    d |= (uint64_t)(kChunkBytes >> 4) << 16;           // leading dimension: from 64 elements to the next
    d |= (uint64_t)(1024 >> 4) << 32;                  // stride dimension: from 8 deep to the next
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
constexpr uint32_t kStepK = 2, kStepMn = (UMMA_K * 128) >> 4;  // 16 deep further, in 16-byte units

struct Tile { int um, nt, share; };
__device__ __forceinline__ Tile tile_at(const LossGemm &P, int t)
{
    Tile w;
    const int tiles = P.um_tiles * P.n_tiles;
    w.share = t / tiles;
    t -= w.share * tiles;
    const int per = P.um_tiles * P.panel, pn = t / per, n0 = pn * P.panel, width = min(P.panel, P.n_tiles - n0), r = t - pn * per;
    w.um = r / width;
    w.nt = n0 + r - w.um * width;
    return w;
}

__device__ __forceinline__ void st_v8(void *p, const uint32_t (&v)[8])
{
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t cluster_addr)
{
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// One of a lane's registers by its number; as a choice in C the registers would become an array in local memory.
__device__ __forceinline__ void store_if(float *p, float v, bool yes)
{
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %2, 0;\n @p st.global.f32 [%0], %1;\n}" ::"l"(p), "f"(v), "r"((int)yes) : "memory");
}
__device__ __forceinline__ float exp2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ int64_t target_of(const void *y, int wide, int64_t t) { return wide ? ((const int64_t *)y)[t] : (int64_t)((const int32_t *)y)[t]; }

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float *v)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]),
                   "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]) : "memory");
}

// Half a tile's columns of a row stay in registers: the accumulator is free again before any of them is worked on.
constexpr int kHalf = kMaxCols / 2;
__device__ __forceinline__ void tmem_half(uint32_t addr, float (&v)[kHalf])
{
    uint32_t r[kHalf / 32][32];
#pragma unroll
    for (int q = 0; q < kHalf / 32; ++q) tmem_ld32(addr + q * 32, r[q]);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < kHalf; ++i) v[i] = __uint_as_float(r[i / 32][i % 32]);
}

__device__ __forceinline__ void tmem_64(uint32_t addr, float (&v)[64])
{
    uint32_t r[2][32];
    tmem_ld32(addr, r[0]);
    tmem_ld32(addr + 32, r[1]);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i / 32][i % 32]);
}

// tmem_half in steps of 32 columns, for single CTAs: each of them has a few tiles at most, the code above would come from memory once for
// every tile (7 tokens x 32000 x 4096: 55 against 50 us), and memory sets the pace anyway.
__device__ __forceinline__ void tmem_32(uint32_t addr, int left, float (&v)[32])
{
    uint32_t r[32];
    tmem_ld32(addr, r);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = i < left ? __uint_as_float(r[i]) : -INFINITY;
}
template <int C> __device__ __forceinline__ void put_exp(__half *e, const float (&v)[C], int room)
{
#pragma unroll
    for (int c = 0; c < C; c += 16)
        if (c < room) {
            uint32_t o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const __half2 h = __floats2half2_rn(v[c + 2 * i], v[c + 2 * i + 1]);
                o[i] = *(const uint32_t *)&h;
            }
            st_v8(e + c, o);
        }
}

// v: eight 16-byte pieces of the lane's row; to: the first piece of the warp's first row; rows, pieces: that exist.
__device__ __forceinline__ void turn_store(uint8_t *box, const uint4 (&v)[8], int lane, uint8_t *to, int64_t row_bytes, int rows, int pieces)
{
    __syncwarp();  // what was here has been read
#pragma unroll
    for (int c = 0; c < 8; ++c) *(uint4 *)(box + lane * 128 + (c ^ (lane & 7)) * 16) = v[c];
    __syncwarp();
    const int c = lane & 7;
    if (c < pieces)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + (lane >> 3);
            if (r < rows) *(uint4 *)(to + r * row_bytes + c * 16) = *(const uint4 *)(box + r * 128 + (c ^ (r & 7)) * 16);
        }
}

// The same for fp32: v: 32 columns of the lane's row; sum, out: the warp's first row and column; rows, cols: that exist.  What is added to
// is read a whole line at a time too (512 tokens x 128256 x 4096 2.2 ms; with rows added to in 16-byte pieces of a lane 3.3 ms).
__device__ __forceinline__ void turn_sum(uint8_t *box, const float *v, int lane, int kind, float *sum, __nv_bfloat16 *out, int64_t ld, int rows, int cols)
{
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 8; ++c) *(float4 *)(box + lane * 128 + (c ^ (lane & 7)) * 16) = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
    __syncwarp();
    const int c = lane & 7;
    if (c * 4 >= cols) return;
    float4 g[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = i * 4 + (lane >> 3);
        g[i] = kind != VL_F32 && r < rows ? __ldcs((const float4 *)(sum + r * ld + c * 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = i * 4 + (lane >> 3);
        if (r >= rows) continue;
        const float4 x = *(const float4 *)(box + r * 128 + (c ^ (r & 7)) * 16);
        const float4 y = make_float4(g[i].x + x.x, g[i].y + x.y, g[i].z + x.z, g[i].w + x.w);
        if (kind == VL_ADD_BF16)
            *(uint2 *)(out + r * ld + c * 4) = make_uint2(pack_bf16(__float_as_uint(y.x), __float_as_uint(y.y)), pack_bf16(__float_as_uint(y.z), __float_as_uint(y.w)));
        else
            __stcs((float4 *)(sum + r * ld + c * 4), y);
    }
}

// kParts (scores): the accumulators take turns with the parts of a tile's depth, whose sums the epilogue adds.
template <int MODE, bool kPair, bool kParts>
__global__ void __launch_bounds__(kThreads, 1) vocab_loss_gemm(const __grid_constant__ LossGemm P)
{
    static_assert(!kParts || MODE == SCORES);
    extern __shared__ uint8_t smem_raw[];
    LossShared &S = *(LossShared *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    constexpr int kCtas = kPair ? 2 : 1;
    constexpr bool kMnA = MODE == DW, kMnB = MODE != SCORES;
    const uint32_t stages = (uint32_t)P.stages, stage_bytes = P.stage_bytes, a_bytes = P.a_bytes;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t cta_r = kPair ? cluster_ctarank() : 0u;
    const int unit = (int)blockIdx.x / kCtas, total = P.um_tiles * P.n_tiles * P.split;
    volatile uint32_t *fail = &S.fail;

    pdl_trigger();
    if (threadIdx.x == 0) {
        S.fail = 0;
        for (int i = 0; i < kMaxStages; ++i) { mbar_init(&S.full_bar[i], 1); mbar_init(&S.empty_bar[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&S.tmem_full[i], 1); mbar_init(&S.tmem_empty[i], kPair && kParts ? 2 * kEpiWarps : kEpiWarps); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetch_tensormap(&P.tmA);
        prefetch_tensormap(&P.tmB);
    }
    if (warp == 1) {
        if (kPair) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&S.tmem_base)), "r"(kTmemCols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&S.tmem_base)), "r"(kTmemCols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if (kPair) cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = S.tmem_base;
    pdl_wait();

    if (warp == 0) {
        // ------------------------------------------------------------------ TMA producer
        if (elect_one()) {
            uint32_t s = 0, ph = 0;
            const int bcols = P.cols / kCtas;
            for (int t = unit; t < total && !*fail; t += P.units) {
                const Tile w = tile_at(P, t);
                const int arow = (w.um * kCtas + (int)cta_r) * BM, brow = w.nt * P.cols + (int)cta_r * bcols;
                const int k0 = (int)((int64_t)P.k_iters * w.share / P.split), k1 = (int)((int64_t)P.k_iters * (w.share + 1) / P.split);
                for (int k = k0; k < k1; ++k) {
                    if (!mbar_wait_t<kPair>(&S.empty_bar[s], ph ^ 1, fail)) break;
                    uint8_t *sa = S.tiles + (size_t)s * stage_bytes, *sb = sa + a_bytes;
                    uint32_t full = smem_u32(&S.full_bar[s]);
                    if (kPair) {  // the bytes of both CTAs' loads are counted on the leader's barrier
                        if (cta_r == 0) mbar_expect_tx(&S.full_bar[s], 2 * stage_bytes);
                        full = mapa_u32(full, 0);
                    } else
                        mbar_expect_tx(&S.full_bar[s], stage_bytes);
                    auto load = [&](uint8_t *dst, const CUtensorMap *map, int x, int y) {
                        if (kPair) tma_load_2d_pair(dst, map, full, x, y); else tma_load_2d(dst, map, &S.full_bar[s], x, y);
                    };
                    if (kMnA) {
#pragma unroll
                        for (int c = 0; c < BM / 64; ++c) load(sa + c * kChunkBytes, &P.tmA, arow + c * 64, k * BK);
                    } else
                        load(sa, &P.tmA, k * BK, arow);
                    if (kMnB) {
                        for (int c = 0; c < bcols / 64; ++c) load(sb + c * kChunkBytes, &P.tmB, brow + c * 64, k * BK);
                    } else
                        load(sb, &P.tmB, k * BK, brow);
                    if (++s == stages) { s = 0; ph ^= 1; }
                }
            }
        }
        if (*fail)  // loads in flight land before the CTA lets go of its shared memory
            for (int i = 0; i < 200; ++i) __nanosleep(1000);
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA issuer (pair: the leader, for both CTAs)
        if (cta_r == 0 && elect_one()) {
            uint32_t s = 0, ph = 0, n = 0;
            for (int t = unit; t < total && !*fail; t += P.units) {
                const Tile w = tile_at(P, t);
                const int k0 = (int)((int64_t)P.k_iters * w.share / P.split), k1 = (int)((int64_t)P.k_iters * (w.share + 1) / P.split);
                const int part = kParts ? P.part : k1 - k0;
                for (int p0 = k0; p0 < k1; p0 += part, ++n) {
                    const int p1 = kParts ? min(p0 + part, k1) : k1;
                    const uint32_t buf = n & 1, use = n >> 1, d = tmem_base + buf * kMaxCols;
                    if (!mbar_wait_t<kPair>(&S.tmem_empty[buf], (use & 1) ^ 1, fail)) break;
                    tc_fence_after();
                    for (int k = p0; k < p1; ++k) {
                        if (!mbar_wait_t<kPair>(&S.full_bar[s], ph, fail)) break;
                        tc_fence_after();
                        const uint8_t *sa = S.tiles + (size_t)s * stage_bytes, *sb = sa + a_bytes;
                        const uint64_t da = kMnA ? make_desc_mn(sa) : make_smem_desc(sa), db = kMnB ? make_desc_mn(sb) : make_smem_desc(sb);
#pragma unroll
                        for (int kk = 0; kk < BK / UMMA_K; ++kk) {
                            const uint64_t a = da + (uint64_t)(kk * (kMnA ? kStepMn : kStepK)), b = db + (uint64_t)(kk * (kMnB ? kStepMn : kStepK));
                            if (kPair) umma_pair(d, a, b, k != p0 || kk != 0, P.idesc); else umma(d, a, b, k != p0 || kk != 0, P.idesc);
                        }
                        if (kPair) umma_commit_pair(&S.empty_bar[s]); else umma_commit(&S.empty_bar[s]);
                        if (++s == stages) { s = 0; ph ^= 1; }
                    }
                    if (kPair) umma_commit_pair(&S.tmem_full[buf]); else umma_commit(&S.tmem_full[buf]);
                    if (*fail) break;
                }
            }
        }
    } else {
        // ------------------------------------------------------------------ epilogue: a warp reaches its TMEM lane quarter.  Single: the two
        // warps of a quarter take half of the columns each.  Pair: they take tiles in turn, one accumulator each, so that one waits for
        // TMEM while the other stores.  In parts: half of the columns each, since a lane has registers for the sums of so many.
        constexpr bool kTurns = kPair && !kParts;
        const int q4 = warp & 3, group = (warp - 2) >> 2, rl = q4 * 32 + lane;
        const int mid = (P.cols / 16 + 1) / 2 * 16, half0 = kTurns ? 0 : group, halves = kTurns ? 2 : 1;
        const int every = kTurns ? 2 : 1;  // tile of this warp
        uint8_t *box = S.tiles + kStageSpace - kTurnSpace + (warp - 2) * kTurnWarp;
        uint32_t n = kTurns ? group : 0;
        bool bad = false;
        // This warp has read the accumulator.  Relaxed: the loads are complete, and a release would wait for the results stored so far
        // to reach memory, a microsecond and more on every tile (1531 x 50257 x 1000: scores 153 us, tensor cores busy for 51 %).
        auto release = [&](uint32_t buf) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0 && !bad) {
                if (kPair) mbar_arrive_cluster_relaxed(mapa_u32(smem_u32(&S.tmem_empty[buf]), 0)); else mbar_arrive(&S.tmem_empty[buf]);
            }
        };
        float scale = P.scale;
        if (MODE != SCORES && P.total) scale = *P.total != 0.f ? scale / *P.total : 0.f;
        for (int t = unit + (int)n * P.units; t < total; t += every * P.units, n += kParts ? 0 : every) {
            const Tile w = tile_at(P, t);
            const int row = (w.um * kCtas + (int)cta_r) * BM + rl, col0 = w.nt * P.cols;
            const bool rows = row - lane < P.M;  // a warp of rows that do not exist has nothing to do
            const uint32_t lanes = tmem_base + ((uint32_t)(q4 * 32) << 16);
            uint32_t buf = n & 1;
            int64_t y = -1;
            if (MODE == SCORES && row < P.M) {
                const int64_t id = target_of(P.y, P.wide_y, row);
                if (id != P.ignore) y = id - P.first - col0;  // of this tile's columns; far outside elsewhere
            }
            float v[MODE == SCORES && kPair || kParts ? kHalf : 1];
            if constexpr (kParts) {
#pragma unroll
                for (int i = 0; i < kHalf; ++i) v[i] = 0.f;
                const uint32_t from = lanes + (group ? mid : 0);
                const int width = group ? P.cols - mid : mid;  // a multiple of 16
#pragma unroll 1
                for (int p0 = 0; p0 < P.k_iters; p0 += P.part, ++n) {
                    buf = n & 1;
                    bad = bad || !mbar_wait_t<kPair>(&S.tmem_full[buf], (n >> 1) & 1, fail);
                    bad = __any_sync(0xffffffffu, bad);
                    tc_fence_after();
                    const bool end = p0 + P.part >= P.k_iters;
                    if (rows && !bad) {
#pragma unroll
                        for (int c = 0; c < kHalf; c += 16)
                            if (c < width) {
                                uint32_t x[16];
                                tmem_ld16(from + buf * kMaxCols + c, x);
                                tmem_ld_wait();
#pragma unroll
                                for (int i = 0; i < 16; ++i) v[c + i] += __uint_as_float(x[i]);
                                // single: the code below takes the sums from where the last part was
                                if (!kPair && end) tmem_st16(from + buf * kMaxCols + c, v + c);
                            }
                        if (!kPair && end) asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    }
                    if (kPair || !end || !rows) release(buf);
                }
                if (!rows) continue;
            } else {
                bad = bad || !mbar_wait_t<kPair>(&S.tmem_full[buf], (n >> 1) & 1, fail);
                bad = __any_sync(0xffffffffu, bad);
                tc_fence_after();
                if (!rows) {
                    release(buf);
                    continue;
                }
            }
            const uint32_t taddr = lanes + buf * kMaxCols;
#pragma unroll 1
            for (int half = half0; half < half0 + halves; ++half) {
                const int c_lo = half ? mid : 0, c_hi = half ? P.cols : mid;
                const bool last = half == half0 + halves - 1;  // the accumulator is free when its last half is read
                if constexpr (MODE == SCORES) {
                    const int exist = min(c_hi, P.N - col0) - c_lo;  // columns of this half that exist, the first of them
                    const int room = (int)min((int64_t)c_hi, P.width - col0) - c_lo;  // the row ends on a multiple of 32, in zeros
                    const int yl = y >= c_lo && y < c_lo + exist ? (int)y - c_lo : -1;
                    __half *e = P.e + (int64_t)row * P.ld + col0 + c_lo;
                    float m = -INFINITY, z = 0.f;
                    if constexpr (kPair) {
                        if constexpr (!kParts) {
                            if (!bad) tmem_half(taddr + c_lo, v);
                            if (last) release(buf);
                        }
                        if (exist < kHalf)
#pragma unroll
                            for (int i = 0; i < kHalf; ++i) v[i] = i < exist ? v[i] : -INFINITY;
                        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, z4[4] = {};
#pragma unroll
                        for (int i = 0; i < kHalf; ++i) m4[i & 3] = fmaxf(m4[i & 3], v[i]);
                        m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                        const float ref = m == -INFINITY ? 0.f : m;
                        if (yl >= 0)
#pragma unroll
                            for (int i = 0; i < kHalf; ++i) store_if(P.target + row, v[i], i == yl);
                        // v - m first: the product with m alone would carry m's size into every exponent
#pragma unroll
                        for (int i = 0; i < kHalf; ++i) {
                            v[i] = exp2_approx(fmaf(v[i] - ref, kLog2e, kExpBits));
                            z4[i & 3] += v[i];
                        }
                        z = (z4[0] + z4[1]) + (z4[2] + z4[3]);
                        if (P.e && row < P.M) put_exp(e, v, room);
                    } else {
                        float v[32];
                        if (!bad) {
#pragma unroll 1
                            for (int c = 0; c < exist; c += 32) {
                                tmem_32(taddr + c_lo + c, exist - c, v);
#pragma unroll
                                for (int i = 0; i < 32; ++i) m = fmaxf(m, v[i]);
                            }
                            const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll 1
                            for (int c = 0; c < c_hi - c_lo; c += 32) {
                                tmem_32(taddr + c_lo + c, exist - c, v);
                                if (yl >= c && yl < c + 32)
#pragma unroll
                                    for (int i = 0; i < 32; ++i) store_if(P.target + row, v[i], i == yl - c);
#pragma unroll
                                for (int i = 0; i < 32; ++i) {
                                    v[i] = exp2_approx(fmaf(v[i] - ref, kLog2e, kExpBits));
                                    z += v[i];
                                }
                                if (P.e && row < P.M) put_exp(e + c, v, room - c);
                            }
                        }
                        if (last) release(buf);
                    }
                    if (row < P.M) {
                        P.stats[(int64_t)row * (2 * P.n_tiles) + 2 * w.nt + half] = make_float2(m, bad ? __uint_as_float(0x7fffffffu) : z * kExpScale);
                    }
                } else {
                    float *sum = P.sum + (P.split > 1 ? (int64_t)w.share * P.M * P.N : 0);
                    const int left = min(c_hi, P.N - col0) - c_lo, exist = row < P.M ? left : 0;
                    const int64_t at = (int64_t)row * P.N + col0 + c_lo;
#pragma unroll
                    for (int c = 0; c < kHalf; c += 64) {
                        float v[64];
                        if (!bad) tmem_64(taddr + c_lo + c, v);
                        else
#pragma unroll
                            for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(0x7fffffffu);
                        if (last && c + 64 == kHalf) release(buf);
#pragma unroll
                        for (int i = 0; i < 64; ++i) v[i] *= scale;
                        if constexpr (kTurn<MODE, kPair>)
                            if (P.kind != VL_BF16) {
#pragma unroll
                                for (int i = 0; i < 64; i += 32)
                                    if (c + i < left)
                                        turn_sum(box, v + i, lane, P.kind, sum + at - (int64_t)lane * P.N + c + i, P.out + at - (int64_t)lane * P.N + c + i, P.N,
                                                 P.M - (row - lane), left - c - i);
                                continue;
                            }
                        if (P.kind == VL_ADD || P.kind == VL_ADD_BF16)
#pragma unroll
                            for (int i = 0; i < 64; i += 4)
                                if (c + i < exist) {
                                    const float4 f = *(const float4 *)(sum + at + c + i);
                                    v[i] += f.x; v[i + 1] += f.y; v[i + 2] += f.z; v[i + 3] += f.w;
                                }
                        if (P.kind == VL_F32 || P.kind == VL_ADD) {
#pragma unroll
                            for (int i = 0; i < 64; i += 4)
                                if (c + i < exist) *(float4 *)(sum + at + c + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                        } else if (c < left) {
                            uint4 o[8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                o[j].x = pack_bf16(__float_as_uint(v[8 * j]), __float_as_uint(v[8 * j + 1])); o[j].y = pack_bf16(__float_as_uint(v[8 * j + 2]), __float_as_uint(v[8 * j + 3]));
                                o[j].z = pack_bf16(__float_as_uint(v[8 * j + 4]), __float_as_uint(v[8 * j + 5])); o[j].w = pack_bf16(__float_as_uint(v[8 * j + 6]), __float_as_uint(v[8 * j + 7]));
                            }
                            if constexpr (kTurn<MODE, kPair>)
                                turn_store(box, o, lane, (uint8_t *)(P.out + at - (int64_t)lane * P.N + c), (int64_t)P.N * 2, P.M - (row - lane), (left - c) / 8);
                            else
#pragma unroll
                                for (int j = 0; j < 8; ++j)
                                    if (c + 8 * j < exist) *(uint4 *)(P.out + at + c + 8 * j) = o[j];
                        }
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (kPair) cluster_sync_all();  // the leader's MMAs use both CTAs' stages and TMEM, its commits arrive on both
    if (warp == 1) {
        tc_fence_after();
        if (kPair) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
    }
}

// ---------------------------------------------------------------------------------------------------- rows
struct RowArgs {
    const float2 *stats;
    const float *parts;              // combine: [shards][2][tokens]
    const void *y;
    const float *weights, *losses_in, *total;
    float *lse, *target, *losses, *out;
    uint32_t *arrived;               // whole step: CTAs that have a token's loss; the last one adds the losses to `out` (null: none does)
    uint8_t *e;                      // [row][ld] 2 bytes each
    const uint8_t *x, *w;
    uint8_t *xc;
    int64_t tokens, first, vocab, whole, ignore, ld, width, x_stride, w_stride;  // x_stride, w_stride: in bytes
    int wide, halves, cols, shards, xvec, grad;
};

__device__ __forceinline__ bool counts(const RowArgs &a, int64_t id) { return id != a.ignore && id >= 0 && id < a.whole; }

__device__ __forceinline__ float weight(const RowArgs &a, int64_t t, int64_t id) { return !counts(a, id) ? 0.f : a.weights ? a.weights[t] : 1.f; }

__device__ __forceinline__ float warp_max(float x)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}
__device__ __forceinline__ float warp_sum(float x)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

constexpr int kRowThreads = 128, kRowRegs = 8;

// Sum of v over the CTA's threads in one order; the result in thread 0 (in its warp).
template <int THREADS> __device__ __forceinline__ float block_sum(float v, float *s_w)
{
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) s_w[threadIdx.x >> 5] = v;
    __syncthreads();
    return threadIdx.x < 32 ? warp_sum(threadIdx.x < THREADS / 32 ? s_w[threadIdx.x] : 0.f) : 0.f;
}
// A thread's share of the sum of the weights (losses null) or of weights * losses.
template <int THREADS> __device__ __forceinline__ float weights_sum(const RowArgs &a, const float *losses)
{
    float sum = 0.f;
#pragma unroll 4
    for (int64_t t = threadIdx.x; t < a.tokens; t += THREADS) {
        const float q = weight(a, t, target_of(a.y, a.wide, t));
        sum += !losses ? q : q == 0.f ? 0.f : q * __ldcg(losses + t);
    }
    return sum;
}

struct RowState { float top, log_z, target; };  // lse = top + log_z
template <int THREADS> struct RowShared { float m[THREADS / 32], z[THREADS / 32], d[THREADS / 32]; };

// A token's sums over its half tiles, by the whole CTA.
template <int THREADS> __device__ __forceinline__ RowState row_state(const RowArgs &a, int64_t t, int64_t id, RowShared<THREADS> &s)
{
    constexpr int W = THREADS / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint64_t at = (uint64_t)id - (uint64_t)a.first;
    const bool here = counts(a, id) && at < (uint64_t)a.vocab;
    float dot = 0.f, given = 0.f;  // the target's logit, as it is and as the tensor cores have it
    if (here) {
        given = a.target[t];
        const uint4 *x = (const uint4 *)(a.x + t * a.x_stride), *w = (const uint4 *)(a.w + (int64_t)at * a.w_stride);
#pragma unroll 4
        for (int v = threadIdx.x; v < a.xvec; v += THREADS) {
            const uint4 p = x[v], q = w[v];
            const uint32_t pw[4] = {p.x, p.y, p.z, p.w}, qw[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // bf16 is the upper half of an fp32
                dot = fmaf(__uint_as_float(pw[i] << 16), __uint_as_float(qw[i] << 16), dot);
                dot = fmaf(__uint_as_float(pw[i] & 0xffff0000u), __uint_as_float(qw[i] & 0xffff0000u), dot);
            }
        }
        dot = warp_sum(dot);
        if (lane == 0) s.d[warp] = dot;
    }
    const float2 *p = a.stats + t * a.halves;
    float m = -INFINITY, z = 0.f;
    for (int i0 = 0; i0 < a.halves; i0 += THREADS * kRowRegs) {
        float2 v[kRowRegs];
        float top = m;
#pragma unroll
        for (int k = 0; k < kRowRegs; ++k) {
            const int i = i0 + k * THREADS + threadIdx.x;
            v[k] = i < a.halves ? p[i] : make_float2(-INFINITY, 0.f);
            top = fmaxf(top, v[k].x);
        }
        const float ref = top == -INFINITY ? 0.f : top;
        z *= __expf(m - ref);
#pragma unroll
        for (int k = 0; k < kRowRegs; ++k) z = fmaf(v[k].y, __expf(v[k].x - ref), z);
        m = top;
    }
    const float wm = warp_max(m);
    if (lane == 0) s.m[warp] = wm;
    __syncthreads();
    RowState r;
    r.top = s.m[0];
#pragma unroll
    for (int w = 1; w < W; ++w) r.top = fmaxf(r.top, s.m[w]);
    const float ref = r.top == -INFINITY ? 0.f : r.top;
    z = warp_sum(z * __expf(m - ref));
    if (lane == 0) s.z[warp] = z;
    __syncthreads();  // also: every thread has read the target's logit that the caller replaces
    z = s.z[0];
#pragma unroll
    for (int w = 1; w < W; ++w) z += s.z[w];
    r.log_z = logf(z);
    r.target = -INFINITY;
    if (here) {
        dot = s.d[0];
#pragma unroll
        for (int w = 1; w < W; ++w) dot += s.d[w];
        const float off = dot - given;  // far off only where logits have no digits behind the point: both stay as they are then
        r.target = given;
        if (fabsf(off) < 0.5f) {
            r.log_z += log1pf(__expf((given - r.top) - r.log_z) * expm1f(off));
            r.target = dot;
        }
    }
    return r;
}

// What a token's CTA leaves; in a whole step the CTA that is last adds the losses, in the order of the tokens.
template <int THREADS> __device__ __forceinline__ void row_end(const RowArgs &a, int64_t t, int64_t id, const RowState &r, float *s_w)
{
    __shared__ int s_last;
    if (threadIdx.x == 0) {
        a.lse[t] = r.top + r.log_z;
        a.target[t] = r.target;
        if (a.losses) a.losses[t] = counts(a, id) && !(a.grad && weight(a, t, id) == 0.f) ? (r.top - r.target) + r.log_z : 0.f;
        if (a.arrived) {
            __threadfence();
            s_last = atomicAdd(a.arrived, 1u) == a.tokens - 1;
            __threadfence();
        }
    }
    if (!a.arrived) return;
    __syncthreads();
    if (!s_last) return;
    float sum = block_sum<THREADS>(weights_sum<THREADS>(a, a.losses), s_w);
    if (threadIdx.x) return;
    if (a.total) sum = *a.total != 0.f ? sum / *a.total : 0.f;
    *a.out = sum;
}

// One CTA per token.
__global__ void __launch_bounds__(kRowThreads) vocab_loss_rows(const __grid_constant__ RowArgs a)
{
    __shared__ RowShared<kRowThreads> s;
    pdl_trigger();
    pdl_wait();
    const int64_t t = blockIdx.x, id = target_of(a.y, a.wide, t);
    const RowState r = row_state<kRowThreads>(a, t, id, s);
    row_end<kRowThreads>(a, t, id, r, s.m);
}

// Joint lse and loss from the shards'.
__global__ void __launch_bounds__(kRowThreads) vocab_loss_join(const __grid_constant__ RowArgs a)
{
    pdl_trigger();
    const int64_t t = (int64_t)blockIdx.x * kRowThreads + threadIdx.x;
    pdl_wait();
    if (t >= a.tokens) return;
    float m = -INFINITY, target = -INFINITY;
    for (int r = 0; r < a.shards; ++r) {
        m = fmaxf(m, a.parts[(int64_t)(2 * r) * a.tokens + t]);
        target = fmaxf(target, a.parts[(int64_t)(2 * r + 1) * a.tokens + t]);
    }
    const float ref = m == -INFINITY ? 0.f : m;
    float z = 0.f;
    for (int r = 0; r < a.shards; ++r) z += expf(a.parts[(int64_t)(2 * r) * a.tokens + t] - ref);
    const float log_z = logf(z);
    a.lse[t] = m + log_z;
    a.losses[t] = counts(a, target_of(a.y, a.wide, t)) ? (m - target) + log_z : 0.f;
}

constexpr int kSumThreads = 1024;
// Sum over the tokens that count of the weights (losses_in null) or of weights * losses, in one order.
__global__ void __launch_bounds__(kSumThreads) vocab_loss_reduce(const __grid_constant__ RowArgs a)
{
    __shared__ float s_w[kSumThreads / 32];
    pdl_trigger();
    pdl_wait();
    float sum = block_sum<kSumThreads>(weights_sum<kSumThreads>(a, a.losses_in), s_w);
    if (threadIdx.x) return;
    if (a.total) sum = *a.total != 0.f ? sum / *a.total : 0.f;
    *a.out = sum;
}

constexpr int kCopyThreads = 256;
// Rows of x to rows of xc that start on 128-byte boundaries; with gradients zeros for tokens that have no part in them.
__global__ void __launch_bounds__(kCopyThreads) vocab_loss_x(const __grid_constant__ RowArgs a)
{
    __shared__ float s_w[kCopyThreads / 32];
    pdl_trigger();
    const int64_t i = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x, t = i / a.xvec;
    const int v = (int)(i - t * a.xvec);
    pdl_wait();
    if (a.arrived && blockIdx.x == gridDim.x - 1) {  // a whole step: the CTA behind the copies has the sum of the weights
        const float sum = block_sum<kCopyThreads>(weights_sum<kCopyThreads>(a, nullptr), s_w);
        if (threadIdx.x == 0) {
            *a.arrived = 0;
            if (a.out) *a.out = sum;
        }
        return;
    }
    if (t >= a.tokens) return;
    const bool on = !a.grad || weight(a, t, target_of(a.y, a.wide, t)) != 0.f;
    ((uint4 *)a.xc)[t * (a.ld / 8) + v] = on ? ((const uint4 *)(a.x + t * a.x_stride))[v] : make_uint4(0, 0, 0, 0);
}

constexpr int kDThreads = 256, kDBatch = 4, kDVecs = kDThreads * kDBatch;
// Exponentials -> d, in place: kDVecs vectors of 8 columns at a time, from the part-th on, every parts-th.  behind: target's logit - lse.
__device__ __forceinline__ void row_to_d(const RowArgs &a, int64_t t, int64_t id, float lse, float behind, uint32_t part, uint32_t parts)
{
    const float q = weight(a, t, id);
    uint4 *row = (uint4 *)(a.e + t * a.ld * 2);
    const uint32_t vecs = (uint32_t)(a.width / 8), cols = (uint32_t)a.cols, mid = (cols / 16 + 1) / 2 * 16;
    const int64_t y = id - a.first;  // may lie in another shard
    const float dy = q * expm1f(behind);
    const float2 *stats = a.stats + t * a.halves;
    for (uint32_t v0 = part * kDVecs + threadIdx.x; v0 < vecs; v0 += parts * kDVecs) {
        uint4 v[kDBatch];
        float f[kDBatch];
        if (q != 0.f)
#pragma unroll
            for (int k = 0; k < kDBatch; ++k) {
                const uint32_t i = v0 + k * kDThreads, col = i * 8, n = col / cols;
                if (i < vecs) {
                    v[k] = row[i];
                    f[k] = stats[2 * n + (col - n * cols >= mid)].x;
                }
            }
#pragma unroll
        for (int k = 0; k < kDBatch; ++k) {
            const uint32_t i = v0 + k * kDThreads;
            if (i >= vecs) break;
            uint4 o = make_uint4(0, 0, 0, 0);
            if (q != 0.f) {
                const float fac = __expf(f[k] - lse) * q * kExpScale;  // lse's rounding is relative here, 2^-24 |lse|: nothing beside bf16's step
                float d[8];
                const __half2 *h = (const __half2 *)&v[k];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 u = __half22float2(h[j]);
                    d[2 * j] = u.x * fac; d[2 * j + 1] = u.y * fac;
                }
                const int64_t at = y - (int64_t)i * 8;
                if (at >= 0 && at < 8 && y < a.vocab)
#pragma unroll
                    for (int j = 0; j < 8; ++j) d[j] = j == (int)at ? dy : d[j];
                o.x = pack_bf16(__float_as_uint(d[0]), __float_as_uint(d[1])); o.y = pack_bf16(__float_as_uint(d[2]), __float_as_uint(d[3]));
                o.z = pack_bf16(__float_as_uint(d[4]), __float_as_uint(d[5])); o.w = pack_bf16(__float_as_uint(d[6]), __float_as_uint(d[7]));
            }
            row[i] = o;
        }
    }
}

// grid (parts of a row, tokens)
__global__ void __launch_bounds__(kDThreads) vocab_loss_d(const __grid_constant__ RowArgs a)
{
    pdl_trigger();
    pdl_wait();
    const int64_t t = blockIdx.y;
    row_to_d(a, t, target_of(a.y, a.wide, t), a.lse[t], a.losses_in ? -a.losses_in[t] : a.target[t] - a.lse[t], blockIdx.x, gridDim.x);
}

// rows and d of a token by one CTA
__global__ void __launch_bounds__(kDThreads) vocab_loss_rows_d(const __grid_constant__ RowArgs a)
{
    __shared__ RowShared<kDThreads> s;
    pdl_trigger();
    pdl_wait();
    const int64_t t = blockIdx.x, id = target_of(a.y, a.wide, t);
    const RowState r = row_state<kDThreads>(a, t, id, s);
    row_to_d(a, t, id, r.top + r.log_z, (r.target - r.top) - r.log_z, 0, 1);
    row_end<kDThreads>(a, t, id, r, s.m);
}

struct ShareArgs { const float *shares; __nv_bfloat16 *out; int64_t n; int split; };
constexpr int kShareSlices = 8;
// Shares of dx added: a warp's lanes hold 8 values each, the warps of a CTA a part of the shares each, whose sums are added in order.
__global__ void __launch_bounds__(32 * kShareSlices) vocab_loss_shares(const __grid_constant__ ShareArgs a)
{
    __shared__ float s_v[kShareSlices][8][33];
    pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t i = ((int64_t)blockIdx.x * 32 + lane) * 8;
    pdl_wait();
    float v[8] = {};
    if (i < a.n)
#pragma unroll 4
        for (int q = warp; q < a.split; q += kShareSlices) {
            const float4 *p = (const float4 *)(a.shares + q * a.n + i);
            const float4 x = p[0], y = p[1];
            v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
            v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
        }
#pragma unroll
    for (int k = 0; k < 8; ++k) s_v[warp][k][lane] = v[k];
    __syncthreads();
    if (warp || i >= a.n) return;
#pragma unroll
    for (int w = 1; w < kShareSlices; ++w)
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] += s_v[w][k][lane];
    uint4 o;
    o.x = pack_bf16(__float_as_uint(v[0]), __float_as_uint(v[1])); o.y = pack_bf16(__float_as_uint(v[2]), __float_as_uint(v[3]));
    o.z = pack_bf16(__float_as_uint(v[4]), __float_as_uint(v[5])); o.w = pack_bf16(__float_as_uint(v[6]), __float_as_uint(v[7]));
    *(uint4 *)(a.out + i) = o;
}

// ---------------------------------------------------------------------------------------------------- launches
const void *gemm_of(int mode, bool pair, bool parts)
{
    if (mode == SCORES && parts) return pair ? (const void *)vocab_loss_gemm<SCORES, true, true> : (const void *)vocab_loss_gemm<SCORES, false, true>;
    if (mode == SCORES) return pair ? (const void *)vocab_loss_gemm<SCORES, true, false> : (const void *)vocab_loss_gemm<SCORES, false, false>;
    if (mode == DX) return pair ? (const void *)vocab_loss_gemm<DX, true, false> : (const void *)vocab_loss_gemm<DX, false, false>;
    return pair ? (const void *)vocab_loss_gemm<DW, true, false> : (const void *)vocab_loss_gemm<DW, false, false>;
}

struct LossDevice { int sms = 0, pairs = 0; };

// Asked once per device; sets the kernels' shared-memory limits on the way.
HcclResult loss_device(LossDevice *out)
{
    static std::mutex mu;
    static LossDevice known[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return HCCL_E_RUNTIME;
    std::lock_guard<std::mutex> lk(mu);
    LossDevice &d = known[dev];
    if (!d.sms) {
        int sms = 0, pairs = 0;
        cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
        for (int mode = SCORES; mode <= DW && e == cudaSuccess; ++mode)
            for (int form = 0; form < 4 && e == cudaSuccess; ++form)
                e = cudaFuncSetAttribute(gemm_of(mode, form & 1, form >> 1), cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes);
        if (e == cudaSuccess) {
            cudaLaunchConfig_t q;
            memset(&q, 0, sizeof(q));
            q.gridDim = dim3((unsigned)(sms / 2 * 2)); q.blockDim = dim3(kThreads); q.dynamicSmemBytes = kSmemBytes;
            cudaLaunchAttribute at[1];
            at[0].id = cudaLaunchAttributeClusterDimension;
            at[0].val.clusterDim.x = 2; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
            q.attrs = at; q.numAttrs = 1;
            e = cudaOccupancyMaxActiveClusters(&pairs, gemm_of(SCORES, true, false), &q);
        }
        if (e != cudaSuccess || pairs < 1) { HLOG_ERROR("vocabulary loss set-up failed: %s", cudaGetErrorString(e)); return HCCL_E_RUNTIME; }
        d.pairs = std::min(pairs, sms / 2);
        d.sms = sms;
    }
    *out = d;
    return HCCL_SUCCESS;
}

// Columns of a tile of the scores: the fewest columns (and ends of tiles, about 48 columns' worth each) for the busiest unit.
int score_cols(int64_t um, int64_t vocab, bool pair, int units)
{
    int best = kMaxCols;
    int64_t least = INT64_MAX;
    for (int cols = kMaxCols; cols >= (pair ? 64 : 32); cols -= 32) {
        const int64_t tiles = um * ((vocab + cols - 1) / cols), t = (tiles + units - 1) / units * (cols + 48);
        if (t < least) { least = t; best = cols; }
    }
    return best;
}

struct Layout { int cols, n_tiles; int64_t ld, width, xld, stats, xc, shares, bytes; bool pair, copy; int split; };

int shares_of(int64_t tokens, int64_t vocab, int32_t hidden, const LossDevice &d, bool pair)
{
    const int units = pair ? d.pairs : d.sms;
    const int64_t tiles = (tokens + (pair ? 255 : 127)) / (pair ? 256 : 128) * ((hidden + kMaxCols - 1) / kMaxCols), k = (vocab + BK - 1) / BK;
    int best = 1;
    double least = 1e30;
    for (int s = 1; s <= 64 && s <= k / 8; ++s) {
        // ns: waves of k steps, then the shares written and read
        const double waves = (double)((tiles * s + units - 1) / units);
        const double t = waves * ((double)(k + s - 1) / s * (pair ? 260. : 290.) + 800.) + (s > 1 ? 3000. + 8. * s * tokens * hidden / 5e3 : 0.);
        if (t < least) { least = t; best = s; }
    }
    return std::max(1, best);
}

// Fewer tokens may need more scratch: their dx is cut into more shares, and their tiles may be narrower.
void layout_on(const LossDevice &d, int64_t tokens, int64_t vocab, int32_t hidden, bool grad, Layout *l)
{
    auto up = [](int64_t n) { return (n + 1023) / 1024 * 1024; };
    l->pair = tokens > BM;
    l->cols = score_cols((tokens + (l->pair ? 255 : 127)) / (l->pair ? 256 : 128), vocab, l->pair, l->pair ? d.pairs : d.sms);
    l->n_tiles = (int)((vocab + l->cols - 1) / l->cols);
    l->ld = (vocab + 63) / 64 * 64;      // rows of the exponentials start on 128-byte lines,
    l->width = (vocab + 31) / 32 * 32;   // and are written as far as the tiles (multiples of 32 columns) reach for certain
    l->split = grad ? shares_of(tokens, vocab, hidden, d, l->pair) : 1;
    l->stats = grad ? up(tokens * l->ld * 2) : 0;
    l->xc = l->stats + up(tokens * l->n_tiles * 2 * (int64_t)sizeof(float2));
    l->xld = (hidden + 63) / 64 * 64;
    // Gradients need the copy for the tokens that do not count.  Rows of x that cross 128-byte lines cost the TMA two requests instead of
    // one, which bounds the product (1531 x 50257 x 1000: scores 150 us, DW 127): more than one row of tiles is worth the copy.
    l->copy = grad || (hidden % 64 != 0 && l->pair);
    l->shares = l->xc + (l->copy ? up(tokens * l->xld * 2) : 0);
    l->bytes = std::max<int64_t>(1024, l->shares + (l->split > 1 ? up((int64_t)l->split * tokens * hidden * 4) : 0));
}

HcclResult layout_of(int64_t tokens, int64_t vocab, int32_t hidden, bool grad, Layout *l)
{
    LossDevice d;
    CHK_RET(loss_device(&d));
    layout_on(d, tokens, vocab, hidden, grad, l);
    return HCCL_SUCCESS;
}

// The caller's scratch has the bytes that the call is about to use.
HcclResult check_scratch(const VocabLossCall &c, int64_t bytes)
{
    CHK_RET_LOG(c.scratch_bytes && c.scratch_bytes < bytes, HCCL_E_PARA, "vocabulary loss: scratch of %lld bytes, %lld tokens need %lld", (long long)c.scratch_bytes,
                (long long)c.tokens, (long long)bytes);
    return HCCL_SUCCESS;
}

// Rows of A in a stage.  Of fewer than 128 rows only those that exist are loaded (in eights, the swizzle's period) where B is long enough:
// the tensor cores read what follows them in shared memory, B, for results that nobody reads (7 tokens x 32000 x 4096: 62 -> 56 us).
int a_rows(int mode, int m, int cols) { return mode == DW || m >= BM || (uint32_t)cols * BK * 2 < kABytes ? BM : (m + 7) / 8 * 8; }

HcclResult launch_gemm(int mode, bool pair, LossGemm &P, void *stream)
{
    LossDevice d;
    CHK_RET(loss_device(&d));
    const int ctas = pair ? 2 : 1;
    P.um_tiles = (P.M + ctas * BM - 1) / (ctas * BM);
    P.n_tiles = (P.N + P.cols - 1) / P.cols;
    P.units = pair ? d.pairs : d.sms;
    P.a_bytes = (uint32_t)a_rows(mode, P.M, P.cols) * BK * 2;
    P.stage_bytes = P.a_bytes + (uint32_t)(P.cols / ctas) * BK * 2;
    const bool turned = pair && mode == DW;
    P.stages = (int)std::min<uint32_t>(kMaxStages, (kStageSpace - (turned ? kTurnSpace : 0)) / P.stage_bytes);
    P.idesc = instr_desc((uint32_t)(ctas * BM), (uint32_t)P.cols) | (mode == DW ? 1u << 15 : 0u) | (mode != SCORES ? 1u << 16 : 0u);
    // a panel's columns of B stay in L2 (40 MB of it) while the rows stream past
    P.panel = (int)std::min<int64_t>(P.n_tiles, std::max<int64_t>(8, (40ll << 20) / ((int64_t)P.cols * P.k_iters * BK * 2)));
    const int parts = mode == SCORES ? std::max(1, P.k_iters / (pair ? kPartLeast<true> : kPartLeast<false>)) : 1;
    P.part = (P.k_iters + parts - 1) / parts;
    const int64_t total = (int64_t)P.um_tiles * P.n_tiles * P.split;
    CHK_RET_LOG(total > INT32_MAX / 2, HCCL_E_PARA, "vocabulary loss: too many tiles");
    return launch_pdl(gemm_of(mode, pair, parts > 1), dim3((unsigned)(std::min<int64_t>(P.units, total) * ctas)), kThreads, kSmemBytes, &P, stream, "vocabulary loss", ctas);
}

RowArgs row_args(const VocabLossCall &c)
{
    RowArgs a;
    memset(&a, 0, sizeof(a));
    a.y = c.targets; a.wide = c.wide; a.weights = c.weights;
    a.tokens = c.tokens; a.first = c.first; a.vocab = c.vocab; a.whole = c.whole; a.ignore = c.ignore;
    return a;
}

}  // namespace

int64_t vocab_loss_chunk(int64_t vocab, bool grad)
{
    // two thousand million bytes of exponentials, or 128 MB of sums of half tiles (16 bytes for 256 columns, or for 128 at worst); the copy of x
    // (as large as the chunk's x) and shares of dx (up to 0.9 GB, of fewer tokens) come on top
    const int64_t ld = (vocab + 63) / 64 * 64, rows = grad ? (int64_t)(1ll << 31) / (ld * 2) : (int64_t)(128ll << 20) / (ld / 128 * 16 + 16);
    return std::min<int64_t>(1 << 20, std::max<int64_t>(256, rows / 256 * 256));
}

int64_t vocab_loss_scratch_bytes(int64_t tokens, int64_t vocab, int32_t hidden, bool grad)
{
    Layout l;
    return layout_of(tokens, vocab, hidden, grad, &l) == HCCL_SUCCESS ? l.bytes : -1;
}

int64_t vocab_loss_scratch_bytes_on(int sms, int pairs, int64_t tokens, int64_t vocab, int32_t hidden, bool grad)
{
    LossDevice d;
    d.sms = sms; d.pairs = pairs;
    Layout l;
    layout_on(d, tokens, vocab, hidden, grad, &l);
    return l.bytes;
}

namespace {

// The copy of x (with the sum of the weights of a whole step) and the scores; leaves what the rows need in *a.
HcclResult scores(const VocabLossCall &c, const Layout &l, bool grad, float *target, uint8_t *s, void *stream, RowArgs *a)
{
    LossGemm P;
    memset(&P, 0, sizeof(P));
    P.M = (int)c.tokens; P.N = (int)c.vocab; P.cols = l.cols; P.split = 1;
    P.k_iters = (c.hidden + BK - 1) / BK;
    P.stats = (float2 *)(s + l.stats); P.target = target;
    P.e = grad ? (__half *)s : nullptr; P.ld = l.ld; P.width = l.width;
    P.y = c.targets; P.wide_y = c.wide; P.first = c.first; P.ignore = c.ignore;
    a->x = (const uint8_t *)c.x; a->x_stride = c.x_stride * 2; a->xvec = c.hidden / 8; a->grad = grad;
    if (l.copy) {
        RowArgs q = *a;
        q.xc = s + l.xc; q.ld = l.xld;
        const int64_t ctas = (c.tokens * q.xvec + kCopyThreads - 1) / kCopyThreads + (a->arrived ? 1 : 0);
        CHK_RET(launch_pdl((const void *)vocab_loss_x, dim3((unsigned)ctas), kCopyThreads, 0, &q, stream, "vocabulary loss (x)"));
    }
    CHK_RET(encode_2d(&P.tmA, l.copy ? s + l.xc : c.x, c.tokens, c.hidden, a_rows(SCORES, (int)c.tokens, l.cols), l.copy ? l.xld : c.x_stride));
    CHK_RET(encode_2d(&P.tmB, c.w, c.vocab, c.hidden, l.cols / (l.pair ? 2 : 1), c.w_stride));
    CHK_RET(launch_gemm(SCORES, l.pair, P, stream));
    a->stats = P.stats; a->halves = 2 * l.n_tiles; a->cols = l.cols;
    a->w = (const uint8_t *)c.w; a->w_stride = c.w_stride * 2;
    a->e = s; a->ld = l.ld; a->width = l.width;
    return HCCL_SUCCESS;
}

HcclResult rows_to_d(const VocabLossCall &c, const Layout &l, const RowArgs &a, void *stream)
{
    // enough CTAs to fill the GPU a few times, none without work (129 tokens x 160000 by one CTA each: 50 us)
    const int64_t parts = std::min<int64_t>((l.width / 8 + kDVecs - 1) / kDVecs, std::max<int64_t>(1, 4096 / c.tokens));
    // tokens along y, 65535 of them at most in a launch
    for (int64_t t0 = 0; t0 < c.tokens; t0 += 65535) {
        RowArgs q = a;
        const int64_t n = std::min<int64_t>(65535, c.tokens - t0);
        q.y = (const uint8_t *)a.y + t0 * (a.wide ? 8 : 4);
        q.weights = a.weights ? a.weights + t0 : nullptr;
        q.losses_in = a.losses_in ? a.losses_in + t0 : nullptr;
        q.e += t0 * a.ld * 2; q.lse += t0; q.target += t0; q.stats += t0 * a.halves;
        CHK_RET(launch_pdl((const void *)vocab_loss_d, dim3((unsigned)parts, (unsigned)n), kDThreads, 0, &q, stream, "vocabulary loss (d)"));
    }
    return HCCL_SUCCESS;
}

HcclResult products(const VocabLossCall &c, const Layout &l, const float *total, float scale, void *dx, void *dw, float *dw_sum, int out, uint8_t *s, void *stream)
{
    LossGemm P;
    memset(&P, 0, sizeof(P));
    P.M = (int)c.tokens; P.N = c.hidden; P.cols = kMaxCols;
    P.total = total; P.scale = scale;
    P.k_iters = (int)((c.vocab + BK - 1) / BK);
    P.split = l.split;
    P.kind = l.split > 1 ? VL_F32 : VL_BF16;
    P.out = (__nv_bfloat16 *)dx; P.sum = (float *)(s + l.shares);
    CHK_RET(encode_2d(&P.tmA, s, c.tokens, l.width, a_rows(DX, (int)c.tokens, kMaxCols), l.ld));
    CHK_RET(encode_2d(&P.tmB, c.w, c.vocab, c.hidden, BK, c.w_stride));
    CHK_RET(launch_gemm(DX, l.pair, P, stream));
    if (l.split > 1) {
        ShareArgs q = {P.sum, P.out, c.tokens * c.hidden, l.split};
        CHK_RET(launch_pdl((const void *)vocab_loss_shares, dim3((unsigned)((q.n / 8 + 31) / 32)), 32 * kShareSlices, 0, &q, stream, "vocabulary loss (dx)"));
    }

    memset(&P, 0, sizeof(P));
    P.M = (int)c.vocab; P.N = c.hidden; P.cols = kMaxCols; P.split = 1;
    P.total = total; P.scale = scale;
    P.k_iters = (int)((c.tokens + BK - 1) / BK);
    P.kind = out; P.out = (__nv_bfloat16 *)dw; P.sum = dw_sum;
    CHK_RET(encode_2d(&P.tmA, s, c.tokens, l.width, BK, l.ld));
    CHK_RET(encode_2d(&P.tmB, s + l.xc, c.tokens, c.hidden, BK, l.xld));
    return launch_gemm(DW, c.vocab > BM, P, stream);
}

}  // namespace

HcclResult vocab_loss_scores(const VocabLossCall &c, bool grad, float *lse, float *target, float *losses, void *scratch, void *stream)
{
    Layout l;
    CHK_RET(layout_of(c.tokens, c.vocab, c.hidden, grad, &l));
    CHK_RET(check_scratch(c, l.bytes));
    RowArgs a = row_args(c);
    CHK_RET(scores(c, l, grad, target, (uint8_t *)scratch, stream, &a));
    a.lse = lse; a.target = target; a.losses = losses;
    return launch_pdl((const void *)vocab_loss_rows, dim3((unsigned)c.tokens), kRowThreads, 0, &a, stream, "vocabulary loss (rows)");
}

HcclResult vocab_loss_combine(const VocabLossCall &c, const float *parts, int shards, float *lse, float *losses, void *stream)
{
    RowArgs a = row_args(c);
    a.parts = parts; a.shards = shards; a.lse = lse; a.losses = losses;
    return launch_pdl((const void *)vocab_loss_join, dim3((unsigned)((c.tokens + kRowThreads - 1) / kRowThreads)), kRowThreads, 0, &a, stream, "vocabulary loss (shards)");
}

HcclResult vocab_loss_total(const VocabLossCall &c, float *total, void *stream)
{
    RowArgs a = row_args(c);
    a.out = total;
    return launch_pdl((const void *)vocab_loss_reduce, dim3(1), kSumThreads, 0, &a, stream, "vocabulary loss (weights)");
}

HcclResult vocab_loss_sum(const VocabLossCall &c, const float *losses, const float *total, float *loss, void *stream)
{
    RowArgs a = row_args(c);
    a.losses_in = losses; a.total = total; a.out = loss;
    return launch_pdl((const void *)vocab_loss_reduce, dim3(1), kSumThreads, 0, &a, stream, "vocabulary loss (sum)");
}

HcclResult vocab_loss_grad(const VocabLossCall &c, const float *lse, const float *target, const float *total, float scale, void *dx, void *dw, float *dw_sum,
                           int out, void *scratch, void *stream)
{
    Layout l;
    CHK_RET(layout_of(c.tokens, c.vocab, c.hidden, true, &l));
    CHK_RET(check_scratch(c, l.bytes));
    uint8_t *s = (uint8_t *)scratch;
    RowArgs a = row_args(c);
    a.stats = (const float2 *)(s + l.stats); a.halves = 2 * l.n_tiles; a.cols = l.cols;
    a.e = s; a.ld = l.ld; a.width = l.width; a.lse = (float *)lse; a.target = (float *)target; a.losses_in = c.losses;
    CHK_RET(rows_to_d(c, l, a, stream));
    return products(c, l, total, scale, dx, dw, dw_sum, out, s, stream);
}

// Behind the scratch of its parts: lse, target logit and loss of every token, the sum of the weights, the tokens that have arrived.
static int64_t step_bytes(int64_t parts, int64_t tokens) { return (parts + 255) / 256 * 256 + (3 * tokens + 2) * 4; }

int64_t vocab_loss_step_bytes(int64_t tokens, int64_t vocab, int32_t hidden)
{
    const int64_t n = vocab_loss_scratch_bytes(tokens, vocab, hidden, true);
    return n < 0 ? -1 : step_bytes(n, tokens);
}

HcclResult vocab_loss_step(const VocabLossCall &c, bool mean, float scale, float *loss, void *dx, void *dw, float *dw_sum, int out, void *scratch, void *stream)
{
    Layout l;
    CHK_RET(layout_of(c.tokens, c.vocab, c.hidden, true, &l));
    CHK_RET(check_scratch(c, step_bytes(l.bytes, c.tokens)));
    uint8_t *s = (uint8_t *)scratch;
    float *words = (float *)(s + (l.bytes + 255) / 256 * 256), *total = words + 3 * c.tokens;
    RowArgs a = row_args(c);
    a.lse = words; a.target = words + c.tokens; a.losses = words + 2 * c.tokens;
    a.arrived = (uint32_t *)total + 1; a.out = mean ? total : nullptr;
    CHK_RET(scores(c, l, true, a.target, s, stream, &a));
    a.out = loss; a.total = mean ? total : nullptr;
    // one launch for rows and d where a CTA per token fills the GPU, or has little to do
    if (c.tokens >= 1024 || l.width <= 8 * kDVecs)
        CHK_RET(launch_pdl((const void *)vocab_loss_rows_d, dim3((unsigned)c.tokens), kDThreads, 0, &a, stream, "vocabulary loss (rows, d)"));
    else {
        CHK_RET(launch_pdl((const void *)vocab_loss_rows, dim3((unsigned)c.tokens), kRowThreads, 0, &a, stream, "vocabulary loss (rows)"));
        a.losses_in = a.losses;
        CHK_RET(rows_to_d(c, l, a, stream));
    }
    return products(c, l, a.total, scale, dx, dw, dw_sum, out, s, stream);
}

}  // namespace hcclb
