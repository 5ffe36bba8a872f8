// Loss of a linear head for few rows (scoring a handful of positions against a large vocabulary): at most 64 rows, no gradient.
//
// With so few rows the weights are all there is to read and every one is used rows times only, so the split pass of
// linear_ce.cu (4 bytes written and read again for every 4 read) would cost more than the products.
//
// Up to 8 rows: fp32 on the CUDA cores (rows 2 N K operations are below the time of reading 4 N K bytes up to about 10 rows).
// x sits in shared memory; the weights stream through registers, several 16-byte loads in flight per thread.
//
// 9 to 64 rows: the weights go from HBM into shared memory once, as they are, and the tensor core multiplies them as tf32: a 128-class tile is the M side of the
// MMA, the rows (padded to 16, 32 or 64) its N side.  3xTF32: the tensor core itself reads the high part out of the fp32 word
// (its top 19 bits); eight warps compute the low part of each landed tile, element by element at the same shared-memory offset
// (so the swizzle and either weight layout need no index arithmetic), and x comes in both parts from a small pass.
// Per CTA: one thread feeds the ring by TMA, one issues the MMAs, eight warps split, four drain the accumulator (every 64 of K,
// see gemm_split16.cuh) and keep each row's running maximum and sum of exponentials over the classes the CTA has seen.  The
// classes are dealt out in granules of 16 (32 where the weight rows hold the features), so that all CTAs get the same
// number within one and the weights are read at the same pace everywhere.
// Measured: 1 x 32000 x 2048 (262 MB) 65 us with its three launches, 8 x 131072 x 4096 (2.1 GB) 0.39 ms, both bound by HBM;
// 40 x 50021 x 1024 (205 MB) 101 us, bound by the MMAs: 12 of 128 x 64 x 8 per 16 KB of weights at about 140 cycles each, the same
// with 16 rows, with independent accumulators and with the weights fetched into L2 ahead.
#include <cuda_runtime.h>

#include <cmath>
#include <cstring>

#include "../../include/odl_b200.h"
#include "gemm_split16.cuh"
#include "gemm_tc.cuh"
#include "host_util.h"
#include "internal.h"
#include "linear_ce.h"
#include "ptx_sm100.cuh"
#include "tmap.h"

namespace odl
{

namespace
{
constexpr int kRowsMost = 64;
constexpr int kClasses  = 128;         // of a tile
constexpr int kTileA    = kClasses * 128;  // bytes: 32 fp32 of K
constexpr int kLow      = 3;           // low-part buffers, each with a pair of warps that fills it: a tile costs a pair several
constexpr int kPair     = 2;           // latencies one behind the other (wait, load, store, proxy fence, arrive)
constexpr int kConv     = kLow * kPair;
constexpr int kDrain    = 4;
constexpr int kThreads  = 64 + 32 * (kDrain + kConv);
constexpr float kLog2e  = 1.4426950408889634f;

inline size_t a256(size_t x)
{
    return (x + 255) & ~size_t(255);
}

struct FewWords  // device
{
    int count, bad;
    unsigned done;  // rows whose loss is written
};

// Rows with a label, in order, and their x in two tf32 parts, padded with zeros to rows_pad x k_pad.  Every block lists the rows
// by itself (at most 64 labels); block 0 writes the list down.
__global__ void __launch_bounds__(256) few_rows_kernel(const float *__restrict__ x, const void *__restrict__ labels, int is64, int64_t ignore, int M, int N,
                                                       int K, int rows_pad, int k_pad, float *__restrict__ big, float *__restrict__ small,
                                                       int *__restrict__ idx, int *__restrict__ cls, FewWords *words, float *__restrict__ lse_out)
{
    __shared__ int s_idx[kRowsMost], s_cls[kRowsMost], s_count, s_bad;
    if (threadIdx.x < 32)
    {
        int base = 0, bad = 0;
        for (int r0 = 0; r0 < kRowsMost; r0 += 32)
        {
            const int r = r0 + threadIdx.x;
            int c       = -1;
            if (r < M)
            {
                const int64_t t = is64 ? static_cast<const int64_t *>(labels)[r] : static_cast<const int32_t *>(labels)[r];
                c               = t != ignore && t >= 0 && t < N ? static_cast<int>(t) : -1;
                bad |= t != ignore && c < 0;
                if (c < 0 && blockIdx.x == 0 && lse_out)
                    lse_out[r] = 0.f;
            }
            const unsigned have = __ballot_sync(0xffffffffu, c >= 0);
            if (c >= 0)
            {
                const int pos = base + __popc(have & ((1u << threadIdx.x) - 1));
                s_idx[pos] = r, s_cls[pos] = c;
            }
            base += __popc(have);
        }
        bad = __any_sync(0xffffffffu, bad);
        if (threadIdx.x == 0)
            s_count = base, s_bad = bad;
    }
    __syncthreads();
    const int count = s_count;
    if (blockIdx.x == 0)
    {
        if (threadIdx.x < kRowsMost)
        {
            const bool on   = static_cast<int>(threadIdx.x) < count;
            idx[threadIdx.x] = on ? s_idx[threadIdx.x] : -1;
            cls[threadIdx.x] = on ? s_cls[threadIdx.x] : -1;
        }
        if (threadIdx.x == 0)
            words->count = count, words->bad = s_bad, words->done = 0;
    }
    const int n = rows_pad * k_pad;
    for (int i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256)
    {
        const int r = i / k_pad, c = i - r * k_pad;
        const float v = r < count && c < K ? x[static_cast<int64_t>(s_idx[r]) * K + c] : 0.f;
        big[i]        = v;
        small[i]      = tf32_small(v);
    }
}

template <int NX, int TERMS>
struct FewCfg
{
    static constexpr int b_bytes = NX * 128;
    static constexpr int parts   = TERMS == 3 ? 2 : 1;
    static constexpr int stage   = kTileA + parts * b_bytes;  // weights as landed, x in its parts
    static constexpr int low     = TERMS == 3 ? kLow * kTileA : 0;
    static constexpr int stages  = (208 * 1024 - low) / stage > 8 ? 8 : (208 * 1024 - low) / stage;
    static constexpr int smem    = 1024 + stages * stage + low + 2048;
    static constexpr int stride  = NX < 32 ? 32 : NX;  // TMEM columns of an accumulator (drained 32 at a time)
};

struct FewTmaps
{
    CUtensorMap w, x, x_small;
};

struct FewArgs
{
    const float *bias;
    const int *cls;
    const FewWords *words;
    float2 *part;   // [row][parts]
    float *picked;
    int *err;
    int N, K, w_mn, parts;
};

// reduces v[0..31] over the 32 lanes; lane l receives the result of v[l]
template <bool MAX>
__device__ __forceinline__ float across(float (&v)[32], int lane)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
    {
#pragma unroll
        for (int i = 0; i < o; ++i)
        {
            const bool up    = lane & o;
            const float keep = up ? v[i + o] : v[i], give = up ? v[i] : v[i + o];
            const float got  = __shfl_xor_sync(0xffffffffu, give, o);
            v[i]             = MAX ? fmaxf(keep, got) : keep + got;
        }
    }
    return v[0];
}

template <int NX, int TERMS>
__global__ void __launch_bounds__(kThreads, 1) few_logits_kernel(const __grid_constant__ FewTmaps tm, const FewArgs p)
{
    using C = FewCfg<NX, TERMS>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *tiles      = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *lows       = tiles + C::stages * C::stage;
    uint8_t *aux        = lows + C::low;
    uint64_t *full_bar  = reinterpret_cast<uint64_t *>(aux);
    uint64_t *conv_bar  = full_bar + C::stages;
    uint64_t *done_bar  = conv_bar + kLow;
    uint64_t *acc_full  = done_bar + C::stages;
    uint64_t *acc_empty = acc_full + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + 2);
    volatile int *abort_f = reinterpret_cast<volatile int *>(tmem_slot + 1);
    int *early_out        = const_cast<int *>(abort_f) + 1;
    float *ref_all        = reinterpret_cast<float *>(aux + 512);   // [kDrain][32]
    int *s_cls            = reinterpret_cast<int *>(aux + 1024);    // [64]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0)
    {
        *early_out = *reinterpret_cast<volatile int *>(p.err) == 1;
        *abort_f   = 0;
        for (int s = 0; s < C::stages; ++s)
        {
            ptx::mbar_init(&full_bar[s], 1);
            ptx::mbar_init(&done_bar[s], 1);
        }
        for (int l = 0; l < kLow; ++l)
            ptx::mbar_init(&conv_bar[l], kPair);
        for (int b = 0; b < 2; ++b)
        {
            ptx::mbar_init(&acc_full[b], 1);
            ptx::mbar_init(&acc_empty[b], kDrain);
        }
        ptx::fence_mbar_init();
        ptx::prefetch_tmap(&tm.w);
        ptx::prefetch_tmap(&tm.x);
        ptx::prefetch_tmap(&tm.x_small);
    }
    if (threadIdx.x < 64)
        s_cls[threadIdx.x] = static_cast<int>(threadIdx.x) < p.words->count ? p.cls[threadIdx.x] : -1;
    if (warp == 1)
    {
        ptx::tmem_alloc(tmem_slot, 2 * C::stride);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    const bool skip          = *early_out != 0;

    // this CTA's classes: granules of 16 (32 for MN-major weights), dealt out evenly, walked in tiles of equal size <= 128
    const int gran = p.w_mn ? 32 : 16, per_tile = kClasses / gran;
    const int grans = (p.N + gran - 1) / gran;
    const int g0 = static_cast<int>(static_cast<int64_t>(grans) * blockIdx.x / gridDim.x);
    const int g1 = static_cast<int>(static_cast<int64_t>(grans) * (blockIdx.x + 1) / gridDim.x);
    const int n_tiles = (g1 - g0 + per_tile - 1) / per_tile;
    const int tile_g  = n_tiles ? (g1 - g0 + n_tiles - 1) / n_tiles : 0;  // granules of a tile
    const int n_kb    = (p.K + 31) / 32;

    if (skip)
    {
        // nothing
    }
    else if (warp == 0)
    {
        uint32_t gk = 0;
        bool ok     = true;
        for (int t = 0; ok && t < n_tiles; ++t)
        {
            const int ga = g0 + t * tile_g, gb = min(g1, ga + tile_g);
            for (int kb = 0; kb < n_kb; ++kb, ++gk)
            {
                const int s = gk % C::stages;
                ok          = __all_sync(0xffffffffu, ptx::mbar_wait(&done_bar[s], ((gk / C::stages) & 1) ^ 1, abort_f));
                if (!ok)
                    break;
                if (lane == 0)
                {
                    uint8_t *st = tiles + s * C::stage;
                    ptx::mbar_arrive_expect_tx(&full_bar[s], (gb - ga) * gran * 128 + C::parts * C::b_bytes);
                    for (int g = ga; g < gb; ++g)
                    {
                        uint8_t *dst = st + (g - ga) * gran * 128;
                        if (p.w_mn)
                            ptx::tma_load_2d(dst, &tm.w, &full_bar[s], g * gran, kb * 32);
                        else
                            ptx::tma_load_2d(dst, &tm.w, &full_bar[s], kb * 32, g * gran);
                    }
                    uint8_t *sb = st + kTileA;
                    ptx::tma_load_2d(sb, &tm.x, &full_bar[s], kb * 32, 0);
                    if (TERMS == 3)
                        ptx::tma_load_2d(sb + C::b_bytes, &tm.x_small, &full_bar[s], kb * 32, 0);
                }
                __syncwarp();
            }
        }
        if (*abort_f && lane == 0)
        {
            // let the copies still in flight land before the CTA goes away
            const uint32_t from = gk > C::stages ? gk - C::stages : 0;
            for (uint32_t k = from; k < gk; ++k)
                ptx::mbar_wait(&full_bar[k % C::stages], (k / C::stages) & 1, nullptr);
        }
    }
    else if (warp == 1)
    {
        if (lane == 0)
        {
            const uint32_t idesc  = ptx::make_idesc_tf32(kClasses, NX, p.w_mn != 0, false);
            const uint32_t a_step = p.w_mn ? 1024u : 32u, a_lbo = p.w_mn ? 4096u : 16u, a_sbo = p.w_mn ? 512u : 1024u;
            const uint32_t a_lay  = p.w_mn ? ptx::kLayoutSw128Base32 : ptx::kLayoutSw128;
            uint32_t gk = 0, gc = 0;
            bool ok     = true;
            for (int t = 0; ok && t < n_tiles; ++t)
                for (int kb = 0; ok && kb < n_kb; ++gc)
                {
                    const int buf = gc & 1;
                    if (!ptx::mbar_wait(&acc_empty[buf], ((gc >> 1) & 1) ^ 1, abort_f))
                    {
                        ok = false;
                        break;
                    }
                    ptx::tc_fence_after_sync();
                    const uint32_t d = tmem_base + buf * C::stride;
                    const int end    = min(n_kb, kb + 2);
                    for (bool first = true; kb < end; ++kb, ++gk)
                    {
                        const int s = gk % C::stages, l = gk % kLow;
                        if (!ptx::mbar_wait(&full_bar[s], (gk / C::stages) & 1, abort_f) ||
                            (TERMS == 3 && !ptx::mbar_wait(&conv_bar[l], (gk / kLow) & 1, abort_f)))
                        {
                            ok = false;
                            break;
                        }
                        ptx::tc_fence_after_sync();
                        const uint32_t sa = ptx::smem_u32(tiles + s * C::stage), sb = sa + kTileA, sl = ptx::smem_u32(lows + l * kTileA);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                        {
                            const uint64_t da = ptx::make_smem_desc(sa + k * a_step, a_lbo, a_sbo, a_lay);
                            const uint64_t db = ptx::make_smem_desc(sb + k * 32, 16, 1024, ptx::kLayoutSw128);
                            if (TERMS == 3)
                            {
                                const uint64_t das = ptx::make_smem_desc(sl + k * a_step, a_lbo, a_sbo, a_lay);
                                const uint64_t dbs = ptx::make_smem_desc(sb + C::b_bytes + k * 32, 16, 1024, ptx::kLayoutSw128);
                                ptx::mma_tf32_ss(d, das, db, idesc, !first);
                                ptx::mma_tf32_ss(d, da, dbs, idesc, 1);
                                ptx::mma_tf32_ss(d, da, db, idesc, 1);
                            }
                            else
                                ptx::mma_tf32_ss(d, da, db, idesc, !first);
                            first = false;
                        }
                        ptx::mma_commit(&done_bar[s]);
                    }
                    if (ok)
                        ptx::mma_commit(&acc_full[buf]);
                }
        }
    }
    else if (warp >= 2 + kDrain)
    {
        // ================================================================= low parts of landed weight tiles
        if (TERMS == 3)
        {
            const int group   = (warp - 2 - kDrain) / kPair;
            const int me      = threadIdx.x - 32 * (2 + kDrain + group * kPair);
            const int n_total = n_tiles * n_kb;
            for (int gk = group; gk < n_total; gk += kLow)
            {
                // The buffer is free once the MMAs of K-block gk - kLow are done.  That wait comes first: with it the stage's
                // previous use is over too, so that the barrier is at most one phase behind the one asked for (a parity
                // cannot tell two).
                const int s = gk % C::stages, before = gk - kLow;
                if (before >= 0 && !__all_sync(0xffffffffu, ptx::mbar_wait(&done_bar[before % C::stages], (before / C::stages) & 1, abort_f)))
                    break;
                if (!__all_sync(0xffffffffu, ptx::mbar_wait(&full_bar[s], (gk / C::stages) & 1, abort_f)))
                    break;
                const float4 *src = reinterpret_cast<const float4 *>(tiles + s * C::stage) + me;
                float4 *dst       = reinterpret_cast<float4 *>(lows + group * kTileA) + me;
                constexpr int kEach = kTileA / 16 / (32 * kPair);
#pragma unroll
                for (int i0 = 0; i0 < kEach; i0 += 8)
                {
                    float4 v[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        v[i] = src[(i0 + i) * 32 * kPair];
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        dst[(i0 + i) * 32 * kPair] = make_float4(tf32_small(v[i].x), tf32_small(v[i].y), tf32_small(v[i].z), tf32_small(v[i].w));
                }
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0)
                    ptx::mbar_arrive(&conv_bar[group]);
            }
        }
    }
    else
    {
        // ================================================================= drain, statistics (warps 2..5)
        const int q = warp & 3;
        float *ref  = ref_all + 32 * q;
        constexpr int kBlocks = C::stride / 32;  // of 32 rows
        float run_m[kBlocks], run_s[kBlocks];
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
            run_m[b] = -INFINITY, run_s[b] = 0.f;
        uint32_t gc = 0;
        bool ok     = true;
        for (int t = 0; ok && t < n_tiles; ++t)
        {
            const int c0 = (g0 + t * tile_g) * gran, c1 = min(p.N, min(g1, g0 + (t + 1) * tile_g) * gran);
            const int cl = c0 + 32 * q + lane;
            float acc[C::stride];
#pragma unroll
            for (int i = 0; i < C::stride; ++i)
                acc[i] = 0.f;
            for (int kb = 0; kb < n_kb; kb += 2, ++gc)
            {
                const int buf = gc & 1;
                ok            = __all_sync(0xffffffffu, ptx::mbar_wait(&acc_full[buf], (gc >> 1) & 1, abort_f));
                if (!ok)
                    break;
                ptx::tc_fence_after_sync();
#pragma unroll
                for (int j = 0; j < kBlocks; ++j)
                {
                    uint32_t r[32];
                    ptx::tmem_ld_32x32(tmem_base + (static_cast<uint32_t>(32 * q) << 16) + buf * C::stride + 32 * j, r);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        acc[32 * j + i] += __uint_as_float(r[i]);
                }
                ptx::tc_fence_before_sync();
                __syncwarp();
                if (lane == 0)
                    ptx::mbar_arrive(&acc_empty[buf]);
            }
            if (!ok)
                break;
            const bool in    = cl < c1;
            const float bias = in && p.bias ? __ldg(p.bias + cl) : 0.f;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
            {
                float v[32];
                const int mine  = s_cls[32 * b + lane];  // (64 entries; -1 past the last row)
                const bool hits = mine >= c0 + 32 * q && mine < c0 + 32 * q + 32;
                unsigned rows   = __ballot_sync(0xffffffffu, hits);
#pragma unroll
                for (int i = 0; i < 32; ++i)
                {
                    const float z = acc[32 * b + i] + bias;
                    // row 32 b + i has its label among this warp's classes: the lane that holds it writes the logit
                    if ((rows >> i) & 1u)
                        if (s_cls[32 * b + i] == cl && in)
                            p.picked[32 * b + i] = z;
                    acc[32 * b + i] = in ? z : -INFINITY;
                    v[i]            = acc[32 * b + i];
                }
                const float top  = fmaxf(run_m[b], across<true>(v, lane));
                const float base = top == -INFINITY ? 0.f : top;
                __syncwarp();
                ref[lane] = base;
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    v[i] = s16::fast_exp2((acc[32 * b + i] - ref[i]) * kLog2e);
                run_s[b] = run_s[b] * s16::fast_exp2((run_m[b] - base) * kLog2e) + across<false>(v, lane);
                run_m[b] = top;
            }
        }
        if (ok)
        {
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
                p.part[static_cast<int64_t>(32 * b + lane) * p.parts + blockIdx.x * kDrain + q] = make_float2(run_m[b], run_s[b]);
        }
        ptx::tc_fence_before_sync();
    }

    __syncthreads();
    if (warp == 1)
    {
        __syncwarp();
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc(tmem_base, 2 * C::stride);
    }
    if (threadIdx.x == 0 && *abort_f)
        atomicExch(p.err, 1);
}

__device__ __forceinline__ void join(float &m, float &s, float om, float os)
{
    const float t = fmaxf(m, om), b = t == -INFINITY ? 0.f : t;
    s = s * s16::fast_exp2((m - b) * kLog2e) + os * s16::fast_exp2((om - b) * kLog2e);
    m = t;
}

// a block per row joins its statistics; the last one to finish adds up the loss, in order
__global__ void __launch_bounds__(256) few_finish_kernel(const float2 *__restrict__ part, int parts, const int *__restrict__ idx, const float *__restrict__ picked,
                                                         FewWords *words, float *__restrict__ row_loss, float *__restrict__ lse_out, float *loss, int *err)
{
    const int row = blockIdx.x, lane = threadIdx.x & 31;
    const int count = words->count;
    __shared__ float2 box[8];
    __shared__ int last;
    if (row < count)
    {
        float m = -INFINITY, s = 0.f;
        for (int k = threadIdx.x; k < parts; k += 256)
        {
            const float2 v = part[static_cast<int64_t>(row) * parts + k];
            join(m, s, v.x, v.y);
        }
        for (int o = 16; o > 0; o >>= 1)
        {
            const float om = __shfl_xor_sync(0xffffffffu, m, o), os = __shfl_xor_sync(0xffffffffu, s, o);
            // both partners must compute the same bits: the lower lane's value first
            float m0 = (lane & o) ? om : m, s0 = (lane & o) ? os : s;
            join(m0, s0, (lane & o) ? m : om, (lane & o) ? s : os);
            m = m0, s = s0;
        }
        if (lane == 0)
            box[threadIdx.x >> 5] = make_float2(m, s);
        __syncthreads();
        if (threadIdx.x == 0)
        {
            for (int w = 1; w < 8; ++w)
                join(m, s, box[w].x, box[w].y);
            const float l = m + logf(s);
            row_loss[row] = l - picked[row];
            if (lse_out)
                lse_out[idx[row]] = l;
        }
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0)
        last = atomicAdd(&words->done, 1u) == gridDim.x - 1;
    __syncthreads();
    if (last && threadIdx.x == 0)
    {
        __threadfence();
        double s = 0;
        for (int r = 0; r < count; ++r)
            s += __ldcg(row_loss + r);
        if (loss)
            *loss = count > 0 ? static_cast<float>(s / count) : 0.f;
        if (words->bad && *err == 0)
            atomicExch(err, 4);  // last: launches of the library leave early while the flag is up
    }
}

// ---- up to 8 rows on the CUDA cores -------------------------------------------------------------------------------------------
constexpr int kSimtRows  = 8;
constexpr int kSimtWarps = 16;

struct SimtArgs
{
    const float *w, *x;  // x: [R][k_pad], gathered, padded with zeros
    const float *bias;
    const int *cls;
    const FewWords *words;
    float2 *part;        // [row][parts]
    float *picked;
    int N, K, k_pad, parts;
};

// sums v[0..V) over the 32 lanes; every lane receives the sum of v[lane % V]
template <int V>
__device__ __forceinline__ float fold(float (&v)[V], int lane)
{
#pragma unroll
    for (int o = 16; o >= V; o >>= 1)
    {
#pragma unroll
        for (int i = 0; i < V; ++i)
            v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
#pragma unroll
    for (int o = V / 2; o > 0; o >>= 1)
    {
#pragma unroll
        for (int i = 0; i < o; ++i)
        {
            const bool up    = lane & o;
            const float keep = up ? v[i + o] : v[i], give = up ? v[i] : v[i + o];
            v[i]             = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
    }
    return v[0];
}

// Weights [N][K]: a warp takes C classes at a time, its lanes the features; the C R sums are folded over the lanes, and each
// lane keeps the running statistics of one (class mod C, row).
template <int R, bool VEC>
__global__ void __launch_bounds__(32 * kSimtWarps) few_simt_rows_kernel(const SimtArgs p)
{
    constexpr int C = R <= 4 ? 8 : 4, V = C * R;
    extern __shared__ float4 xs4[];
    float *xs      = reinterpret_cast<float *>(xs4);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int i = threadIdx.x; i < R * p.k_pad / 4; i += 32 * kSimtWarps)
        xs4[i] = reinterpret_cast<const float4 *>(p.x)[i];
    __syncthreads();
    const int all    = gridDim.x * kSimtWarps, me = warp * gridDim.x + blockIdx.x;
    const int my_row = (lane % V) / C;
    const int label  = my_row < p.words->count ? p.cls[my_row] : -1;
    float m = -INFINITY, s = 0.f;
    for (int64_t c0 = static_cast<int64_t>(me) * C; c0 < p.N; c0 += static_cast<int64_t>(all) * C)
    {
        float acc[V];
#pragma unroll
        for (int i = 0; i < V; ++i)
            acc[i] = 0.f;
        const float *row[C];
#pragma unroll
        for (int c = 0; c < C; ++c)
            row[c] = p.w + (c0 + c < p.N ? c0 + c : p.N - 1) * p.K;
        if (VEC)
        {
#pragma unroll 2
            for (int k = 4 * lane; k < p.K; k += 128)
            {
                float4 wv[C];
#pragma unroll
                for (int c = 0; c < C; ++c)
                    wv[c] = __ldcs(reinterpret_cast<const float4 *>(row[c] + k));
#pragma unroll
                for (int r = 0; r < R; ++r)
                {
                    const float4 xv = *reinterpret_cast<const float4 *>(xs + r * p.k_pad + k);
#pragma unroll
                    for (int c = 0; c < C; ++c)
                    {
                        float a = acc[r * C + c];
                        a       = fmaf(wv[c].x, xv.x, a);
                        a       = fmaf(wv[c].y, xv.y, a);
                        a       = fmaf(wv[c].z, xv.z, a);
                        acc[r * C + c] = fmaf(wv[c].w, xv.w, a);
                    }
                }
            }
        }
        else
        {
#pragma unroll 2
            for (int k = lane; k < p.K; k += 32)
            {
                float wv[C];
#pragma unroll
                for (int c = 0; c < C; ++c)
                    wv[c] = __ldcs(row[c] + k);
#pragma unroll
                for (int r = 0; r < R; ++r)
                {
                    const float xv = xs[r * p.k_pad + k];
#pragma unroll
                    for (int c = 0; c < C; ++c)
                        acc[r * C + c] = fmaf(wv[c], xv, acc[r * C + c]);
                }
            }
        }
        const float sum = fold<V>(acc, lane);
        const int64_t c = c0 + (lane % V) % C;
        const bool in   = c < p.N;
        const float z   = sum + (in && p.bias ? __ldg(p.bias + c) : 0.f);
        if (in && c == label && lane < V)
            p.picked[my_row] = z;
        if (in)
            join(m, s, z, 1.f);
    }
    // lanes lane, lane ^ 1, .. of a row's C classes; the lower one's value first, so that both get the same bits
#pragma unroll
    for (int o = C / 2; o > 0; o >>= 1)
    {
        const float om = __shfl_xor_sync(0xffffffffu, m, o), os = __shfl_xor_sync(0xffffffffu, s, o);
        float m0 = (lane & o) ? om : m, s0 = (lane & o) ? os : s;
        join(m0, s0, (lane & o) ? m : om, (lane & o) ? s : os);
        m = m0, s = s0;
    }
    if (lane < V && lane % C == 0)
        p.part[static_cast<int64_t>(my_row) * p.parts + me] = make_float2(m, s);
}

// Weights [K][N]: a block takes 128 classes (4 a lane), its warps the features; the warps' sums meet in shared memory.
template <int R, bool VEC>
__global__ void __launch_bounds__(32 * kSimtWarps) few_simt_cols_kernel(const SimtArgs p)
{
    extern __shared__ float4 xs4[];
    float *xs      = reinterpret_cast<float *>(xs4);
    float *sums    = xs + R * p.k_pad;  // [warp][R][128]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int i = threadIdx.x; i < R * p.k_pad / 4; i += 32 * kSimtWarps)
        xs4[i] = reinterpret_cast<const float4 *>(p.x)[i];
    __syncthreads();
    // thread = (row, class) of the block's statistics
    constexpr int kEach = (R * 128 + 32 * kSimtWarps - 1) / (32 * kSimtWarps);
    float m[kEach], s[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e)
        m[e] = -INFINITY, s[e] = 0.f;
    const int count = p.words->count;
    for (int64_t c0 = static_cast<int64_t>(blockIdx.x) * 128; c0 < p.N; c0 += static_cast<int64_t>(gridDim.x) * 128)
    {
        float acc[R][4];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                acc[r][j] = 0.f;
        const int64_t c = c0 + 4 * lane;
#pragma unroll 8
        for (int k = warp; k < p.K; k += kSimtWarps)
        {
            const float *row = p.w + static_cast<int64_t>(k) * p.N + c;
            float wv[4]      = {0.f, 0.f, 0.f, 0.f};
            if (VEC)
            {
                if (c < p.N)
                {
                    const float4 q = __ldcs(reinterpret_cast<const float4 *>(row));
                    wv[0] = q.x, wv[1] = q.y, wv[2] = q.z, wv[3] = q.w;
                }
            }
            else
            {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c + j < p.N)
                        wv[j] = __ldcs(row + j);
            }
#pragma unroll
            for (int r = 0; r < R; ++r)
            {
                const float xv = xs[r * p.k_pad + k];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[r][j] = fmaf(wv[j], xv, acc[r][j]);
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
            *reinterpret_cast<float4 *>(sums + (warp * R + r) * 128 + 4 * lane) = make_float4(acc[r][0], acc[r][1], acc[r][2], acc[r][3]);
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kEach; ++e)
        {
            const int i     = threadIdx.x + e * 32 * kSimtWarps, r = i / 128;
            const int64_t n = c0 + i % 128;
            if (i < R * 128 && n < p.N)
            {
                float z = p.bias ? __ldg(p.bias + n) : 0.f, t = 0.f;
                for (int w = 0; w < kSimtWarps; ++w)
                    t += sums[w * R * 128 + i];
                z += t;
                if (r < count && p.cls[r] == n)
                    p.picked[r] = z;
                join(m[e], s[e], z, 1.f);
            }
        }
        __syncthreads();
    }
    // a warp's 32 classes of a row, then one part per (block, 32 classes)
#pragma unroll
    for (int e = 0; e < kEach; ++e)
    {
        const int i = threadIdx.x + e * 32 * kSimtWarps;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
        {
            const float om = __shfl_xor_sync(0xffffffffu, m[e], o), os = __shfl_xor_sync(0xffffffffu, s[e], o);
            float m0 = (lane & o) ? om : m[e], s0 = (lane & o) ? os : s[e];
            join(m0, s0, (lane & o) ? m[e] : om, (lane & o) ? s[e] : os);
            m[e] = m0, s[e] = s0;
        }
        if (lane == 0 && i < R * 128)
            p.part[static_cast<int64_t>(i / 128) * p.parts + blockIdx.x * 4 + (i % 128) / 32] = make_float2(m[e], s[e]);
    }
}

size_t simt_smem(int rows, int k_pad, int mn)
{
    return static_cast<size_t>(rows) * k_pad * 4 + (mn ? static_cast<size_t>(kSimtWarps) * rows * 128 * 4 : 0);
}

template <int R>
int launch_simt(const SimtArgs &p, int mn, bool vec, int blocks, cudaStream_t stream)
{
    auto kernel = mn ? (vec ? few_simt_cols_kernel<R, true> : few_simt_cols_kernel<R, false>)
                     : (vec ? few_simt_rows_kernel<R, true> : few_simt_rows_kernel<R, false>);
    const size_t smem = simt_smem(R, p.k_pad, mn);
    if (smem > 48 * 1024)
        ODL_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    kernel<<<blocks, 32 * kSimtWarps, smem, stream>>>(p);
    ++g_launch_count;
    ODL_CUDA_TRY(cudaGetLastError());
    return kOk;
}

int simt_rows(int64_t M)
{
    return M <= 1 ? 1 : M <= 2 ? 2 : M <= 4 ? 4 : 8;
}

bool simt_fits(int64_t M, int64_t K, int mn)
{
    return M <= kSimtRows && K <= 65536 && simt_smem(simt_rows(M), static_cast<int>((K + 31) / 32 * 32), mn) <= 200 * 1024;
}

template <int NX, int TERMS>
int launch_few(const FewTmaps &tm, const FewArgs &p, cudaStream_t stream)
{
    using C = FewCfg<NX, TERMS>;
    static bool set = false;
    if (!set)
    {
        ODL_CUDA_TRY(cudaFuncSetAttribute(few_logits_kernel<NX, TERMS>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::smem));
        set = true;
    }
    few_logits_kernel<NX, TERMS><<<p.parts / kDrain, kThreads, C::smem, stream>>>(tm, p);
    ++g_launch_count;
    ODL_CUDA_TRY(cudaGetLastError());
    return kOk;
}
}  // namespace

// Up to 8 rows any weights do; above, TMA reads the weights as they are: rows of a multiple of 16 bytes from a 16-byte boundary.
bool linear_ce_few_eligible(int64_t M, int64_t N, int64_t K, const float *w, int w_layout)
{
    if (simt_fits(M, K, w_layout == ODL_W_IN_OUT) && N <= 0x7fffff00)
        return true;
    const int64_t ld = w_layout == ODL_W_OUT_IN ? K : N;
    return M <= kRowsMost && !(ld & 3) && !(reinterpret_cast<uintptr_t>(w) & 15) && N <= 0x7fffff00;
}

int linear_ce_few(const float *x, const float *w, const float *b, const void *labels, int is64, int64_t ignore_index, int64_t M, int64_t N,
                  int64_t K, int w_layout, float *loss, float *lse_out, int precision, cudaStream_t stream)
{
    const int mn    = w_layout == ODL_W_IN_OUT;
    const bool simt = simt_fits(M, K, mn);
    const int nx    = simt ? simt_rows(M) : M <= 16 ? 16 : M <= 32 ? 32 : 64;
    const int rows  = nx < 32 ? 32 : nx;
    const int k_pad = static_cast<int>((K + 31) / 32 * 32);
    const int sms   = s16::sm_count();
    int ctas, parts;
    if (simt)
    {
        // as many blocks as run at once (2048 threads an SM), a warp (block) for every group of classes at most
        const size_t smem   = simt_smem(nx, k_pad, mn);
        const int per_sm    = smem <= 50 * 1024 ? 4 : smem <= 100 * 1024 ? 2 : 1;
        const int64_t units = mn ? (N + 127) / 128 : (N + (nx <= 4 ? 8 : 4) * kSimtWarps - 1) / ((nx <= 4 ? 8 : 4) * kSimtWarps);
        ctas                = static_cast<int>(units < sms * per_sm ? units : sms * per_sm);
        parts               = ctas * (mn ? 4 : kSimtWarps);
    }
    else
    {
        const int64_t grans = (N + (mn ? 31 : 15)) / (mn ? 32 : 16);
        ctas                = static_cast<int>(grans < sms ? grans : sms);
        parts               = ctas * kDrain;
    }
    const size_t xb = a256(static_cast<size_t>(nx) * k_pad * 4);
    int rc = arena_begin(2 * xb + a256(static_cast<size_t>(rows) * parts * 8) + 5 * 512, stream);
    if (rc)
        return rc;
    const ArenaUse use{stream};
    float *big      = static_cast<float *>(arena_alloc(xb));
    float *small    = static_cast<float *>(arena_alloc(xb));
    float2 *part    = static_cast<float2 *>(arena_alloc(static_cast<size_t>(rows) * parts * 8));
    int *idx        = static_cast<int *>(arena_alloc(kRowsMost * 4));
    int *cls        = static_cast<int *>(arena_alloc(kRowsMost * 4));
    float *picked   = static_cast<float *>(arena_alloc(kRowsMost * 4));
    float *row_loss = static_cast<float *>(arena_alloc(kRowsMost * 4));
    FewWords *words = static_cast<FewWords *>(arena_alloc(sizeof(FewWords)));
    const int64_t blocks = (static_cast<int64_t>(nx) * k_pad + 1023) / 1024;
    few_rows_kernel<<<(int)(blocks < 592 ? blocks : 592), 256, 0, stream>>>(x, labels, is64, ignore_index, (int)M, (int)N, (int)K, nx, k_pad, big, small,
                                                                           idx, cls, words, lse_out);
    ++g_launch_count;
    ODL_CUDA_TRY(cudaGetLastError());
    if (simt)
    {
        const SimtArgs a{w, big, b, cls, words, part, picked, (int)N, (int)K, k_pad, parts};
        const bool vec = !((mn ? N : K) & 3) && !(reinterpret_cast<uintptr_t>(w) & 15);
        rc = nx == 1 ? launch_simt<1>(a, mn, vec, ctas, stream) : nx == 2 ? launch_simt<2>(a, mn, vec, ctas, stream)
           : nx == 4 ? launch_simt<4>(a, mn, vec, ctas, stream) : launch_simt<8>(a, mn, vec, ctas, stream);
        if (rc)
            return rc;
        few_finish_kernel<<<(int)M, 256, 0, stream>>>(part, parts, idx, picked, words, row_loss, lse_out, loss, device_error_flag());
        ++g_launch_count;
        ODL_CUDA_TRY(cudaGetLastError());
        return kOk;
    }
    FewTmaps tm;
    std::memset(&tm, 0, sizeof(tm));
    if ((rc = mn ? make_tmap(&tm.w, w, K, N, N, 32, 32, CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B) : make_tmap(&tm.w, w, N, K, K, 32, 16, CU_TENSOR_MAP_SWIZZLE_128B)) ||
        (rc = make_tmap(&tm.x, big, nx, k_pad, k_pad, 32, nx, CU_TENSOR_MAP_SWIZZLE_128B)) ||
        (rc = make_tmap(&tm.x_small, small, nx, k_pad, k_pad, 32, nx, CU_TENSOR_MAP_SWIZZLE_128B)))
        return rc;
    const FewArgs p{b, cls, words, part, picked, device_error_flag(), (int)N, (int)K, mn, parts};
    if (precision == ODL_PRECISION_3XTF32)
        rc = nx == 16 ? launch_few<16, 3>(tm, p, stream) : nx == 32 ? launch_few<32, 3>(tm, p, stream) : launch_few<64, 3>(tm, p, stream);
    else
        rc = nx == 16 ? launch_few<16, 1>(tm, p, stream) : nx == 32 ? launch_few<32, 1>(tm, p, stream) : launch_few<64, 1>(tm, p, stream);
    if (rc)
        return rc;
    few_finish_kernel<<<(int)M, 256, 0, stream>>>(part, parts, idx, picked, words, row_loss, lse_out, loss, device_error_flag());
    ++g_launch_count;
    ODL_CUDA_TRY(cudaGetLastError());
    return kOk;
}

}  // namespace odl
