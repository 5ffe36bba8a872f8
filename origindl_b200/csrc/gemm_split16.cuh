// GEMM on fp32 values carried as two halves: v = s (hi + lo), hi = fp16(v / s), lo = fp16(v / s - hi), with a power of two
// s, so that hi + lo holds 22 bits of v (relative error 2^-23) down to 2^-39 of the largest value s allows.  The product of
// two such matrices is three fp16 products, hi hi + lo hi + hi lo (the dropped lo lo is at most 2^-22), with fp32
// accumulation: the accuracy of the 3xTF32 GEMM at twice its rate, since tcgen05 multiplies fp16 twice as fast as tf32 and
// both have 11-bit significands.  fp16's short exponent is what s is for: an operand has one s for all of it (Newton-Schulz
// iterates, whose entries are bounded; softmax probabilities) or one for each 128 x 128 tile (see Split16 below).
//
// Layout of a split matrix of R rows and C columns (C padded to a multiple of 64 with zeros): row after row, and within a
// row, block of 64 columns after block, [64 hi][64 lo]: 256 bytes, exactly the bytes of the 64 fp32 values, so that a matrix
// can be split in place.  The same layout is read K-major (reduction along a row) and MN-major (reduction over the rows).
//
// The kernel: persistent, one CTA (128 x BN tiles) or a CTA pair (256 x 256, tcgen05 cta_group::2) per SM (pair), warp 0 feeds a
// ring of 64-deep K-blocks by TMA (no multicast), one thread of warp 1 issues the MMAs, eight warps drain the accumulator.
// TMEM accumulation truncates (a step of the accumulator per instruction, always towards zero), so an accumulator holds little of
// the reduction: two TMEM buffers alternate, and the drain adds them up in fp32 registers, scaled by the tiles' s where the
// operands have many.  Of each K-block the small products go first, so that only four instructions truncate at full size.  A loss
// takes chunks of 128, which its tile scales cover; Newton-Schulz, whose steps amplify errors, 64 (five steps of 300 x 900: 1.7e-6
// off in the 2-norm, 3.7e-6 with 128; plain fp32 products 2.0e-6).  The epilogue holds up the drain (8 to 18 thousand cycles a
// tile, when all SMs store at once, against 1536 a K-block) and the MMA thread runs only two chunks ahead of it: long
// reductions without scales begin with two chunks of 128.
// Every wait is bounded; a wait that gives up raises the abort flag, which releases the others, and the error flag.
#pragma once
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>

#include "gemm_tc.cuh"
#include "host_util.h"
#include "ptx_sm100.cuh"
#include "tmap.h"

namespace odl
{
namespace s16
{

constexpr int kBK      = 64;   // reduction per stage: 128 bytes of halves
constexpr int kEpi     = 8;    // epilogue warps
constexpr int kThreads = 64 + 32 * kEpi;
constexpr int kGroupM  = 8;    // row tiles walked together (their operand panels stay in L2)
constexpr int kSlab    = 32 * 33 * 4;

// a split matrix in memory
struct Split16
{
    const __half *data = nullptr;
    int64_t pitch      = 0;        // halves from row to row (2 * padded columns)
    int rows = 0, cols_pad = 0;
    int batch            = 1;
    int64_t batch_stride = 0;      // halves
    const float *scale   = nullptr;  // s of each 128 x 128 tile, [ceil(rows / 128)][ceil(cols_pad / 128)]; nullptr: one s, in `alpha`
};

inline int pad64(int64_t c)
{
    return static_cast<int>((c + 63) & ~int64_t(63));
}

struct GemmArgs
{
    int M, N, K;               // of op(A) op(B); upper bounds where `count` limits one of them
    int a_mn, b_mn;            // operand's reduction runs over its rows
    int batch, splits;         // splits: slices of the reduction, summed by whoever reads the slices
    int sym;                   // only tiles on and above the diagonal (the epilogue writes both halves)
    const int *count;          // device: rows that exist from row 0 of the whole batch; nullptr = all
    int count_base, count_dim; // this call starts at count_base; 1: limits M, 2: limits K
    const float *sa, *sb;      // per-tile scales or nullptr
    int diag;                  // where B's 128 x 128 blocks on the diagonal differ: they come from the third map, [rows][128]
    int lda_s, ldb_s;
    int *err;
};

struct Tmaps
{
    CUtensorMap a, b, d;
};

__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void mma_f16_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}
// kind::f16, both operands fp16 (format 0), fp32 accumulator
__device__ __forceinline__ uint32_t idesc_f16(int m, int n, bool a_mn, bool b_mn)
{
    return (1u << 4) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
           (static_cast<uint32_t>(m >> 4) << 24);
}

// hi and lo of two values, packed as half2 words
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo)
{
    const __half2 h  = __floats2half2_rn(a, b);
    const float2 f   = __half22float2(h);
    const __half2 l  = __floats2half2_rn(a - f.x, b - f.y);
    hi               = *reinterpret_cast<const uint32_t *>(&h);
    lo               = *reinterpret_cast<const uint32_t *>(&l);
}

// 32 lanes x 8 consecutive 32-bit columns of TMEM
__device__ __forceinline__ void tmem_ld_32x8(uint32_t taddr, uint32_t (&r)[8])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}

// 2^x to 2^-22 of itself, 0 below the normal range
__device__ __forceinline__ float fast_exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Programmatic launches: a kernel of these operators may be resident before the one in front of it has finished; it sets itself
// up (barriers, TMEM, tensor maps) and then waits here for that one's results.  Every kernel launched with launch_after() calls
// both, so that completion carries over from kernel to kernel.
__device__ __forceinline__ void after_previous()
{
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void let_next_in()
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <int CG, int BN, int TERMS>
struct Cfg
{
    static constexpr int a_bytes = 128 * kBK * 2;
    static constexpr int bn_cta  = CG == 2 ? BN / 2 : BN;  // rows of B this CTA holds
    static constexpr int b_bytes = bn_cta * kBK * 2;
    static constexpr int parts   = TERMS == 3 ? 2 : 1;
    static constexpr int stage   = parts * (a_bytes + b_bytes);
    static constexpr int stages  = 192 * 1024 / stage > 8 ? 8 : 192 * 1024 / stage;
    static constexpr int smem    = 1024 + stages * stage + kEpi * kSlab + 512;
    static constexpr int strip   = BN / 2;  // columns of the tile one epilogue warp holds
};

// K-blocks of a tile's c-th chunk (what one accumulator buffer holds) of n
template <bool SCALED>
__device__ __forceinline__ int chunk_blocks(int c, int n)
{
    return SCALED || (c < 2 && n >= 16) ? 2 : 1;
}

// what the epilogue is told about a tile
struct TileAt
{
    int row;        // of this thread in op(A) op(B)
    int rows;       // M in force
    int col;        // first column of this warp's strip
    int strip;      // index of the strip over the whole matrix (columns / strip width)
    int batch, split;
    int tm, tn;     // tile (symmetric outputs: tm == tn is written once)
    int lane;
};

template <int CG, int BN, int TERMS, bool SCALED, class Epi>
__global__ void __launch_bounds__(kThreads, 1)
gemm_split16_kernel(const __grid_constant__ Tmaps tm, const GemmArgs g, const typename Epi::Params ep)
{
    using C = Cfg<CG, BN, TERMS>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *tiles      = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float *slabs        = reinterpret_cast<float *>(tiles + C::stages * C::stage);
    uint64_t *full_bar  = reinterpret_cast<uint64_t *>(tiles + C::stages * C::stage + kEpi * kSlab);
    uint64_t *empty_bar = full_bar + C::stages;  // a stage's MMAs are complete: its buffers are free
    uint64_t *acc_full  = empty_bar + C::stages;
    uint64_t *acc_empty = acc_full + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + 2);
    volatile int *abort_f = reinterpret_cast<volatile int *>(tmem_slot + 1);
    int *early_out        = const_cast<int *>(abort_f) + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CG == 2 ? ptx::cluster_ctarank() : 0u;
    const bool leader   = rank == 0;

    let_next_in();
    if (threadIdx.x == 0)
    {
        *early_out = (leader && *reinterpret_cast<volatile int *>(g.err) == 1) ? 1 : 0;  // an earlier wait gave up
        *abort_f   = 0;
        for (int s = 0; s < C::stages; ++s)
        {
            ptx::mbar_init(&full_bar[s], 1);
            ptx::mbar_init(&empty_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b)
        {
            ptx::mbar_init(&acc_full[b], 1);
            ptx::mbar_init(&acc_empty[b], CG * kEpi);
        }
        ptx::fence_mbar_init();
        ptx::prefetch_tmap(&tm.a);
        ptx::prefetch_tmap(&tm.b);
    }
    if (warp == 1)
    {
        if (CG == 2)
        {
            ptx::tmem_alloc_pair(tmem_slot, 2 * BN);
            ptx::tmem_relinquish_pair();
        }
        else
        {
            ptx::tmem_alloc(tmem_slot, 2 * BN);
            ptx::tmem_relinquish();
        }
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    if (CG == 2)
        ptx::cluster_sync();
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    const bool skip = CG == 2 ? ptx::ld_shared_cluster_u32(ptx::map_to_cta(ptx::smem_u32(early_out), 0)) != 0 : *early_out != 0;

    after_previous();
    int M = g.M, K = g.K;
    if (g.count)
    {
        const int left = *g.count - g.count_base;
        if (g.count_dim == 1)
            M = max(0, min(M, left));
        else
            K = max(0, min(K, left));
    }
    const int tiles_m  = (M + CG * 128 - 1) / (CG * 128);
    const int tiles_n  = (g.N + BN - 1) / BN;
    const int n_tiles  = g.sym ? tiles_n * (tiles_n + 1) / 2 : tiles_m * tiles_n;
    // (a later piece of the reduction with no row left adds nothing)
    const int n_units  = g.count && g.count_dim == 2 && g.count_base > 0 && K == 0 ? 0 : n_tiles * g.splits * g.batch;
    const int n_kb     = (K + kBK - 1) / kBK;
    const int kb_slice = ((n_kb + g.splits - 1) / g.splits + 1) & ~1;  // (whole chunks)
    const int first    = blockIdx.x / CG, step = gridDim.x / CG;

    auto decode = [&](int u, int &t_m, int &t_n, int &kb0, int &kb1, int &batch, int &split) {
        int t = u;
        split = batch = 0;
        if (u >= n_tiles)
        {
            u /= n_tiles;
            t -= u * n_tiles;
            batch = u;
            if (g.splits > 1)
            {
                batch = u / g.splits;
                split = u - batch * g.splits;
            }
        }
        kb0   = min(n_kb, split * kb_slice);
        kb1   = min(n_kb, kb0 + kb_slice);
        if (g.sym)
        {
            // t = t_n (t_n + 1) / 2 + t_m, t_m <= t_n
            int n = static_cast<int>((sqrtf(8.f * static_cast<float>(t) + 1.f) - 1.f) * 0.5f);
            while (n * (n + 1) / 2 > t)
                --n;
            while ((n + 1) * (n + 2) / 2 <= t)
                ++n;
            t_n = n;
            t_m = t - n * (n + 1) / 2;
        }
        else
        {
            const int per_group = kGroupM * tiles_n;
            const int grp       = t / per_group;
            const int gsz       = min(tiles_m - grp * kGroupM, kGroupM);
            const int local     = t - grp * per_group;
            t_n                 = local / gsz;
            t_m                 = grp * kGroupM + local - t_n * gsz;
        }
    };

    if (skip)
    {
        // nothing
    }
    else if (warp == 0)
    {
        // ================================================================= TMA producer (every CTA)
        if (lane == 0)
        {
            uint32_t gk = 0;
            bool ok     = true;
            for (int u = first; ok && u < n_units; u += step)
            {
                int t_m, t_n, kb0, kb1, batch, split;
                decode(u, t_m, t_n, kb0, kb1, batch, split);
                const int m0 = (t_m * CG + static_cast<int>(rank)) * 128;
                const int b0 = t_n * BN + static_cast<int>(rank) * C::bn_cta;
                for (int kb = kb0; kb < kb1; ++kb, ++gk)
                {
                    const int s = gk % C::stages;
                    if (!ptx::mbar_wait(&empty_bar[s], ((gk / C::stages) & 1) ^ 1, abort_f))
                    {
                        ok = false;
                        break;
                    }
                    if (leader)
                        ptx::mbar_arrive_expect_tx(&full_bar[s], CG * C::stage);
                    const uint32_t bar = CG == 2 ? ptx::map_to_cta(ptx::smem_u32(&full_bar[s]), 0) : 0u;
                    auto load          = [&](uint8_t *dst, const CUtensorMap *map, int x, int y) {
                        if (CG == 2)
                            ptx::tma_load_3d_pair(dst, map, bar, x, y, batch);
                        else
                            ptx::tma_load_3d(dst, map, &full_bar[s], x, y, batch);
                    };
                    uint8_t *st = tiles + s * C::stage;
#pragma unroll
                    for (int p = 0; p < C::parts; ++p)
                    {
                        // x in halves: block of 64 columns b starts at 128 b, its lo part 64 further
                        uint8_t *sa = st + p * C::a_bytes;
                        if (!g.a_mn)
                            load(sa, &tm.a, 128 * kb + 64 * p, m0);
                        else
                            for (int j = 0; j < 2; ++j)
                                load(sa + j * 8192, &tm.a, 2 * m0 + 128 * j + 64 * p, kb * kBK);
                        uint8_t *sb = st + C::parts * C::a_bytes + p * C::b_bytes;
                        if (g.diag && (kb >> 1) == (b0 >> 7))
                            load(sb, &tm.d, 128 * (kb & 1) + 64 * p, b0);
                        else if (!g.b_mn)
                            load(sb, &tm.b, 128 * kb + 64 * p, b0);
                        else
                            for (int j = 0; j < C::bn_cta / 64; ++j)
                                load(sb + j * 8192, &tm.b, 2 * b0 + 128 * j + 64 * p, kb * kBK);
                    }
                }
            }
            if (*abort_f && leader)
            {
                // let the copies still in flight land before the CTA goes away
                const uint32_t from = gk > C::stages ? gk - C::stages : 0;
                for (uint32_t k = from; k < gk; ++k)
                    ptx::mbar_wait(&full_bar[k % C::stages], (k / C::stages) & 1, nullptr);
            }
        }
    }
    else if (warp == 1)
    {
        // ================================================================= MMA issuer (leader)
        if (lane == 0 && leader)
        {
            const uint32_t idesc = idesc_f16(CG * 128, BN, g.a_mn != 0, g.b_mn != 0);
            // 16 of the reduction: 32 bytes along a 128-byte row (K-major), 16 rows of 128 bytes (MN-major); MN-major
            // operands are boxes of 64 columns, 8192 bytes apart
            const uint32_t a_step = g.a_mn ? 2048u : 32u, b_step = g.b_mn ? 2048u : 32u;
            const uint32_t a_lbo = g.a_mn ? 8192u : 16u, b_lbo = g.b_mn ? 8192u : 16u;
            uint32_t gk = 0, gc = 0;
            bool ok     = true;
            for (int u = first; ok && u < n_units; u += step)
            {
                int t_m, t_n, kb0, kb1, batch, split;
                decode(u, t_m, t_n, kb0, kb1, batch, split);
                int c = 0, chunk_end = kb0;
                for (int kb = kb0; kb < kb1; ++kb, ++gk)
                {
                    const bool opens = kb == chunk_end;
                    if (opens)
                    {
                        chunk_end = min(kb1, kb + chunk_blocks<SCALED>(c++, kb1 - kb0));
                        if (!ptx::mbar_wait(&acc_empty[gc & 1], ((gc >> 1) & 1) ^ 1, abort_f))
                        {
                            ok = false;
                            break;
                        }
                    }
                    const int buf = gc & 1, s = gk % C::stages;
                    if (!ptx::mbar_wait(&full_bar[s], (gk / C::stages) & 1, abort_f))
                    {
                        ok = false;
                        break;
                    }
                    ptx::tc_fence_after_sync();
                    const uint32_t d  = tmem_base + buf * BN;
                    const uint32_t sa = ptx::smem_u32(tiles + s * C::stage);
                    const uint32_t sb = sa + C::parts * C::a_bytes;
                    auto mma          = [&](uint32_t a, uint32_t b, uint32_t acc) {
                        const uint64_t da = ptx::make_smem_desc(a, a_lbo, 1024, ptx::kLayoutSw128);
                        const uint64_t db = ptx::make_smem_desc(b, b_lbo, 1024, ptx::kLayoutSw128);
                        if (CG == 2)
                            mma_f16_pair(d, da, db, idesc, acc);
                        else
                            mma_f16(d, da, db, idesc, acc);
                    };
                    if (TERMS == 3)
                    {
#pragma unroll
                        for (int k = 0; k < kBK / 16; ++k)
                        {
                            mma(sa + C::a_bytes + k * a_step, sb + k * b_step, !opens || k != 0);
                            mma(sa + k * a_step, sb + C::b_bytes + k * b_step, 1);
                        }
                    }
#pragma unroll
                    for (int k = 0; k < kBK / 16; ++k)
                        mma(sa + k * a_step, sb + k * b_step, TERMS == 3 || !opens || k != 0);
                    if (CG == 2)
                        ptx::mma_commit_pair_both(&empty_bar[s]);
                    else
                        ptx::mma_commit(&empty_bar[s]);
                    if (kb + 1 == chunk_end)
                    {
                        if (CG == 2)
                            ptx::mma_commit_pair_both(&acc_full[buf]);
                        else
                            ptx::mma_commit(&acc_full[buf]);
                        ++gc;
                    }
                }
            }
        }
    }
    else
    {
        // ================================================================= drain + epilogue (warps 2..9)
        const int e = warp - 2, q = warp & 3, h = e >> 2;  // TMEM lanes 32 q .. 32 q + 31, strip h
        float *slab = slabs + e * (kSlab / 4);
        float acc[C::strip];
        uint32_t gc = 0;
        bool ok     = true;
        for (int u = first; ok && u < n_units; u += step)
        {
            TileAt at;
            int kb0, kb1;
            decode(u, at.tm, at.tn, kb0, kb1, at.batch, at.split);
            const int m0 = (at.tm * CG + static_cast<int>(rank)) * 128;
            at.row       = m0 + 32 * q + lane;
            at.rows      = M;
            at.col       = at.tn * BN + h * C::strip;
            at.strip     = at.tn * 2 + h;
            at.lane      = lane;
#pragma unroll
            for (int i = 0; i < C::strip; ++i)
                acc[i] = 0.f;
            // scales: one of A's 128 rows, one of B's 128 columns (a strip crosses no block of 128)
            const float *pa = nullptr, *pb = nullptr;
            if (SCALED)
            {
                const int m = min(m0, M - 1) >> 7, n = min(at.col, g.N - 1) >> 7;
                pa          = g.sa ? g.sa + (g.a_mn ? m : m * g.lda_s) : nullptr;
                pb          = g.sb ? g.sb + (g.b_mn ? n : n * g.ldb_s) : nullptr;
            }
            for (int kb = kb0, c = 0; kb < kb1; ++c, ++gc)
            {
                const int buf = gc & 1;
                float f       = 1.f;
                if (SCALED)
                {
                    const int k = kb >> 1;
                    f           = (pa ? __ldg(pa + (g.a_mn ? k * g.lda_s : k)) : 1.f) * (pb ? __ldg(pb + (g.b_mn ? k * g.ldb_s : k)) : 1.f);
                }
                kb += chunk_blocks<SCALED>(c, kb1 - kb0);
                ok = __all_sync(0xffffffffu, ptx::mbar_wait(&acc_full[buf], (gc >> 1) & 1, abort_f));
                if (!ok)
                    break;
                ptx::tc_fence_after_sync();
                const uint32_t taddr = tmem_base + (static_cast<uint32_t>(32 * q) << 16) + buf * BN + h * C::strip;
#pragma unroll
                for (int j = 0; j < C::strip / 32; ++j)
                {
                    uint32_t r[32];
                    ptx::tmem_ld_32x32(taddr + 32 * j, r);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        acc[32 * j + i] = SCALED ? fmaf(__uint_as_float(r[i]), f, acc[32 * j + i])
                                                 : acc[32 * j + i] + __uint_as_float(r[i]);
                }
                ptx::tc_fence_before_sync();
                __syncwarp();
                if (lane == 0)
                {
                    if (CG == 2)
                        ptx::mbar_arrive_cluster_relaxed(ptx::map_to_cta(ptx::smem_u32(&acc_empty[buf]), 0));
                    else
                        ptx::mbar_arrive(&acc_empty[buf]);
                }
            }
            if (ok)
                Epi::template store<C::strip>(ep, g, at, acc, slab);
        }
        ptx::tc_fence_before_sync();
    }

    __syncthreads();
    if (CG == 2)
        ptx::cluster_sync();
    if (warp == 1)
    {
        __syncwarp();
        ptx::tc_fence_after_sync();
        if (CG == 2)
            ptx::tmem_dealloc_pair(tmem_base, 2 * BN);
        else
            ptx::tmem_dealloc(tmem_base, 2 * BN);
    }
    if (threadIdx.x == 0 && *abort_f)
        atomicExch(g.err, 1);
}

// ---- epilogue helpers: one warp, thread = row, N consecutive columns in registers -------------------------------------------
// 32 rows x 32 columns out of registers through a padded slab, so that a warp instruction writes (reads) 128 bytes of a row.
// put(row in 0..31, value of column `lane`) is called row by row.
template <class Put>
__device__ __forceinline__ void by_rows(const float *v, float *slab, int lane, Put &&put)
{
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 32; ++i)
        slab[lane * 33 + i] = v[i];
    __syncwarp();
#pragma unroll 4
    for (int r = 0; r < 32; ++r)
        put(r, slab[r * 33 + lane]);
}

// ---- host side ------------------------------------------------------------------------------------------------------------
int make_tmap_split16(CUtensorMap *out, const Split16 &m, int box_rows);
int sm_count();
int resident_ctas(const void *kernel, int cluster, int smem);

// kernel<<<grid, block, smem, stream>>>(args...) as a programmatic launch (see after_previous)
template <class... P, class... A>
int launch_after(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, A... args)
{
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim          = grid;
    cfg.blockDim         = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream           = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs       = attr;
    cfg.numAttrs    = 1;
    cudaError_t e   = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
    ++g_launch_count;
    if (e != cudaSuccess)
    {
        set_last_error("kernel launch failed: %s", cudaGetErrorString(e));
        return kCudaError;
    }
    return kOk;
}

template <int CG, int BN, int TERMS, bool SCALED, class Epi>
int launch(const Split16 &A, const Split16 &B, GemmArgs g, const typename Epi::Params &ep, cudaStream_t stream, const Split16 *D)
{
    using C     = Cfg<CG, BN, TERMS>;
    auto kernel = gemm_split16_kernel<CG, BN, TERMS, SCALED, Epi>;
    Tmaps tm;
    int rc;
    if ((rc = make_tmap_split16(&tm.a, A, g.a_mn ? kBK : 128)) || (rc = make_tmap_split16(&tm.b, B, g.b_mn ? kBK : C::bn_cta)))
        return rc;
    tm.d   = tm.b;
    g.diag = D != nullptr;
    if (D && (rc = make_tmap_split16(&tm.d, *D, C::bn_cta)))
        return rc;
    g.sa = A.scale, g.lda_s = (A.cols_pad + 127) / 128;
    g.sb = B.scale, g.ldb_s = (B.cols_pad + 127) / 128;
    static int resident = 0;  // CTAs (pairs) the GPU holds at once; one device per process
    if (resident == 0)
    {
        if ((rc = resident_ctas(reinterpret_cast<const void *>(kernel), CG, C::smem)) <= 0)
            return kCudaError;
        resident = rc;
    }
    const int64_t tm_ = (g.M + CG * 128 - 1) / (CG * 128), tn_ = (g.N + BN - 1) / BN;
    const int64_t units = (g.sym ? tn_ * (tn_ + 1) / 2 : tm_ * tn_) * g.splits * g.batch;
    if (units > 0x3fffffff)
    {
        set_last_error("gemm: %lld tiles exceed 2^30", (long long)units);
        return kTooLarge;
    }
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim          = dim3(static_cast<unsigned>(CG * (units < resident ? units : resident)), 1, 1);
    cfg.blockDim         = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = C::smem;
    cfg.stream           = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id               = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = CG;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs                = attr;
    cfg.numAttrs             = 2;
    cudaError_t e            = cudaLaunchKernelEx(&cfg, kernel, tm, g, ep);
    ++g_launch_count;
    if (e != cudaSuccess)
    {
        set_last_error("gemm_split16_kernel launch failed: %s", cudaGetErrorString(e));
        return kCudaError;
    }
    return kOk;
}

// Which tile and how many slices of the reduction, by the estimate in plan_tiles.
struct Plan
{
    int cg = 2, bn = 256, splits = 1;
    int tiles_n(int64_t n) const { return static_cast<int>((n + bn - 1) / bn); }
};
Plan plan_tiles(int64_t M, int64_t N, int64_t K, int terms, int batch, bool may_split, bool sym = false);

template <int TERMS, bool SCALED, class Epi>
int launch_plan(const Plan &plan, const Split16 &A, const Split16 &B, const GemmArgs &g, const typename Epi::Params &ep, cudaStream_t stream,
                const Split16 *D = nullptr)
{
    if (plan.cg == 2)
        return launch<2, 256, TERMS, SCALED, Epi>(A, B, g, ep, stream, D);
    if constexpr (!Epi::kSquare)  // (a symmetric output has square tiles)
        if (plan.bn == 64)
            return launch<1, 64, TERMS, SCALED, Epi>(A, B, g, ep, stream, D);
    return launch<1, 128, TERMS, SCALED, Epi>(A, B, g, ep, stream, D);
}

}  // namespace s16
}  // namespace odl
