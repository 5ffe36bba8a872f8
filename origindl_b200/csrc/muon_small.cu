// Newton-Schulz and the Muon step for matrices with a side of at most 128: one launch for everything.
//
// A matrix belongs to a cluster of 1 to 8 CTAs.  X (taken with its short side as rows) lies in their shared memory for the whole
// iteration, split-fp16 (gemm_split16.cuh, muon.cu), each CTA holding a range of columns; nothing but the gradient, the momentum
// and the result touches global memory.  A step in each CTA:
//   partial A = X_loc X_loc^T      (X_loc read K-major twice; as many accumulators as TMEM holds, so that each sums few blocks of 64)
//   A = sum over the cluster       (each CTA adds a slice of columns of all partials in rank order, and writes its halves to all)
//   S = a I + b A + c A^2          (every CTA the whole of it: 24 MMAs, less than moving it)
//   X_loc = S X_loc                (the same X_loc read MN-major)
// A product of 128 x 128 takes under a microsecond here, so the steps' latencies (commit, TMEM reads, two cluster barriers)
// bound the kernel; the form of three GEMM launches per step pays set-up, ring fill and global stores 3 * steps times instead.
// 128 x 128: 59 us for five steps (the chain of launches 122), 32 of 64 x 512 52 us (116), 15 of 5 x 5888 92 us (414).
// The waits on the tensor core are bounded; one that gives up raises the error flag and the kernel runs on to its end (the cluster
// barriers need every CTA).
#include <cuda_runtime.h>

#include <cmath>
#include <cstring>
#include <type_traits>

#include "gemm_split16.cuh"
#include "host_util.h"
#include "internal.h"
#include "muon.h"
#include "ptx_sm100.cuh"

namespace odl
{

namespace
{
constexpr int kThreads = 256;
constexpr int kMaxCluster = 8;

struct SmallArgs
{
    const float *p;
    float *g, *buf;
    MomentumArgs m;
    NsOut out;
    int *err;
    int rows, cols;  // as stored
    int s, l;        // short and long side
    int s_pad;       // s rounded up to 16
    int blocks;      // blocks of 64 columns per CTA
    int cluster, steps, terms;
    float eps;
};

// RB: rows of a block in shared memory (16, 32, 64 or 128); the MMAs' M is 128 whatever RB, rows past RB are whatever follows (their
// accumulator lanes are not read).  A, S and the partial A in fp32 take turns in one place: the partial sums are read before A is
// written, and every thread writes the elements of S over the ones of A that it has just read.
template <int RB>
struct SmallCfg
{
    static constexpr int block = RB * 128;                           // bytes of 64 columns of halves
    static constexpr int sq    = RB > 64 ? 2 * block : block;        // bytes of an RB x RB matrix of halves
    static constexpr int accs  = 512 / RB;                           // accumulators of partial A in TMEM
    // X: hi blocks, lo blocks; A / S: hi, lo; the cluster's reduced slices of A (fp32)
    __host__ __device__ static constexpr int x_lo(int blocks) { return blocks * block; }
    __host__ __device__ static constexpr int a_hi(int blocks) { return 2 * blocks * block; }
    __host__ __device__ static constexpr int red(int blocks) { return a_hi(blocks) + 2 * sq; }
    // (an M = 128 read of the last matrix ends 128 rows from its start)
    __host__ __device__ static constexpr int aux(int blocks, int cluster)
    {
        const int r = cluster > 1 ? RB * RB * 4 / cluster : 0, past = (128 - RB) * 128;
        return red(blocks) + (r > past ? r : past);
    }
    __host__ __device__ static constexpr int bytes(int blocks, int cluster) { return 1024 + aux(blocks, cluster) + 512; }
    __host__ __device__ static constexpr bool fits(int blocks, int cluster) { return bytes(blocks, cluster) <= 227 * 1024; }
};

// byte of element (row, col) inside a matrix of 64-column blocks, 128-byte swizzle
template <int RB>
__device__ __forceinline__ uint32_t place(int row, int col)
{
    return static_cast<uint32_t>((col >> 6) * SmallCfg<RB>::block + row * 128 + ((((col & 63) >> 3) ^ (row & 7)) << 4) + (col & 7) * 2);
}

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
    return v;
}

template <int RB>
__global__ void __launch_bounds__(kThreads, 1) muon_small_kernel(const SmallArgs p)
{
    using C = SmallCfg<RB>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *sm         = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int o_xlo = C::x_lo(p.blocks), o_ahi = C::a_hi(p.blocks), o_alo = o_ahi + C::sq, o_red = C::red(p.blocks), o_aux = C::aux(p.blocks, p.cluster);
    uint64_t *bar       = reinterpret_cast<uint64_t *>(sm + o_aux);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bar + 1);
    volatile int *abort_f = reinterpret_cast<volatile int *>(tmem_slot + 1);
    double *box           = reinterpret_cast<double *>(sm + o_aux + 32);   // [8] warps
    double *cl_box        = reinterpret_cast<double *>(sm + o_aux + 128);  // this CTA's sum of squares
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank   = static_cast<int>(ptx::cluster_ctarank());
    const int matrix = blockIdx.x / p.cluster;
    const bool tall  = p.rows > p.cols;
    const int64_t off = static_cast<int64_t>(matrix) * p.rows * p.cols;
    const int j0 = rank * p.blocks * 64, n_loc = p.blocks * 64;  // this CTA's columns of the wide form

    if (tid == 0)
    {
        *abort_f = 0;
        ptx::mbar_init(bar, 1);
        ptx::fence_mbar_init();
    }
    if (warp == 0)
    {
        ptx::tmem_alloc(tmem_slot, 512);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    const uint32_t base = ptx::smem_u32(sm);

    // ---- momentum and the norm -------------------------------------------------------------------------------------------------
    // A thread's elements come in pairs along the long side (columns j, j + 1 of the wide form), N pairs at a time, their loads
    // unconditional (from the matrix's first element where there is nothing) so that they are in flight together.  As stored wide
    // a warp covers 64 columns of a row, a batch 8 rows; as stored tall a warp covers 4 short-side by 8 pairs (a compromise of
    // 16-byte pieces of global rows and of shared-memory banks), a batch 64 columns.
    auto batches = [&](auto &&body) {
        if (!tall)
        {
#pragma unroll 1
            for (int b = 0; b < p.blocks; ++b)
#pragma unroll 1
                for (int i = warp; i < RB; i += 64)
                    body(std::integral_constant<bool, false>(), std::integral_constant<int, (RB < 64 ? RB / 8 : 8)>(), i, 64 * b + 2 * lane);
        }
        else
        {
#pragma unroll 1
            for (int i = 4 * warp + (lane >> 3); i < RB; i += 32)
#pragma unroll 1
                for (int c = 0; c < n_loc; c += 64)
                    body(std::integral_constant<bool, true>(), std::integral_constant<int, 4>(), i, c + 2 * (lane & 7));
        }
    };
    // pair t of a batch: row, column of this CTA, and the places of its elements in the matrix (-1: there is none; a matrix has
    // under 2^31 elements here)
    struct Pair
    {
        int i, c, x0, x1;
    };
    auto pair = [&](auto is_tall, int t, int i, int c) -> Pair {
        constexpr bool T = decltype(is_tall)::value;
        Pair q;
        q.i = T ? i : i + 8 * t, q.c = T ? c + 16 * t : c;
        const int j = j0 + q.c, x = T ? j * p.cols + q.i : q.i * p.cols + j;
        q.x0 = q.i < p.s && j < p.l ? x : -1;
        q.x1 = q.i < p.s && j + 1 < p.l ? x + (T ? p.cols : 1) : -1;
        return q;
    };
    const bool write_g = p.p && (p.m.hook_wd > 0.f || p.m.grad_scale != 1.f), read_p = p.p && p.m.hook_wd > 0.f;
    float *const G = p.g + off, *const B = p.buf ? p.buf + off : nullptr;
    const float *const P = read_p ? p.p + off : nullptr;
    // both elements of a pair as one 8-byte access (both or none exist: cols is even)
    auto even      = [&](const float *q) { return !(reinterpret_cast<uintptr_t>(q) & 7); };
    const bool two = !tall && !(p.cols & 1) && even(G) && even(B) && even(P);
    auto load_pair = [&](const float *src, const Pair &q, bool both, float (&v)[2]) {
        const int y0 = q.x0 < 0 ? 0 : q.x0, y1 = q.x1 < 0 ? 0 : q.x1;
        if (both)
        {
            const float2 f = *reinterpret_cast<const float2 *>(src + y0);
            v[0] = f.x, v[1] = f.y;
        }
        else
            v[0] = src[y0], v[1] = src[y1];
    };
    auto store_pair = [&](float *dst, const Pair &q, bool both, float v0, float v1) {
        if (both)
        {
            if (q.x0 >= 0)
                *reinterpret_cast<float2 *>(dst + q.x0) = make_float2(v0, v1);
            return;
        }
        if (q.x0 >= 0)
            dst[q.x0] = v0;
        if (q.x1 >= 0)
            dst[q.x1] = v1;
    };
    double sum = 0;
    batches([&](auto is_tall, auto n, int i, int c) {
        constexpr int N = decltype(n)::value;
        float g[N][2], b[N][2], w[N][2], u[2 * N];
#pragma unroll
        for (int t = 0; t < N; ++t)
        {
            const Pair q = pair(is_tall, t, i, c);
            load_pair(G, q, two, g[t]);
            b[t][0] = b[t][1] = w[t][0] = w[t][1] = 0.f;
            if (B)
                load_pair(B, q, two, b[t]);
            if (P)
                load_pair(P, q, two, w[t]);
        }
#pragma unroll
        for (int t = 0; t < N; ++t)
        {
            const Pair q = pair(is_tall, t, i, c);
#pragma unroll
            for (int e = 0; e < 2; ++e)
            {
                const float v = momentum_one(g[t][e], b[t][e], w[t][e], B != nullptr, p.m);
                u[2 * t + e]  = (e ? q.x1 : q.x0) >= 0 ? v : 0.f;
            }
            if (B)
                store_pair(B, q, two, b[t][0], b[t][1]);
            if (write_g)
                store_pair(G, q, two, g[t][0], g[t][1]);
        }
        sum += square_sum(u);
    });
    for (int o = 16; o > 0; o >>= 1)
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0)
        box[warp] = sum;
    __syncthreads();
    if (tid == 0)
    {
        for (int w = 1; w < kThreads / 32; ++w)
            sum += box[w];
        *cl_box = sum;
    }
    ptx::cluster_sync();
    double norm = 0;
    for (int r = 0; r < p.cluster; ++r)
    {
        const uint32_t remote = ptx::map_to_cta(ptx::smem_u32(cl_box), r);
        norm += __hiloint2double(static_cast<int>(ptx::ld_shared_cluster_u32(remote + 4)), static_cast<int>(ptx::ld_shared_cluster_u32(remote)));
    }
    norm             = sqrt(norm);
    const InverseNorm inv = inverse_norm(norm, p.eps, kSx);

    // ---- X = u / norm, in halves (u formed again by the thread that formed it: the same operations, the same bits) -----------------
    batches([&](auto is_tall, auto n, int i, int c) {
        constexpr int N = decltype(n)::value;
        float g[N][2], b[N][2];
#pragma unroll
        for (int t = 0; t < N; ++t)
        {
            const Pair q = pair(is_tall, t, i, c);
            g[t][0] = g[t][1] = b[t][0] = b[t][1] = 0.f;
            if (!B || p.m.nesterov)
                load_pair(G, q, two, g[t]);
            if (B)
                load_pair(B, q, two, b[t]);
        }
#pragma unroll
        for (int t = 0; t < N; ++t)
        {
            const Pair q = pair(is_tall, t, i, c);
            float v[2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
            {
                const float u = !B ? g[t][e] : p.m.nesterov ? __fadd_rn(g[t][e], __fmul_rn(b[t][e], p.m.momentum)) : b[t][e];
                v[e]          = (e ? q.x1 : q.x0) >= 0 ? inv.times(u) : 0.f;
            }
            uint32_t hi, lo;
            s16::split2(v[0], v[1], hi, lo);
            const uint32_t to                              = place<RB>(q.i, q.c);
            *reinterpret_cast<uint32_t *>(sm + to)         = hi;
            *reinterpret_cast<uint32_t *>(sm + o_xlo + to) = lo;
        }
    });
    ptx::fence_proxy_async_smem();
    __syncthreads();

    // ---- the iteration -----------------------------------------------------------------------------------------------------------
    uint32_t phase = 0;
    // descriptors: K-major with a 128-byte swizzle; X as the reduction's rows, its blocks of 64 columns C::block apart
    auto k_major = [&](int at) { return ptx::make_smem_desc(base + at, 16, 1024, ptx::kLayoutSw128); };
    auto rows_of_x = [&](int at) { return ptx::make_smem_desc(base + at, C::block, 1024, ptx::kLayoutSw128); };
    // D (+)= hi hi + (lo lo + lo hi + hi lo first), `n` steps of 16; step k's operands a_step(k), b_step(k) 16-byte units further.
    // The accumulator truncates, so it holds 64 of a reduction at most (see gemm_split16.cuh); lo lo is worth its MMA here, where
    // sums are short: 9 x 14 is 0.9e-6 off instead of 1.3e-6 (plain fp32 products 0.7e-6).
    auto products = [&](uint32_t d, uint64_t a_hi, uint64_t a_lo, uint64_t b_hi, uint64_t b_lo, int n, auto &&a_step, auto &&b_step, uint32_t idesc, uint32_t acc) {
        if (p.terms == 3)
        {
#pragma unroll 4
            for (int k = 0; k < n; ++k)
            {
                s16::mma_f16(d, a_lo + a_step(k), b_lo + b_step(k), idesc, acc);
                s16::mma_f16(d, a_lo + a_step(k), b_hi + b_step(k), idesc, 1);
                s16::mma_f16(d, a_hi + a_step(k), b_lo + b_step(k), idesc, 1);
                acc = 1;
            }
        }
#pragma unroll 4
        for (int k = 0; k < n; ++k)
        {
            s16::mma_f16(d, a_hi + a_step(k), b_hi + b_step(k), idesc, acc);
            acc = 1;
        }
    };
    auto along_row  = [](int k) -> uint64_t { return (k >> 2) * (C::block / 16) + 2 * (k & 3); };
    auto along_rows = [](int k) -> uint64_t { return k * (2048 / 16); };
    auto finish_mmas = [&]() {  // all threads
        if (!ptx::mbar_wait(bar, phase & 1, abort_f))
            *abort_f = 1;
        ++phase;
        ptx::tc_fence_after_sync();
    };
    auto threads_meet = [&]() {
        ptx::tc_fence_before_sync();
        ptx::fence_proxy_async_smem();
        __syncthreads();
        ptx::tc_fence_after_sync();
    };
    const int q = warp & 3, h = warp >> 2, row = 32 * q + lane;  // drain: lane quarter, half of the columns
    const bool mine     = 32 * q < RB;                           // (warps past RB have nothing to read)
    const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * q) << 16);
    const int ksq        = p.s_pad / 16;
    const int half_sq    = (p.s_pad / 2 + 7) / 8 * 8;            // columns of an s x s result per half
    const int c_from = h * half_sq, c_to = h ? p.s_pad : half_sq;

    for (int step = 0; step < p.steps; ++step)
    {
        if (tid == 0)
        {
            const uint32_t idesc = s16::idesc_f16(128, p.s_pad, false, false);
            for (int b = 0; b < p.blocks; ++b)
            {
                const uint64_t hi = k_major(b * C::block), lo = k_major(o_xlo + b * C::block);
                products(tmem + b % C::accs * RB, hi, lo, hi, lo, 4, along_row, along_row, idesc, b >= C::accs);
            }
            ptx::mma_commit(bar);
        }
        finish_mmas();
        const int accs    = p.blocks < C::accs ? p.blocks : C::accs;
        constexpr float f = kSa / (kSx * kSx);
        if (mine)
        {
            float *part     = reinterpret_cast<float *>(sm + o_ahi);
            constexpr int W = RB < 64 ? 8 : 32;  // columns at a time: accumulators lie RB columns apart
            for (int c = c_from; c < c_to; c += W)
            {
                float v[W];
                for (int a = 0; a < accs; ++a)
                {
                    uint32_t r[W];
                    if constexpr (W == 8)
                        s16::tmem_ld_32x8(lanes + a * RB + c, r);
                    else
                        ptx::tmem_ld_32x32(lanes + a * RB + c, r);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < W; ++i)
                        v[i] = a ? v[i] + __uint_as_float(r[i]) : __uint_as_float(r[i]);
                }
#pragma unroll
                for (int i = 0; i < W; i += 8)
                    if (c + i < c_to && row < RB)
                    {
                        if (p.cluster == 1)
                        {
                            uint32_t hi[4], lo[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                s16::split2(v[i + 2 * j] * f, v[i + 2 * j + 1] * f, hi[j], lo[j]);
                            const uint32_t at                             = place<RB>(row, c + i);
                            *reinterpret_cast<uint4 *>(sm + o_ahi + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                            *reinterpret_cast<uint4 *>(sm + o_alo + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                        }
                        else
                        {
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                part[(c + i + j) * RB + row] = v[i + j];
                        }
                    }
            }
        }
        if (p.cluster > 1)
        {
            // every CTA adds up a slice of columns of all partial sums, in rank order, and all fetch all slices
            ptx::tc_fence_before_sync();
            ptx::cluster_sync();
            const int slice = p.s_pad / p.cluster;
            for (int k = tid; k < slice * (RB / 4); k += kThreads)
            {
                const int at = (rank * slice * RB + 4 * k) * 4;  // four rows of column rank * slice + k / (RB / 4)
                float4 v[kMaxCluster];
#pragma unroll
                for (int r = 0; r < kMaxCluster; ++r)  // all in flight together
                    v[r] = ld_cluster_f4(ptx::map_to_cta(base + o_ahi + at, r < p.cluster ? r : rank));
                float4 t = v[0];
#pragma unroll
                for (int r = 1; r < kMaxCluster; ++r)
                    if (r < p.cluster)
                        t.x += v[r].x, t.y += v[r].y, t.z += v[r].z, t.w += v[r].w;
                reinterpret_cast<float4 *>(sm + o_red)[k] = t;
            }
            ptx::cluster_sync();
            // a thread: four rows of two columns; eight row groups and four column pairs a warp (shared-memory banks)
            const int groups = (RB + 31) / 32, n = p.s_pad / 8 * groups;
            const bool in    = 4 * (lane & 7) < RB;  // (RB = 16: half the lanes)
            for (int k0 = warp; k0 < n; k0 += 4 * (kThreads / 32))
            {
                float4 v[4][2];
#pragma unroll
                for (int t = 0; t < 4; ++t)
                {
                    const int k = k0 + t * (kThreads / 32);
                    const int j = k < n ? k / groups * 8 + 2 * (lane >> 3) : 0, i = k < n && in ? (k % groups) * 32 + 4 * (lane & 7) : 0;
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                    {
                        const int owner = (j + e) / slice;
                        v[t][e]         = ld_cluster_f4(ptx::map_to_cta(base + o_red + ((j + e - owner * slice) * RB + i) * 4, owner));
                    }
                }
#pragma unroll
                for (int t = 0; t < 4; ++t)
                {
                    const int k = k0 + t * (kThreads / 32);
                    if (k >= n || !in)
                        break;
                    const int j = k / groups * 8 + 2 * (lane >> 3), i = (k % groups) * 32 + 4 * (lane & 7);
                    const float a0[4] = {v[t][0].x, v[t][0].y, v[t][0].z, v[t][0].w}, a1[4] = {v[t][1].x, v[t][1].y, v[t][1].z, v[t][1].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                    {
                        uint32_t hi, lo;
                        s16::split2(a0[e] * f, a1[e] * f, hi, lo);
                        const uint32_t at                                = place<RB>(i + e, j);
                        *reinterpret_cast<uint32_t *>(sm + o_ahi + at) = hi;
                        *reinterpret_cast<uint32_t *>(sm + o_alo + at) = lo;
                    }
                }
            }
        }
        threads_meet();

        // A^2 (A is symmetric: both operands K-major), S = a I + b A + c A^2
        if (tid == 0)
        {
            // the reduction's first and second 64 into accumulators of their own
            for (int k = 0; k < ksq; k += 4)
            {
                const uint64_t hi = k_major(o_ahi) + along_row(k), lo = k_major(o_alo) + along_row(k);
                products(tmem + 32 * k, hi, lo, hi, lo, ksq - k < 4 ? ksq - k : 4, along_row, along_row, s16::idesc_f16(128, p.s_pad, false, false), 0);
            }
            ptx::mma_commit(bar);
        }
        finish_mmas();
        if (mine)
            for (int c = c_from; c < c_to; c += 32)
            {
                uint32_t r[32];
                ptx::tmem_ld_32x32(lanes + c, r);
                ptx::tmem_ld_wait();
                if (RB > 64)
                {
                    uint32_t r2[32];
                    ptx::tmem_ld_32x32(lanes + 128 + c, r2);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        r[i] = __float_as_uint(__uint_as_float(r[i]) + __uint_as_float(r2[i]));
                }
#pragma unroll
                for (int o = 0; o < 32; o += 8)
                {
                    if (c + o >= c_to || row >= RB)
                        break;
                    const uint32_t at = place<RB>(row, c + o);  // (8 columns of a row lie together)
                    const uint4 ah = *reinterpret_cast<const uint4 *>(sm + o_ahi + at), al = *reinterpret_cast<const uint4 *>(sm + o_alo + at);
                    const uint32_t hw[4] = {ah.x, ah.y, ah.z, ah.w}, lw[4] = {al.x, al.y, al.z, al.w};
                    uint32_t sh[4], sl[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                    {
                        const float2 fh = __half22float2(*reinterpret_cast<const __half2 *>(&hw[i])), fl = __half22float2(*reinterpret_cast<const __half2 *>(&lw[i]));
                        float v0 = fmaf(__uint_as_float(r[o + 2 * i]), kNsC * kSs / (kSa * kSa), (fh.x + fl.x) * (kNsB * kSs / kSa));
                        float v1 = fmaf(__uint_as_float(r[o + 2 * i + 1]), kNsC * kSs / (kSa * kSa), (fh.y + fl.y) * (kNsB * kSs / kSa));
                        v0 += c + o + 2 * i == row && row < p.s ? kNsA * kSs : 0.f;
                        v1 += c + o + 2 * i + 1 == row && row < p.s ? kNsA * kSs : 0.f;
                        s16::split2(v0, v1, sh[i], sl[i]);
                    }
                    *reinterpret_cast<uint4 *>(sm + o_ahi + at) = make_uint4(sh[0], sh[1], sh[2], sh[3]);
                    *reinterpret_cast<uint4 *>(sm + o_alo + at) = make_uint4(sl[0], sl[1], sl[2], sl[3]);
                }
            }
        threads_meet();

        // X_loc = S X_loc, as many columns at a time as TMEM holds (RB = 128: twice, see above)
        constexpr int kWidth = RB > 64 ? 256 : 512;
        for (int n0 = 0; n0 < n_loc; n0 += kWidth)
        {
            const int width = n_loc - n0 < kWidth ? n_loc - n0 : kWidth;
            if (tid == 0)
            {
                for (int n = 0; n < width; n += 256)
                {
                    const int cols = width - n < 256 ? width - n : 256, at = (n0 + n) / 64 * C::block;
                    for (int k = 0; k < ksq; k += 4)  // (k = 4: RB = 128, n = 0)
                        products(tmem + n + 64 * k, k_major(o_ahi) + along_row(k), k_major(o_alo) + along_row(k), rows_of_x(at) + along_rows(k),
                                 rows_of_x(o_xlo + at) + along_rows(k), ksq - k < 4 ? ksq - k : 4, along_row, along_rows,
                                 s16::idesc_f16(128, cols, false, true), 0);
                }
                ptx::mma_commit(bar);
            }
            finish_mmas();
            if (mine)
                for (int c = h * (width / 2); c < (h + 1) * (width / 2); c += 32)
                {
                    uint32_t r[32];
                    ptx::tmem_ld_32x32(lanes + c, r);
                    ptx::tmem_ld_wait();
                    if (RB > 64)
                    {
                        uint32_t r2[32];
                        ptx::tmem_ld_32x32(lanes + 256 + c, r2);
                        ptx::tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            r[i] = __float_as_uint(__uint_as_float(r[i]) + __uint_as_float(r2[i]));
                    }
                    if (row < RB)
                    {
#pragma unroll
                        for (int o = 0; o < 32; o += 8)
                        {
                            uint32_t hi[4], lo[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                s16::split2(__uint_as_float(r[o + 2 * i]) * (1.f / kSs), __uint_as_float(r[o + 2 * i + 1]) * (1.f / kSs), hi[i], lo[i]);
                            const uint32_t at                             = place<RB>(row, n0 + c + o);
                            *reinterpret_cast<uint4 *>(sm + at)         = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                            *reinterpret_cast<uint4 *>(sm + o_xlo + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                        }
                    }
                }
            threads_meet();
        }
    }
    // ---- the result out of its halves (2^-23 of a value), by the threads and in the order that read the gradient --------------------
    float *const O = p.out.out + off, *const L = p.out.small ? p.out.small + off : nullptr;
    const bool two_out = !tall && !(p.cols & 1) && even(O) && even(L);
    batches([&](auto is_tall, auto n, int i, int c) {
        constexpr int N = decltype(n)::value;
        float was[N][2];
#pragma unroll
        for (int t = 0; t < N; ++t)
        {
            was[t][0] = was[t][1] = 0.f;
            if (p.out.param)
                load_pair(O, pair(is_tall, t, i, c), two_out, was[t]);
        }
#pragma unroll
        for (int t = 0; t < N; ++t)
        {
            const Pair q   = pair(is_tall, t, i, c);
            const uint32_t at = place<RB>(q.i, q.c);
            const float2 hi = __half22float2(*reinterpret_cast<const __half2 *>(sm + at)), lo = __half22float2(*reinterpret_cast<const __half2 *>(sm + o_xlo + at));
            const float o0 = ns_result(p.out, (hi.x + lo.x) * (1.f / kSx), was[t][0]), o1 = ns_result(p.out, (hi.y + lo.y) * (1.f / kSx), was[t][1]);
            store_pair(O, q, two_out, o0, o1);
            if (L)
                store_pair(L, q, two_out, tf32_small(o0), tf32_small(o1));
        }
    });
    ptx::cluster_sync();  // nobody reads this CTA's shared memory any more
    if (warp == 0)
        ptx::tmem_dealloc(tmem, 512);
    if (tid == 0 && *abort_f)
        atomicExch(p.err, 1);
}
}  // namespace

namespace
{
// CTAs of a matrix: as few as hold X; more, down to two blocks each, while the GPU has SMs for them.  0: it does not fit.
template <int RB>
int cluster_for(int blocks, int64_t batch)
{
    using C = SmallCfg<RB>;
    int c   = 1;
    while (c <= kMaxCluster && !C::fits((blocks + c - 1) / c, c))
        c *= 2;
    if (c > kMaxCluster)
        return 0;
    while (c < kMaxCluster && blocks >= 4 * c && 2 * c * batch <= s16::sm_count() && C::fits((blocks + 2 * c - 1) / (2 * c), 2 * c))
        c *= 2;
    return c;
}
int cluster_of(int s, int blocks, int64_t batch)
{
    return s <= 16 ? cluster_for<16>(blocks, batch) : s <= 32 ? cluster_for<32>(blocks, batch) : s <= 64 ? cluster_for<64>(blocks, batch) : cluster_for<128>(blocks, batch);
}
template <int RB>
int launch_small(SmallArgs &k, int64_t batch, cudaStream_t stream)
{
    static bool set = false;
    if (!set)
    {
        ODL_CUDA_TRY(cudaFuncSetAttribute(muon_small_kernel<RB>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
        set = true;
    }
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim          = dim3(static_cast<unsigned>(batch * k.cluster));
    cfg.blockDim         = dim3(kThreads);
    cfg.dynamicSmemBytes = SmallCfg<RB>::bytes(k.blocks, k.cluster);
    cfg.stream           = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id               = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = k.cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs                = attr;
    cfg.numAttrs             = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, muon_small_kernel<RB>, k);
    ++g_launch_count;
    if (e != cudaSuccess)
    {
        set_last_error("muon_small_kernel launch failed: %s", cudaGetErrorString(e));
        return kCudaError;
    }
    return kOk;
}
}  // namespace

bool muon_small_eligible(int64_t rows, int64_t cols, int steps)
{
    const int64_t s = rows < cols ? rows : cols, l = rows < cols ? cols : rows;
    if (steps <= 0 || s > 128 || l > 1 << 20)
        return false;
    const int blocks = static_cast<int>((l + 63) / 64);
    return cluster_of(static_cast<int>(s), blocks, 1 << 20) > 0;
}

int muon_small(const float *p, float *g, float *buf, const MomentumArgs &a, const NsOut &out, int64_t batch, int64_t rows, int64_t cols, int steps,
               float eps, int terms, cudaStream_t stream)
{
    SmallArgs k{};
    k.p = p, k.g = g, k.buf = buf, k.m = a, k.out = out, k.err = device_error_flag();
    k.rows = (int)rows, k.cols = (int)cols;
    k.s = (int)(rows < cols ? rows : cols), k.l = (int)(rows < cols ? cols : rows);
    k.s_pad = (k.s + 15) / 16 * 16;
    k.steps = steps, k.terms = terms, k.eps = eps;
    const int all = (k.l + 63) / 64;
    k.cluster     = cluster_of(k.s, all, batch);
    k.blocks      = (all + k.cluster - 1) / k.cluster;
    return k.s <= 16 ? launch_small<16>(k, batch, stream) : k.s <= 32 ? launch_small<32>(k, batch, stream)
         : k.s <= 64 ? launch_small<64>(k, batch, stream) : launch_small<128>(k, batch, stream);
}

}  // namespace odl
