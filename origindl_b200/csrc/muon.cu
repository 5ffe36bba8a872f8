// Orthogonalised updates of weight matrices: the quintic Newton-Schulz iteration and the momentum step around it.
//   X_0 = u / max(|u|_F, eps);   X <- S X,  S = a I + b A + c A^2,  A = X X^T
// (X <- X S with A = X^T X for tall matrices: always the smaller side) with (a, b, c) = (3.4445, -4.7750, 2.0315) drives the
// singular values of X towards 1.
//
// Everything between u and the result is held split-fp16 (gemm_split16.cuh) with ONE power of two per matrix, which the
// normalisation makes safe: |X|_F <= 1 at first and the singular values stay below 1.21 afterwards, so no entry of X, A or S
// exceeds 1.21, 1.46 or 3.45; halves scaled by 2^14 (S: 2^13) reach neither the largest fp16 nor, in a way that counts, the
// smallest: the grid 2^-39 of an entry adds at most 2^-39 sqrt(rows cols) to the Frobenius norm 1 of X, less than the 2^-24 of
// fp32 itself up to 2^30 entries.  A and S are symmetric: their GEMMs compute the tiles on and above the diagonal and write each
// twice, which leaves s s l + s^3 + 2 s s l operations a step (s, l the smaller and larger side) of the 2 + 2 + 2.
// a X is folded into S (a on the diagonal), and b A into the product: S = a I + c A (A + h I), h = b / c, so that no epilogue reads
// a matrix.  A + h I differs from A in the blocks on the diagonal alone, and only those are kept a second time.  (The square
// completed, c (A + h/2 I)^2 + d I, would need one operand, but its terms of order 1 cancel: 1.5 times the error.)  A step is
// three GEMMs and nothing else; the last one's epilogue writes the result or the updated parameters.
// Measured: 8192^2 27 to 29 ms for five steps (4 s^3 operations a step, three fp16 products each, under the power cap); twelve 1024^2
// 1.1 ms, where a tile's stores hold the tensor pipe up as long as half its 16 K-blocks take.
#include <cuda_runtime.h>

#include <cmath>

#include "../../include/odl_b200.h"
#include "gemm_epilogue.cuh"
#include "gemm_split16.cuh"
#include "host_util.h"
#include "internal.h"
#include "muon.h"

namespace odl
{

namespace
{
using s16::GemmArgs;
using s16::Split16;
using s16::TileAt;

constexpr int kNormBlocks = 256;                              // at most, per matrix

inline size_t a256(size_t x)
{
    return (x + 255) & ~size_t(255);
}

#define MUON_LAUNCHED()                 \
    do                                  \
    {                                   \
        ++g_launch_count;               \
        ODL_CUDA_TRY(cudaGetLastError()); \
    } while (0)

// grid (blocks, batch): momentum in place and the sum of squares of u, in double (no size of gradient over- or underflows)
__global__ void __launch_bounds__(256) muon_momentum_kernel(const float *__restrict__ p, float *g, float *buf, int64_t n, MomentumArgs a, bool vec,
                                                            double *__restrict__ partial)
{
    s16::let_next_in();
    const int64_t off  = static_cast<int64_t>(blockIdx.y) * n;
    const bool write_g = p && (a.hook_wd > 0.f || a.grad_scale != 1.f), read_p = p && a.hook_wd > 0.f;
    double s = 0;
    g += off;
    buf = buf ? buf + off : nullptr;
    p   = p ? p + off : nullptr;
    // four values at a time, whatever the alignment (the sum has the same bits)
    const int64_t stride = static_cast<int64_t>(gridDim.x) * 256, n4 = (n + 3) >> 2;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n4; i += stride)
    {
        float G[4], M[4] = {0.f, 0.f, 0.f, 0.f}, P[4] = {0.f, 0.f, 0.f, 0.f}, u[4];
        const int have = n - 4 * i < 4 ? static_cast<int>(n - 4 * i) : 4;
        auto load      = [&](const float *src, float (&v)[4]) {
            if (vec)
            {
                const float4 q = reinterpret_cast<const float4 *>(src)[i];
                v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
            }
            else
            {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    v[j] = j < have ? src[4 * i + j] : 0.f;
            }
        };
        auto store = [&](float *dst, const float (&v)[4]) {
            if (vec)
                reinterpret_cast<float4 *>(dst)[i] = make_float4(v[0], v[1], v[2], v[3]);
            else
            {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j < have)
                        dst[4 * i + j] = v[j];
            }
        };
        load(g, G);
        if (buf)
            load(buf, M);
        if (read_p)
            load(p, P);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            u[j] = momentum_one(G[j], M[j], P[j], buf, a);
        if (buf)
            store(buf, M);
        if (write_g)
            store(g, G);
        s += square_sum(u);
    }
    __shared__ double box[8];
    for (int o = 16; o > 0; o >>= 1)
        s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0)
        box[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0)
    {
        for (int w = 1; w < 8; ++w)
            s += box[w];
        partial[blockIdx.y * gridDim.x + blockIdx.x] = s;
    }
}

// X = u / max(|u|, eps) in halves; u is formed again from g and the updated buf (the same operations, the same bits).
// grid (blocks, batch); a warp per block of 64 columns of a row.
__global__ void __launch_bounds__(256) muon_split_kernel(const float *__restrict__ g, const float *__restrict__ buf, int rows, int cols, int cols_pad,
                                                         float momentum, int nesterov, const double *__restrict__ partial, int n_partial, float eps,
                                                         __half *__restrict__ x, int64_t x_stride)
{
    __shared__ double box[8];
    s16::let_next_in();
    s16::after_previous();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double s       = 0;
    for (int i = threadIdx.x; i < n_partial; i += 256)
        s += partial[blockIdx.y * n_partial + i];
    for (int o = 16; o > 0; o >>= 1)
        s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0)
        box[warp] = s;
    __syncthreads();
    double norm = 0;
    for (int w = 0; w < 8; ++w)
        norm += box[w];
    norm             = sqrt(norm);
    const InverseNorm inv = inverse_norm(norm, eps, kSx);
    const int64_t off = static_cast<int64_t>(blockIdx.y) * rows * cols;
    const int blocks  = cols_pad / 64;
    const int64_t all = static_cast<int64_t>(rows) * blocks;
    g += off;
    buf = buf ? buf + off : nullptr;
    uint32_t *out = reinterpret_cast<uint32_t *>(x + blockIdx.y * x_stride);
    for (int64_t k = static_cast<int64_t>(blockIdx.x) * 8 + warp; k < all; k += static_cast<int64_t>(gridDim.x) * 8)
    {
        const int row = static_cast<int>(k / blocks), c = static_cast<int>(k % blocks) * 64 + 2 * lane;
        float v[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (c + j < cols)
            {
                const int64_t at = static_cast<int64_t>(row) * cols + c + j;
                const float m    = buf ? buf[at] : 0.f;
                v[j]             = !buf ? g[at] : nesterov ? __fadd_rn(g[at], __fmul_rn(m, momentum)) : m;
            }
        uint32_t hi, lo;
        s16::split2(inv.times(v[0]), inv.times(v[1]), hi, lo);
        out[k * 64 + lane]      = hi;
        out[k * 64 + 32 + lane] = lo;
    }
}

// ---- epilogues -----------------------------------------------------------------------------------------------------------
// N columns of this thread's row into a split matrix: 64-column blocks of [hi][lo], 32 bytes a store (whole sectors)
__device__ __forceinline__ void st_words8(__half *p, const uint32_t (&w)[8])
{
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                 "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

template <int NC>
__device__ __forceinline__ void store_split_row(__half *row, int col, int cols_pad, const float (&v)[NC])
{
#pragma unroll
    for (int i = 0; i < NC; i += 16)
    {
        const int c = col + i;
        if (c < cols_pad)
        {
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                s16::split2(v[i + 2 * j], v[i + 2 * j + 1], hi[j], lo[j]);
            __half *p = row + (c >> 6) * 128 + (c & 63);
            st_words8(p, hi);
            st_words8(p + 64, lo);
        }
    }
}

// the transpose of a warp's 32 rows x NC columns: row `col + i` of the matrix receives 32 consecutive columns.  Neighbouring
// lanes swap one of two values, so that a lane holds two neighbouring columns of one row and stores them as a word.
template <int NC>
__device__ __forceinline__ void store_split_mirror(__half *base, int64_t pitch, int row0, int col, int rows, int cols_pad, int lane, const float (&v)[NC])
{
    // lane's element pair: columns row0 + (lane & ~1), + 1 of matrix row col + i + (lane & 1)
    const int c = row0 + (lane & ~1);
#pragma unroll
    for (int i = 0; i < NC; i += 2)
    {
        const float give = (lane & 1) ? v[i] : v[i + 1];
        const float got  = __shfl_xor_sync(0xffffffffu, give, 1);
        const float x0 = (lane & 1) ? got : v[i], x1 = (lane & 1) ? v[i + 1] : got;
        const int r = col + i + (lane & 1);
        if (r < rows && c < cols_pad)
        {
            uint32_t hi, lo;
            s16::split2(x0, x1, hi, lo);
            __half *p                            = base + r * pitch + (c >> 6) * 128 + (c & 63);
            *reinterpret_cast<uint32_t *>(p)      = hi;
            *reinterpret_cast<uint32_t *>(p + 64) = lo;
        }
    }
}

// A symmetric result in halves, both triangles: alpha * accumulator (+ diag on the diagonal); with `blocks` its 128 x 128 blocks on
// the diagonal, `blocks_diag` added on the diagonal, a second time
struct EpiSym
{
    static constexpr bool kSquare = true;
    struct Params
    {
        __half *out;
        int64_t pitch, stride;
        int cols_pad;
        float alpha, diag;  // in units of the halves
        __half *blocks;     // [row][128 columns], blocks_stride halves from matrix to matrix
        int64_t blocks_stride;
        float blocks_diag;
    };
    template <int NC>
    static __device__ __forceinline__ void store(const Params &p, const GemmArgs &, const TileAt &at, float (&v)[NC], float *)
    {
#pragma unroll
        for (int i = 0; i < NC; ++i)
            v[i] *= p.alpha;
        if (at.tm == at.tn)
        {
#pragma unroll
            for (int i = 0; i < NC; ++i)
                v[i] += at.col + i == at.row && at.row < at.rows ? p.diag : 0.f;
        }
        __half *out = p.out + at.batch * p.stride;
        if (at.row < at.rows)
            store_split_row<NC>(out + at.row * p.pitch, at.col, p.cols_pad, v);
        if (p.blocks && at.row >> 7 == at.col >> 7)  // (the same for a warp)
        {
#pragma unroll
            for (int i = 0; i < NC; ++i)
                v[i] += at.col + i == at.row && at.row < at.rows ? p.blocks_diag : 0.f;
            if (at.row < at.rows)
                store_split_row<NC>(p.blocks + at.batch * p.blocks_stride + at.row * 256, at.col & 127, 128, v);
        }
        if (at.tm != at.tn)
            store_split_mirror<NC>(out, p.pitch, at.row - at.lane, at.col, at.rows, p.cols_pad, at.lane, v);
    }
};

// X of the next step, in halves
struct EpiX
{
    static constexpr bool kSquare = false;
    struct Params
    {
        __half *out;
        int64_t pitch, stride;
        int cols_pad;
        float alpha;
    };
    template <int NC>
    static __device__ __forceinline__ void store(const Params &p, const GemmArgs &, const TileAt &at, float (&v)[NC], float *)
    {
#pragma unroll
        for (int i = 0; i < NC; ++i)
            v[i] *= p.alpha;
        if (at.row < at.rows)
            store_split_row<NC>(p.out + at.batch * p.stride + at.row * p.pitch, at.col, p.cols_pad, v);
    }
};

// the last step's result: written out, or the parameters' update
struct EpiOut
{
    static constexpr bool kSquare = false;
    struct Params : NsOut
    {
        int64_t ld, stride;
        float alpha;     // accumulator -> X
        int vec;
    };
    static __device__ __forceinline__ float one(const Params &p, float x, float was)
    {
        return ns_result(p, x * p.alpha, was);
    }
    template <int NC>
    static __device__ __forceinline__ void store(const Params &p, const GemmArgs &g, const TileAt &at, float (&v)[NC], float *slab)
    {
        float *out   = p.out + at.batch * p.stride;
        float *small = p.small ? p.small + at.batch * p.stride : nullptr;
        if (p.vec)
        {
            if (at.row >= at.rows)
                return;
            float *row = out + at.row * p.ld + at.col;
#pragma unroll
            for (int i = 0; i < NC; i += 8)
                if (at.col + i < g.N)  // (ld and with it N are multiples of 8)
                {
                    float was[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, o[8];
                    if (p.param)
                        ld_global_v8(row + i, was);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        o[j] = one(p, v[i + j], was[j]);
                    st_global_v8(row + i, o);
                    if (small)
                    {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            o[j] = tf32_small(o[j]);
                        st_global_v8(small + at.row * p.ld + at.col + i, o);
                    }
                }
            return;
        }
        const int row0 = at.row - at.lane;
#pragma unroll
        for (int b = 0; b < NC / 32; ++b)
            s16::by_rows(v + 32 * b, slab, at.lane, [&](int r, float x) {
                const int c = at.col + 32 * b + at.lane;
                if (row0 + r < at.rows && c < g.N)
                {
                    const int64_t k = (row0 + r) * p.ld + c;
                    const float o   = one(p, x, p.param ? out[k] : 0.f);
                    out[k]          = o;
                    if (small)
                        small[k] = tf32_small(o);
                }
            });
    }
};

// steps == 0: X_0 itself (the division alone)
__global__ void __launch_bounds__(256) muon_direct_kernel(const __half *__restrict__ x, int64_t x_stride, int rows, int cols, int cols_pad,
                                                          EpiOut::Params p)
{
    s16::let_next_in();
    s16::after_previous();
    const int64_t n = static_cast<int64_t>(rows) * cols;
    x += blockIdx.y * x_stride;
    float *out   = p.out + blockIdx.y * p.stride;
    float *small = p.small ? p.small + blockIdx.y * p.stride : nullptr;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256)
    {
        const int64_t r = i / cols;
        const int c     = static_cast<int>(i - r * cols);
        const __half *h = x + r * 2 * cols_pad + (c >> 6) * 128 + (c & 63);
        const float o   = EpiOut::one(p, __half2float(h[0]) + __half2float(h[64]), p.param ? out[i] : 0.f);
        out[i]          = o;
        if (small)
            small[i] = tf32_small(o);
    }
}

template <class Epi>
int gemm(const s16::Plan &plan, int terms, const Split16 &A, const Split16 &B, const GemmArgs &g, const typename Epi::Params &ep, cudaStream_t stream,
         const Split16 *D = nullptr)
{
    return terms == 3 ? s16::launch_plan<3, false, Epi>(plan, A, B, g, ep, stream, D) : s16::launch_plan<1, false, Epi>(plan, A, B, g, ep, stream, D);
}

int orthogonalise(const float *p, float *g, float *buf, const MomentumArgs &a, EpiOut::Params out, int64_t batch, int64_t rows, int64_t cols,
                  int steps, float eps, int precision, cudaStream_t stream)
{
    const int64_t n  = rows * cols;
    const bool tall  = rows > cols;
    const int64_t m  = tall ? cols : rows;
    const int terms  = precision == ODL_PRECISION_3XTF32 ? 3 : 1;
    if (!g_bn_override && muon_small_eligible(rows, cols, steps))
    {
        int rc = check_device();
        return rc ? rc : muon_small(p, g, buf, a, out, batch, rows, cols, steps, eps, terms, stream);
    }
    const int xc = s16::pad64(cols), mc = s16::pad64(m);
    // 256-byte multiples: rows are whole blocks of 64 columns
    const int64_t x_stride = rows * 2 * xc, m_stride = m * 2 * mc, d_stride = m * 2 * 128;
    int64_t blocks         = (n / 4 + 1023) / 1024;
    blocks                 = blocks < 1 ? 1 : blocks > kNormBlocks ? kNormBlocks : blocks;
    int rc = arena_begin(2 * a256(batch * x_stride * 2) + 2 * a256(batch * m_stride * 2) + a256(batch * d_stride * 2) + a256(batch * blocks * 8), stream);
    if (rc)
        return rc;
    const ArenaUse use{stream};
    __half *x[2]    = {static_cast<__half *>(arena_alloc(batch * x_stride * 2)), static_cast<__half *>(arena_alloc(batch * x_stride * 2))};
    __half *A       = static_cast<__half *>(arena_alloc(batch * m_stride * 2));
    __half *S       = static_cast<__half *>(arena_alloc(batch * m_stride * 2));
    __half *D       = static_cast<__half *>(arena_alloc(batch * d_stride * 2));  // the blocks of A + h I on the diagonal
    double *partial = static_cast<double *>(arena_alloc(batch * blocks * 8));
    auto al16       = [](const void *q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
    const bool vec  = !(n & 3) && al16(g) && al16(buf) && al16(p);
    muon_momentum_kernel<<<dim3((unsigned)blocks, (unsigned)batch), 256, 0, stream>>>(p, g, buf, n, a, vec, partial);
    MUON_LAUNCHED();
    int64_t sblocks = (rows * (xc / 64) + 31) / 32;
    sblocks         = sblocks > 1184 ? 1184 : sblocks;
    if ((rc = s16::launch_after(muon_split_kernel, dim3((unsigned)sblocks, (unsigned)batch), dim3(256), 0, stream, g, buf, (int)rows, (int)cols, xc, a.momentum,
                                a.nesterov, partial, (int)blocks, eps, x[0], x_stride)))
        return rc;
    out.ld = cols, out.stride = n;
    out.vec = !(cols & 7) && !(reinterpret_cast<uintptr_t>(out.out) & 31) && !(reinterpret_cast<uintptr_t>(out.small) & 31);
    if (steps == 0)
    {
        out.alpha = 1.f / kSx;
        if ((rc = s16::launch_after(muon_direct_kernel, dim3((unsigned)sblocks, (unsigned)batch), dim3(256), 0, stream, x[0], x_stride, (int)rows, (int)cols, xc,
                                    out)))
            return rc;
        return kOk;
    }
    GemmArgs gg{};
    gg.batch = (int)batch, gg.splits = 1, gg.err = device_error_flag();
    GemmArgs ga = gg, gs = gg, gx = gg;
    ga.M = ga.N = (int)m, ga.K = (int)(tall ? rows : cols), ga.sym = 1, ga.a_mn = ga.b_mn = tall;
    gs.M = gs.N = gs.K = (int)m, gs.sym = 1;
    gx.M = (int)rows, gx.N = (int)cols, gx.K = (int)m, gx.b_mn = !tall;
    const s16::Plan plan_a = s16::plan_tiles(m, m, ga.K, terms, (int)batch, false, true), plan_s = s16::plan_tiles(m, m, m, terms, (int)batch, false, true),
                    plan_x = s16::plan_tiles(rows, cols, m, terms, (int)batch, false);
    auto matrix = [&](const __half *d, int64_t r, int c_pad, int64_t stride) {
        Split16 s;
        s.data = d, s.pitch = 2 * c_pad, s.rows = (int)r, s.cols_pad = c_pad, s.batch = (int)batch, s.batch_stride = stride;
        return s;
    };
    const Split16 MA = matrix(A, m, mc, m_stride), MS = matrix(S, m, mc, m_stride), MD = matrix(D, m, 128, d_stride);
    for (int k = 0; k < steps; ++k)
    {
        const Split16 MX = matrix(x[k & 1], rows, xc, x_stride);
        const EpiSym::Params ea{A, 2 * mc, m_stride, mc, kSa / (kSx * kSx), 0.f, D, d_stride, kNsH * kSa};
        const EpiSym::Params es{S, 2 * mc, m_stride, mc, kNsC * kSs / (kSa * kSa), kNsA * kSs, nullptr, 0, 0.f};
        if ((rc = gemm<EpiSym>(plan_a, terms, MX, MX, ga, ea, stream)) || (rc = gemm<EpiSym>(plan_s, terms, MA, MA, gs, es, stream, &MD)))
            return rc;
        if (k + 1 < steps)
        {
            const EpiX::Params ex{x[(k + 1) & 1], 2 * xc, x_stride, xc, 1.f / kSs};
            rc = gemm<EpiX>(plan_x, terms, tall ? MX : MS, tall ? MS : MX, gx, ex, stream);
        }
        else
        {
            out.alpha = 1.f / (kSs * kSx);
            rc        = gemm<EpiOut>(plan_x, terms, tall ? MX : MS, tall ? MS : MX, gx, out, stream);
        }
        if (rc)
            return rc;
    }
    return kOk;
}

int check_matrix(const char *what, int64_t batch, int64_t rows, int64_t cols, int steps, float eps, int precision)
{
    if (batch <= 0 || rows <= 0 || cols <= 0 || steps < 0 || steps > 100 || !(eps > 0.f))
    {
        set_last_error("%s: invalid argument (batch=%lld rows=%lld cols=%lld steps=%d eps=%g)", what, (long long)batch,
                       (long long)rows, (long long)cols, steps, (double)eps);
        return kInvalidArgument;
    }
    if (rows > 0x3fffffff || cols > 0x3fffffff || batch > 65535)
    {
        set_last_error("%s: dimension exceeds its limit (rows, cols 2^30; batch 65535)", what);
        return kTooLarge;
    }
    if (precision != ODL_PRECISION_3XTF32 && precision != ODL_PRECISION_TF32)
    {
        set_last_error("%s: unknown precision %d", what, precision);
        return kInvalidArgument;
    }
    return kOk;
}

int check_ready()
{
    if (is_ready())
        return kOk;
    set_last_error("odl_init has not been called");
    return kNotInitialized;
}
}  // namespace

}  // namespace odl

using namespace odl;

extern "C" int odl_newton_schulz(const float *g, float *out, int64_t batch, int64_t rows, int64_t cols, int steps, float eps,
                                 int precision, void *stream)
{
    int rc = check_matrix("newton_schulz", batch, rows, cols, steps, eps, precision);
    if (rc)
        return rc;
    if (!g || !out)
    {
        set_last_error("newton_schulz: null buffer");
        return kInvalidArgument;
    }
    if ((rc = check_ready()))
        return rc;
    const MomentumArgs a{0.f, 0.f, 1.f, 0};
    EpiOut::Params o{};
    o.out = out;
    return orthogonalise(nullptr, const_cast<float *>(g), nullptr, a, o, batch, rows, cols, steps, eps, precision,
                         static_cast<cudaStream_t>(stream));
}

extern "C" int odl_muon_step(float *param, float *grad, float *momentum_buf, float *param_small, int64_t batch, int64_t rows,
                             int64_t cols, int w_layout, float lr, float momentum, float weight_decay, int nesterov,
                             float hook_weight_decay, float grad_scale, int steps, float eps, int precision, void *stream)
{
    int rc = check_matrix("muon", batch, rows, cols, steps, eps, precision);
    if (rc)
        return rc;
    if (w_layout != ODL_W_OUT_IN && w_layout != ODL_W_IN_OUT)
    {
        set_last_error("muon: unknown weight layout %d", w_layout);
        return kInvalidArgument;
    }
    if (!param || !grad || (momentum > 0.f && !momentum_buf) || !(momentum >= 0.f))
    {
        set_last_error("muon: invalid argument (null buffer, or momentum=%g without its buffer)", (double)momentum);
        return kInvalidArgument;
    }
    if ((rc = check_ready()))
        return rc;
    const double out = w_layout == ODL_W_OUT_IN ? rows : cols, in = w_layout == ODL_W_OUT_IN ? cols : rows;
    const double s   = out > in ? std::sqrt(out / in) : 1.0;
    const MomentumArgs a{momentum, hook_weight_decay, grad_scale, nesterov};
    EpiOut::Params o{};
    o.out = param, o.small = param_small, o.param = 1;
    o.keep = static_cast<float>(1.0 - static_cast<double>(lr) * weight_decay);
    o.rate = static_cast<float>(lr * s);
    return orthogonalise(param, grad, momentum > 0.f ? momentum_buf : nullptr, a, o, batch, rows, cols, steps, eps, precision,
                         static_cast<cudaStream_t>(stream));
}
