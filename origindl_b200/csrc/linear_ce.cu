// Softmax cross entropy of a linear head: loss, log-sum-exp and the gradients of x, W and b from one call that never holds
// all the logits.
//   z = x W^T + b;   lse_i = log sum_j exp z_ij;   loss = 1/n sum_{i valid} (lse_i - z_{i,t_i}),  n = valid rows
//   P_ij = exp(z_ij - lse_i) - [j = t_i];   dx = g P W,  dW = g P^T x,  db = g colsum(P),  g = grad_scale / n
//
// Rows without a label are left out before anything is computed: the labels pass lists the n others, x is gathered through that
// list while it is split into halves, and every kernel behind it reads n on the device (a batch that is half padding costs
// half).  The matrices are split-fp16 (gemm_split16.cuh): W and x once, with a power of two per 128 x 128 tile.
// Loss alone: the logits' GEMM keeps a running maximum and sum of each row's strip of 128 columns in the epilogue's registers
// and writes those two numbers, nothing else.  With gradients: the rows are taken in pieces whose logits fit kPieceBytes; the
// same epilogue also stores the logits, and once the row statistics are joined one pass turns them into P in place (the 4 bytes
// of a logit become the two halves of P), which the GEMMs for dx (reduction over the classes, split into slices where its few
// tiles would leave SMs idle) and dW (reduction over the rows, added up over the pieces in order) read.  That is 6 M N K
// operations where recomputing the logits for the gradient would be 8.
// P lies in [-1, 1] and has one scale, 2^-15: exact to 2^-23 of itself down to 2^-28, below that to 2^-40 absolute.
// Bound by the products.  8192 x 131072 x 2048: 37 ms (power-capped; 6 M N K at three products each), of which W's split 0.7 and
// the softmax passes 1.4; 4096 x 32768 x 2048 alone: logits 1.2 ms (tensor pipe 78 % busy, the epilogue holds it up 9 thousand
// cycles a tile), dx 1.15 (94 %), dW 1.18 (88 %).
#include <cuda_runtime.h>

#include <cmath>

#include "../../include/odl_b200.h"
#include "gemm_epilogue.cuh"
#include "gemm_split16.cuh"
#include "host_util.h"
#include "internal.h"
#include "linear_ce.h"
#include "split16_encode.h"

namespace odl
{

namespace
{
using s16::GemmArgs;
using s16::Split16;
using s16::TileAt;

constexpr int64_t kPieceBytes = int64_t(1) << 30;  // logits of a piece of rows (at least 256 rows)
constexpr float kPScale       = 32768.f;           // P is stored as P * 2^15
constexpr float kLog2e        = 1.4426950408889634f;

inline size_t a256(size_t x)
{
    return (x + 255) & ~size_t(255);
}

#define LCE_LAUNCHED()                  \
    do                                  \
    {                                   \
        ++g_launch_count;               \
        ODL_CUDA_TRY(cudaGetLastError()); \
    } while (0)

// device words of one call
struct Counters
{
    int count;        // rows with a label
    float inv_count;  // 1 / count, 0 when there is none
    int bad;          // a label was out of range
};

// The rows that have a label, in order: idx[pos] = row, cls[pos] = its class; pos_of[row] = pos or -1.  One block: M is read
// once, 4096 rows a round; a round's positions come from warp sums.
__global__ void __launch_bounds__(1024) lce_labels_kernel(const void *__restrict__ labels, int is64, int64_t ignore, int M, int N,
                                                          int *__restrict__ idx, int *__restrict__ cls, int *__restrict__ pos_of,
                                                          Counters *out)
{
    __shared__ int warp_sum[32], base, any_bad;
    s16::let_next_in();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0)
        base = 0, any_bad = 0;
    __syncthreads();
    for (int r0 = 0; r0 < M; r0 += 4096)
    {
        int c[4], n = 0;
        const int first = r0 + 4 * static_cast<int>(threadIdx.x);
#pragma unroll
        for (int j = 0; j < 4; ++j)
        {
            c[j] = -1;
            if (first + j < M)
            {
                const int64_t t = is64 ? static_cast<const int64_t *>(labels)[first + j] : static_cast<const int32_t *>(labels)[first + j];
                if (t != ignore)
                {
                    if (t >= 0 && t < N)
                        c[j] = static_cast<int>(t);
                    else
                        any_bad = 1;
                }
                n += c[j] >= 0;
            }
        }
        int scan = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1)
        {
            const int v = __shfl_up_sync(0xffffffffu, scan, o);
            if (lane >= o)
                scan += v;
        }
        if (lane == 31)
            warp_sum[warp] = scan;
        __syncthreads();
        int before = base, total = 0;
        for (int w = 0; w < 32; ++w)
        {
            before += w < warp ? warp_sum[w] : 0;
            total += warp_sum[w];
        }
        int pos = before + scan - n;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (first + j < M)
            {
                pos_of[first + j] = c[j] >= 0 ? pos : -1;
                if (c[j] >= 0)
                {
                    idx[pos] = first + j;
                    cls[pos] = c[j];
                    ++pos;
                }
            }
        __syncthreads();
        if (threadIdx.x == 0)
            base += total;
        __syncthreads();
    }
    if (threadIdx.x == 0)
    {
        out->count     = base;
        out->inv_count = base > 0 ? 1.0f / static_cast<float>(base) : 0.f;
        out->bad       = any_bad;
    }
}

// ---- epilogue of the logits' GEMM: row statistics of a strip of columns, the label's logit, the logits themselves --------
struct EpiLogits
{
    static constexpr bool kSquare = false;
    struct Params
    {
        const float *bias;
        const int *cls;     // of this piece's rows
        float2 *part;       // [strip][part_ld]: maximum and sum of exponentials
        int part_ld;
        float *picked;      // logit of the row's label
        float *logits;      // nullptr: statistics alone
        int64_t ld;         // padded columns
    };
    template <int NC>
    static __device__ __forceinline__ void store(const Params &p, const GemmArgs &g, const TileAt &at, float (&v)[NC], float *)
    {
        const bool live = at.row < at.rows;
        if (p.bias)
        {
#pragma unroll
            for (int i = 0; i < NC; ++i)
                if (at.col + i < g.N)
                    v[i] += __ldg(p.bias + at.col + i);
        }
        const int label = live ? p.cls[at.row] - at.col : -1;
        // the strip that holds the label's column writes it (a strip holds one of 32 rows' labels rarely)
        if (__any_sync(0xffffffffu, label >= 0 && label < NC))
        {
            float pick = 0.f;
#pragma unroll
            for (int i = 0; i < NC; ++i)
                pick = label == i ? v[i] : pick;
            if (label >= 0 && label < NC)
                p.picked[at.row] = pick;
        }
        if (p.logits && live)
        {
            float *row = p.logits + at.row * p.ld + at.col;
#pragma unroll
            for (int i = 0; i < NC; i += 8)
                if (at.col + i < p.ld)
                {
                    const float o[8] = {v[i], v[i + 1], v[i + 2], v[i + 3], v[i + 4], v[i + 5], v[i + 6], v[i + 7]};
                    st_global_v8(row + i, o);
                }
        }
        if (at.col + NC > g.N)
        {
#pragma unroll
            for (int i = 0; i < NC; ++i)
                v[i] = at.col + i < g.N ? v[i] : -INFINITY;
        }
        float m = v[0], m1 = v[1];
#pragma unroll
        for (int i = 2; i < NC; i += 2)
        {
            m  = fmaxf(m, v[i]);
            m1 = fmaxf(m1, v[i + 1]);
        }
        m = fmaxf(m, m1);
        const float base = m == -INFINITY ? 0.f : m;  // a strip without a class left: sum 0, not NaN
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int i = 0; i < NC; i += 2)
        {
            s0 += s16::fast_exp2((v[i] - base) * kLog2e);
            s1 += s16::fast_exp2((v[i + 1] - base) * kLog2e);
        }
        if (live)
            p.part[static_cast<int64_t>(at.strip) * p.part_ld + at.row] = make_float2(m, s0 + s1);
    }
};

// ---- epilogue of the gradients' GEMMs: scaled fp32 rows, through a row list, added to what is there, or as a slice -------
struct EpiGrad
{
    static constexpr bool kSquare = false;
    struct Params
    {
        float *out;
        int64_t ld;
        const int *rows;          // row i of the product is row rows[i] of out; nullptr = i
        const Counters *counters; // inv_count is part of the factor
        float alpha;
        int add;
        int64_t slice;            // floats from slice to slice (splits > 1)
        int vec;                  // rows of out are 32-byte aligned
    };
    template <int NC>
    static __device__ __forceinline__ void store(const Params &p, const GemmArgs &g, const TileAt &at, float (&v)[NC], float *slab)
    {
        const float f = p.alpha * p.counters->inv_count;
        float *out    = p.out + at.split * p.slice;
        if (p.vec)
        {
            if (at.row >= at.rows)
                return;
            float *row = out + static_cast<int64_t>(p.rows ? p.rows[at.row] : at.row) * p.ld + at.col;
#pragma unroll
            for (int i = 0; i < NC; i += 8)
            {
                if (at.col + i + 8 <= g.N)
                {
                    float o[8], was[8];
                    if (p.add)
                        ld_global_v8(row + i, was);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        o[j] = p.add ? fmaf(v[i + j], f, was[j]) : v[i + j] * f;
                    st_global_v8(row + i, o);
                }
                else
                {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (at.col + i + j < g.N)
                            row[i + j] = p.add ? fmaf(v[i + j], f, row[i + j]) : v[i + j] * f;
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
                    float *o = out + static_cast<int64_t>(p.rows ? p.rows[row0 + r] : row0 + r) * p.ld + c;
                    *o       = p.add ? fmaf(x, f, *o) : x * f;
                }
            });
    }
};

__device__ __forceinline__ void join(float &m, float &s, float om, float os)
{
    const float t = fmaxf(m, om), b = t == -INFINITY ? 0.f : t;
    s = s * s16::fast_exp2((m - b) * kLog2e) + os * s16::fast_exp2((om - b) * kLog2e);
    m = t;
}

struct LseArgs
{
    const float2 *part;  // [strip][part_ld]
    int part_ld, strips;
    int rows, base;      // of the piece; its first row among those with a label
    const Counters *cnt;
    const int *idx;      // of the piece's rows
    const float *picked;
    float *lse, *row_loss, *lse_out;
};

// lse of 32 rows of a piece from their strips' maxima and sums, by GROUPS warps (lane = row), and the rows' losses
template <int GROUPS>
__device__ __forceinline__ void lse_of_rows(const LseArgs &p, int row0, int live, float2 (&box)[GROUPS][32], float *s_lse)
{
    const int lane = threadIdx.x & 31, group = threadIdx.x >> 5, row = row0 + lane;
    float m = -INFINITY, s = 0.f;
    if (row < live)
    {
        const float2 *src = p.part + row;
        int k             = group;
        for (; k + 3 * GROUPS < p.strips; k += 4 * GROUPS)
        {
            float2 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[i] = src[static_cast<int64_t>(k + i * GROUPS) * p.part_ld];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                join(m, s, v[i].x, v[i].y);
        }
        for (; k < p.strips; k += GROUPS)
        {
            const float2 v = src[static_cast<int64_t>(k) * p.part_ld];
            join(m, s, v.x, v.y);
        }
    }
    box[group][lane] = make_float2(m, s);
    __syncthreads();
    if (group == 0)
    {
        if (row < live)
        {
            for (int k = 1; k < GROUPS; ++k)
                join(m, s, box[k][lane].x, box[k][lane].y);
            const float l = m + logf(s);
            if (s_lse)
                s_lse[lane] = l;
            else
                p.lse[row] = l;
            p.row_loss[p.base + row] = l - p.picked[row];
            if (p.lse_out)
                p.lse_out[p.idx[row]] = l;
        }
        else if (s_lse)
            s_lse[lane] = 0.f;
    }
}

__global__ void __launch_bounds__(512) lce_lse_kernel(const LseArgs p)
{
    __shared__ float2 box[16][32];
    s16::let_next_in();
    s16::after_previous();
    lse_of_rows<16>(p, blockIdx.x * 32, min(p.rows, p.cnt->count - p.base), box, nullptr);
}

// Logits of a piece -> P * 2^15 in halves, in place.  A block: 512 columns (a warp per block of 64) x ROWS rows; a warp reads the
// 256 bytes of 64 logits and writes the same 256 bytes as [64 hi][64 lo].  Rows behind the last (up to a multiple of 128) and
// padding columns become zeros.  colsum (optional): sums of P over the block's rows, [row block][ld].  ROWS = 32: pieces whose
// 128-row blocks would leave SMs idle; there, and with one block over the columns, the block finds its rows' lse itself.
template <int ROWS>
__global__ void __launch_bounds__(256) lce_softmax_kernel(float *z, int64_t ld, int N, int rows, const LseArgs p, const int *__restrict__ cls, int own_lse,
                                                          float *__restrict__ colsum)
{
    __shared__ float s_lse[ROWS];
    __shared__ int s_cls[ROWS];
    __shared__ float2 box[8][32];
    s16::let_next_in();
    s16::after_previous();
    const int r0 = blockIdx.x * ROWS, live = min(p.rows, p.cnt->count - p.base);
    if (r0 >= (live + 127) / 128 * 128)
        return;
    if (threadIdx.x < ROWS)
    {
        const int r = r0 + threadIdx.x;
        if (!own_lse)
            s_lse[threadIdx.x] = r < live ? p.lse[r] : 0.f;
        s_cls[threadIdx.x] = r < live ? cls[r] : -1;
    }
    if (ROWS == 32 && own_lse)
        lse_of_rows<8>(p, r0, live, box, s_lse);
    __syncthreads();
    const int lane = threadIdx.x & 31;
    const int c0   = blockIdx.y * 512 + (threadIdx.x >> 5) * 64;
    if (c0 >= ld)
        return;
    const int c = c0 + 2 * lane;
    float2 sum  = make_float2(0.f, 0.f);
    const int last = min(rows - r0, ROWS);
    for (int r = 0; r < last; r += 8)
    {
        float2 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = r + i < live - r0 ? __ldcs(reinterpret_cast<const float2 *>(z + (r0 + r + i) * ld + c)) : make_float2(0.f, 0.f);
        __syncwarp();  // the warp's 256 bytes have been read before any of them is written
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            if (r + i >= last)
                break;
            const bool on  = r + i < live - r0;
            const float l  = s_lse[r + i];
            const int t    = s_cls[r + i] - c;
            float a        = on && c < N ? s16::fast_exp2((v[i].x - l) * kLog2e) : 0.f;
            float b        = on && c + 1 < N ? s16::fast_exp2((v[i].y - l) * kLog2e) : 0.f;
            a -= t == 0 ? 1.f : 0.f;
            b -= t == 1 ? 1.f : 0.f;
            sum.x += a;
            sum.y += b;
            uint32_t hi, lo;
            s16::split2(a * kPScale, b * kPScale, hi, lo);
            uint32_t *line  = reinterpret_cast<uint32_t *>(z + (r0 + r + i) * ld + c0);
            line[lane]      = hi;
            line[32 + lane] = lo;
        }
    }
    if (colsum)
        *reinterpret_cast<float2 *>(colsum + blockIdx.x * ld + c) = sum;
}

// dx rows of a piece = sum of the reduction's slices, in order
__global__ void __launch_bounds__(256) lce_slices_kernel(const float *__restrict__ part, int64_t slice, int64_t ld, int splits, int rows, int base,
                                                         const Counters *cnt, int K, const int *__restrict__ idx, float *__restrict__ dx)
{
    s16::let_next_in();
    s16::after_previous();
    const int live = min(rows, cnt->count - base);
    for (int row = blockIdx.x; row < live; row += gridDim.x)
    {
        float *out = dx + static_cast<int64_t>(idx[row]) * K;
        for (int c = threadIdx.x; c < K; c += 256)
        {
            float s = 0.f;
            for (int k = 0; k < splits; ++k)
                s += part[k * slice + row * ld + c];
            out[c] = s;
        }
    }
}

// block 0: the loss, its rows added in a fixed order in double; the others: db from the column sums of the row blocks
__global__ void __launch_bounds__(256) lce_finish_kernel(const float *__restrict__ row_loss, const float *__restrict__ colsum, int64_t ld, int rows_per_sum,
                                                         int N, const Counters *cnt, float grad_scale, float *__restrict__ db, float *loss, int *err)
{
    __shared__ double box[8];
    s16::let_next_in();
    s16::after_previous();
    const int n = cnt->count;
    if (blockIdx.x > 0)
    {
        const int c = (blockIdx.x - 1) * 256 + threadIdx.x;
        if (c >= N)
            return;
        // (pieces are multiples of the row blocks)
        const int groups = (n + rows_per_sum - 1) / rows_per_sum;
        float s          = 0.f;
#pragma unroll 8
        for (int k = 0; k < groups; ++k)
            s += colsum[k * ld + c];
        db[c] = s * (grad_scale * cnt->inv_count);
        return;
    }
    double s = 0;
    for (int i = threadIdx.x; i < n; i += 256)
        s += row_loss[i];
    for (int o = 16; o > 0; o >>= 1)
        s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0)
        box[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0)
    {
        for (int w = 1; w < 8; ++w)
            s += box[w];
        if (loss)
            *loss = n > 0 ? static_cast<float>(s / n) : 0.f;
        if (cnt->bad && *err == 0)
            atomicExch(err, 4);  // last: launches of the library leave early while the flag is up
    }
}

template <bool SCALED, class Epi>
int gemm(const s16::Plan &plan, int terms, const Split16 &A, const Split16 &B, const GemmArgs &g, const typename Epi::Params &ep, cudaStream_t stream)
{
    return terms == 3 ? s16::launch_plan<3, SCALED, Epi>(plan, A, B, g, ep, stream) : s16::launch_plan<1, SCALED, Epi>(plan, A, B, g, ep, stream);
}

// Test hook: rows of a piece, a multiple of 256 (0 = from kPieceBytes).
int g_lce_piece = 0;

inline bool aligned32(const float *p, int64_t ld)
{
    return !(reinterpret_cast<uintptr_t>(p) & 31) && !(ld & 7);
}
}  // namespace

int linear_cross_entropy(const float *x, const float *w, const float *b, const void *labels, int is64, int64_t ignore_index,
                         int64_t M, int64_t N, int64_t K, int w_layout, float *loss, float *lse_out, float *dx, float *dw, float *db,
                         float grad_scale, int precision, cudaStream_t stream)
{
    if (w_layout != ODL_W_OUT_IN && w_layout != ODL_W_IN_OUT)
    {
        set_last_error("linear_cross_entropy: unknown weight layout %d", w_layout);
        return kInvalidArgument;
    }
    if (precision != ODL_PRECISION_3XTF32 && precision != ODL_PRECISION_TF32)
    {
        set_last_error("linear_cross_entropy: unknown precision %d", precision);
        return kInvalidArgument;
    }
    if (!x || !w || !labels || M <= 0 || N <= 0 || K <= 0 || (!loss && !lse_out && !dx && !dw && !db))
    {
        set_last_error("linear_cross_entropy: invalid argument (M=%lld N=%lld K=%lld)", (long long)M, (long long)N, (long long)K);
        return kInvalidArgument;
    }
    if (M > 0x3fffffff || N > 0x3fffffff || K > 64 * 65535)
    {
        set_last_error("linear_cross_entropy: M or N exceeds 2^30, or K 64 * 65535");
        return kTooLarge;
    }
    if (!is_ready())
    {
        set_last_error("odl_init has not been called");
        return kNotInitialized;
    }
    const int terms    = precision == ODL_PRECISION_3XTF32 ? 3 : 1;
    const bool grads   = dx || dw || db;
    if (!grads && !g_lce_piece && linear_ce_few_eligible(M, N, K, w, w_layout))
        return linear_ce_few(x, w, b, labels, is64, ignore_index, M, N, K, w_layout, loss, lse_out, precision, stream);
    const bool out_in  = w_layout == ODL_W_OUT_IN;
    const int kp = s16::pad64(K), np = s16::pad64(N), ks = (kp + 127) / 128;  // (scales of 128 columns)
    const int64_t m_pad = (M + 127) / 128 * 128;

    // rows per piece
    int64_t piece = grads ? kPieceBytes / (static_cast<int64_t>(np) * 4) : 65536;
    piece         = piece < 256 ? 256 : piece / 256 * 256;
    if (g_lce_piece > 0)
        piece = g_lce_piece;
    if (piece > m_pad)
        piece = m_pad;
    const int R = static_cast<int>(piece < M ? piece : M);

    GemmArgs gz{};
    gz.M = R, gz.N = (int)N, gz.K = (int)K, gz.batch = 1, gz.splits = 1;
    const s16::Plan plan_z = s16::plan_tiles(R, N, K, terms, 1, false);
    const s16::Plan plan_x = s16::plan_tiles(R, K, N, terms, 1, true);
    const s16::Plan plan_w = out_in ? s16::plan_tiles(N, K, R, terms, 1, false) : s16::plan_tiles(K, N, R, terms, 1, false);
    const int strips       = 2 * plan_z.tiles_n(N);
    // the softmax pass: blocks of 128 rows x 512 columns, of 32 rows where those would be fewer than the SMs
    const int64_t sm_cols = (np + 511) / 512;
    const int sum_rows    = (R + 127) / 128 * sm_cols < s16::sm_count() ? 32 : 128;
    const bool own_lse    = sum_rows == 32 && sm_cols == 1;  // (a block over all columns: nobody else needs its rows' lse)

    const size_t scale_w = a256((N + 127) / 128 * ks * 4), scale_x = a256(m_pad / 128 * ks * 4);
    const size_t bytes   = 3 * a256(M * 4) + 256 + a256(N * static_cast<int64_t>(kp) * 4) + scale_w + a256(m_pad * kp * 4) + scale_x +
                         a256(static_cast<int64_t>(strips) * R * 8) + 3 * a256(piece * 4) + a256(M * 4) +
                         (grads ? a256(piece * np * 4) : 0) + (db ? a256(m_pad / sum_rows * static_cast<int64_t>(np) * 4) : 0) +
                         (dx && plan_x.splits > 1 ? a256(static_cast<int64_t>(plan_x.splits) * R * kp * 4) : 0);
    int rc = arena_begin(bytes, stream);
    if (rc)
        return rc;
    const ArenaUse use{stream};
    auto take          = [&](size_t n) { return arena_alloc(n); };
    int *idx           = static_cast<int *>(take(M * 4));
    int *cls           = static_cast<int *>(take(M * 4));
    int *pos_of        = static_cast<int *>(take(M * 4));
    Counters *cnt      = static_cast<Counters *>(take(256));
    float *row_loss    = static_cast<float *>(take(M * 4));
    Split16 W, X;
    W.data = static_cast<const __half *>(take(N * static_cast<int64_t>(kp) * 4));
    W.pitch = 2 * kp, W.rows = (int)N, W.cols_pad = kp;
    float *w_scale = static_cast<float *>(take(scale_w));
    W.scale        = w_scale;
    X.data         = static_cast<const __half *>(take(m_pad * kp * 4));
    X.pitch = 2 * kp, X.rows = (int)M, X.cols_pad = kp;
    float *x_scale = static_cast<float *>(take(scale_x));
    X.scale        = x_scale;
    float2 *part   = static_cast<float2 *>(take(static_cast<int64_t>(strips) * R * 8));
    float *lse     = static_cast<float *>(take(piece * 4));
    float *picked  = static_cast<float *>(take(piece * 4));
    float *z       = grads ? static_cast<float *>(take(piece * np * 4)) : nullptr;
    float *colsum  = db ? static_cast<float *>(take(m_pad / sum_rows * static_cast<int64_t>(np) * 4)) : nullptr;
    float *slices  = dx && plan_x.splits > 1 ? static_cast<float *>(take(static_cast<int64_t>(plan_x.splits) * R * kp * 4)) : nullptr;

    lce_labels_kernel<<<1, 1024, 0, stream>>>(labels, is64, ignore_index, (int)M, (int)N, idx, cls, pos_of, cnt);
    LCE_LAUNCHED();
    {
        s16::ZeroRows zero{pos_of, dx, lse_out, (int)M, (int)K, 0};
        if (dx || lse_out)
            zero.blocks = (int)((M + 15) / 16 < 296 ? (M + 15) / 16 : 296);
        if ((rc = s16::split16_encode(s16::encode_job(w, out_in ? K : N, !out_in, (int)N, (int)K, nullptr, nullptr, W, w_scale),
                                      s16::encode_job(x, K, 0, (int)M, (int)K, idx, &cnt->count, X, x_scale), zero, stream)))
            return rc;
    }
    gz.err = device_error_flag();
    for (int64_t base = 0; base < M; base += piece)
    {
        const int rows = static_cast<int>(M - base < piece ? M - base : piece);
        // this piece's rows of x
        Split16 Xp = X;
        Xp.data += base * X.pitch;
        Xp.rows  = rows;
        Xp.scale = x_scale + base / 128 * ks;
        GemmArgs g   = gz;
        g.M          = rows;
        g.count      = &cnt->count;
        g.count_base = (int)base;
        g.count_dim  = 1;
        EpiLogits::Params ez{b, cls + base, part, R, picked, z, np};
        if ((rc = gemm<true, EpiLogits>(plan_z, terms, Xp, W, g, ez, stream)))
            return rc;
        const LseArgs lse_args{part, R, strips, rows, (int)base, cnt, idx + base, picked, lse, row_loss, lse_out};
        if (!(grads && own_lse) && (rc = s16::launch_after(lce_lse_kernel, dim3((rows + 31) / 32), dim3(512), 0, stream, lse_args)))
            return rc;
        if (!grads)
            continue;
        auto softmax       = sum_rows == 32 ? lce_softmax_kernel<32> : lce_softmax_kernel<128>;
        const int row_blks = (rows + 127) / 128 * (128 / sum_rows);
        if ((rc = s16::launch_after(softmax, dim3(row_blks, (unsigned)sm_cols), dim3(256), 0, stream, z, np, (int)N, (int)piece, lse_args, cls + base,
                                    own_lse ? 1 : 0, db ? colsum + base / sum_rows * static_cast<int64_t>(np) : nullptr)))
            return rc;
        Split16 P;
        P.data = reinterpret_cast<const __half *>(z);
        P.pitch = 2 * static_cast<int64_t>(np), P.rows = (int)piece, P.cols_pad = np;
        if (dx)
        {
            GemmArgs gx = g;
            gx.N = (int)K, gx.K = (int)N, gx.b_mn = 1, gx.splits = plan_x.splits;
            EpiGrad::Params ex{slices ? slices : dx, slices ? kp : K, slices ? nullptr : idx + base, cnt, grad_scale / kPScale, 0,
                               static_cast<int64_t>(R) * kp, slices ? 1 : aligned32(dx, K)};
            if ((rc = gemm<true, EpiGrad>(plan_x, terms, P, W, gx, ex, stream)))
                return rc;
            if (slices)
            {
                if ((rc = s16::launch_after(lce_slices_kernel, dim3(rows < 1184 ? rows : 1184), dim3(256), 0, stream, slices, ex.slice, kp, plan_x.splits,
                                            rows, (int)base, cnt, (int)K, idx + base, dx)))
                    return rc;
            }
        }
        if (dw)
        {
            GemmArgs gw  = g;
            gw.M         = out_in ? (int)N : (int)K;
            gw.N         = out_in ? (int)K : (int)N;
            gw.K         = rows;
            gw.a_mn = gw.b_mn = 1;
            gw.count_dim      = 2;
            EpiGrad::Params ew{dw, out_in ? K : N, nullptr, cnt, grad_scale / kPScale, base > 0, 0, aligned32(dw, out_in ? K : N)};
            if ((rc = out_in ? gemm<true, EpiGrad>(plan_w, terms, P, Xp, gw, ew, stream) : gemm<true, EpiGrad>(plan_w, terms, Xp, P, gw, ew, stream)))
                return rc;
        }
    }
    if ((rc = s16::launch_after(lce_finish_kernel, dim3(1 + (db ? ((int)N + 255) / 256 : 0)), dim3(256), 0, stream, row_loss, colsum, np, sum_rows, (int)N,
                                cnt, grad_scale, db, loss, device_error_flag())))
        return rc;
    return kOk;
}

}  // namespace odl

extern "C" int odl_debug_set_loss_piece(int rows)
{
    odl::g_lce_piece = rows > 0 ? (rows + 255) / 256 * 256 : 0;
    return 0;
}

extern "C" int odl_linear_cross_entropy(const float *x, const float *w, const float *b, const void *labels, int labels_are_int64,
                                        int64_t ignore_index, int64_t M, int64_t N, int64_t K, int w_layout, float *loss,
                                        float *lse, float *dx, float *dw, float *db, float grad_scale, int precision, void *stream)
{
    return odl::linear_cross_entropy(x, w, b, labels, labels_are_int64, ignore_index, M, N, K, w_layout, loss, lse, dx, dw, db,
                                     grad_scale, precision, static_cast<cudaStream_t>(stream));
}
