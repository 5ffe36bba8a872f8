// Softmax cross entropy of a linear head: loss, log-sum-exp and the gradients of x, W and b from one call that never hands
// the logits out.
//   z = x W^T + b;   lse_i = log sum_j exp z_ij;   loss = 1/n sum_{i valid} (lse_i - z_{i,t_i}),  n = valid rows
//   P_ij = exp(z_ij - lse_i) - [j = t_i]  (0 in rows without a label);   dx = g P W,  dW = g P^T x,  db = g colsum(P),
//   g = grad_scale / n
#include <cuda_runtime.h>

#include <cmath>

#include "../../include/odl_b200.h"
#include "gemm_tc.cuh"
#include "host_util.h"
#include "internal.h"

namespace odl
{

namespace
{
inline size_t a256(size_t x)
{
    return (x + 255) & ~size_t(255);
}

// labels -> 32-bit class of every row, -1 where the row takes no part; count of the others and 1 / count.
__global__ void __launch_bounds__(1024) lce_labels_kernel(const void *labels, int is64, int64_t ignore, int M, int N, int *cls,
                                                          int *count, float *inv_count, int *bad)
{
    __shared__ int total;
    if (threadIdx.x == 0)
        total = 0, *bad = 0;
    __syncthreads();
    int mine = 0;
    for (int i = threadIdx.x; i < M; i += 1024)
    {
        const int64_t t = is64 ? static_cast<const int64_t *>(labels)[i] : static_cast<const int32_t *>(labels)[i];
        int c           = -1;
        if (t != ignore)
        {
            if (t >= 0 && t < N)
                c = static_cast<int>(t);
            else
                atomicExch(bad, 1);
        }
        cls[i] = c;
        mine += c >= 0;
    }
    atomicAdd(&total, mine);
    __syncthreads();
    if (threadIdx.x == 0)
    {
        *count     = total;
        *inv_count = total > 0 ? 1.0f / static_cast<float>(total) : 0.f;
    }
}

// rows without a label become zeros: nothing they hold (NaN, infinities) reaches a product
__global__ void lce_rows_kernel(const float *x, const int *cls, int64_t n, int K, float *out)
{
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * blockDim.x)
        out[i] = cls[i / K] >= 0 ? x[i] : 0.f;
}

__device__ __forceinline__ float block_reduce(float v, bool is_max)
{
    __shared__ float box[32];
    for (int o = 16; o > 0; o >>= 1)
    {
        const float u = __shfl_xor_sync(0xffffffffu, v, o);
        v             = is_max ? fmaxf(v, u) : v + u;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0)
        box[threadIdx.x >> 5] = v;
    __syncthreads();
    v = box[0];
    for (int w = 1; w < static_cast<int>(blockDim.x) / 32; ++w)
        v = is_max ? fmaxf(v, box[w]) : v + box[w];
    return v;
}

// one block per row: statistics, the row's loss, and the logits replaced by g * P
__global__ void __launch_bounds__(256) lce_row_kernel(float *z, int N, const int *cls, const float *inv_count, float grad_scale,
                                                      float *row_loss, float *lse_out, int want_grad)
{
    const int row = blockIdx.x;
    float *zr     = z + static_cast<int64_t>(row) * N;
    const int c   = cls[row];
    float m       = -INFINITY;
    for (int j = threadIdx.x; j < N; j += 256)
        m = fmaxf(m, zr[j]);
    m       = block_reduce(m, true);
    float s = 0.f;
    for (int j = threadIdx.x; j < N; j += 256)
        s += expf(zr[j] - m);
    s               = block_reduce(s, false);
    const float lse = m + logf(s);
    if (threadIdx.x == 0)
    {
        row_loss[row] = c >= 0 ? lse - zr[c] : 0.f;
        if (lse_out)
            lse_out[row] = c >= 0 ? lse : 0.f;
    }
    __syncthreads();
    if (want_grad)
    {
        const float g = grad_scale * *inv_count;
        for (int j = threadIdx.x; j < N; j += 256)
            zr[j] = c >= 0 ? (expf(zr[j] - lse) - (j == c ? 1.f : 0.f)) * g : 0.f;
    }
}

__global__ void __launch_bounds__(1024) lce_loss_kernel(const float *row_loss, int M, const int *count, const int *bad, float *loss, int *err)
{
    __shared__ double box[32];
    double s = 0;
    for (int i = threadIdx.x; i < M; i += 1024)
        s += row_loss[i];
    for (int o = 16; o > 0; o >>= 1)
        s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0)
        box[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0)
    {
        for (int w = 1; w < 32; ++w)
            s += box[w];
        if (loss)
            *loss = *count > 0 ? static_cast<float>(s / *count) : 0.f;
        if (*bad)
            atomicExch(err, 4);  // last: launches of the library leave early while the flag is up
    }
}
}  // namespace

int linear_cross_entropy(const float *x, const float *w, const float *b, const void *labels, int is64, int64_t ignore_index,
                         int64_t M, int64_t N, int64_t K, int w_layout, float *loss, float *lse, float *dx, float *dw, float *db,
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
    if (!x || !w || !labels || M <= 0 || N <= 0 || K <= 0 || (!loss && !lse && !dx && !dw && !db))
    {
        set_last_error("linear_cross_entropy: invalid argument (M=%lld N=%lld K=%lld)", (long long)M, (long long)N, (long long)K);
        return kInvalidArgument;
    }
    if (M > 0x3fffffff || N > 0x3fffffff || K > 0x3fffffff)
    {
        set_last_error("linear_cross_entropy: dimension exceeds 2^30");
        return kTooLarge;
    }
    if (!is_ready())
    {
        set_last_error("odl_init has not been called");
        return kNotInitialized;
    }
    const int terms    = precision == ODL_PRECISION_3XTF32 ? 3 : 1;
    const int64_t ldw  = w_layout == ODL_W_OUT_IN ? K : N;
    const int64_t wr   = w_layout == ODL_W_OUT_IN ? N : K;
    const bool grads   = dx || dw || db;
    auto padded        = [&](int64_t r, int64_t c) { return 2 * a256(static_cast<size_t>(r) * ((c + 3) & ~int64_t(3)) * 4); };
    const size_t total = a256(M * 4) * 2 + 512 + a256(M * K * 4) + a256(M * N * 4) + 2 * padded(M, K) + 2 * padded(wr, ldw) + 2 * padded(M, N);
    int rc             = arena_begin(total, stream);
    if (rc)
        return rc;
    int *cls        = static_cast<int *>(arena_alloc(M * 4));
    float *row_loss = static_cast<float *>(arena_alloc(M * 4));
    int *count      = static_cast<int *>(arena_alloc(256));
    float *inv      = reinterpret_cast<float *>(count + 1);
    int *bad        = count + 2;
    float *xg       = static_cast<float *>(arena_alloc(M * K * 4));
    float *z        = static_cast<float *>(arena_alloc(M * N * 4));
    lce_labels_kernel<<<1, 1024, 0, stream>>>(labels, is64, ignore_index, (int)M, (int)N, cls, count, inv, bad);
    lce_rows_kernel<<<1184, 256, 0, stream>>>(x, cls, M * K, (int)K, xg);
    g_launch_count += 2;
    rc = gemm_dispatch(0, w_layout == ODL_W_OUT_IN ? 1 : 0, M, N, K, xg, nullptr, K, w, nullptr, ldw, z, nullptr, N, b, nullptr, 0,
                       nullptr, b ? kEpiBias : 0, precision, stream, false);
    if (rc)
        return rc;
    lce_row_kernel<<<(int)M, 256, 0, stream>>>(z, (int)N, cls, inv, grad_scale, row_loss, lse, grads);
    ++g_launch_count;
    (void)terms;
    if (dx && (rc = gemm_dispatch(0, w_layout == ODL_W_OUT_IN ? 0 : 1, M, K, N, z, nullptr, N, w, nullptr, ldw, dx, nullptr, K,
                                  nullptr, nullptr, 0, nullptr, 0, precision, stream, false)))
        return rc;
    if (dw && (rc = w_layout == ODL_W_OUT_IN ? gemm_dispatch(1, 0, N, K, M, z, nullptr, N, xg, nullptr, K, dw, nullptr, K, nullptr,
                                                             nullptr, 0, nullptr, 0, precision, stream, false)
                                             : gemm_dispatch(1, 0, K, N, M, xg, nullptr, K, z, nullptr, N, dw, nullptr, N, nullptr,
                                                             nullptr, 0, nullptr, 0, precision, stream, false)))
        return rc;
    if (db)
    {
        ODL_CUDA_TRY(cudaMemsetAsync(db, 0, static_cast<size_t>(N) * 4, stream));
        if ((rc = split_launch(z, N, (int)M, (int)N, nullptr, 0, nullptr, nullptr, N, db, stream)))
            return rc;
    }
    lce_loss_kernel<<<1, 1024, 0, stream>>>(row_loss, (int)M, count, bad, loss, device_error_flag());
    ++g_launch_count;
    ODL_CUDA_TRY(cudaGetLastError());
    return arena_end(stream);
}

}  // namespace odl

extern "C" int odl_linear_cross_entropy(const float *x, const float *w, const float *b, const void *labels, int labels_are_int64,
                                        int64_t ignore_index, int64_t M, int64_t N, int64_t K, int w_layout, float *loss,
                                        float *lse, float *dx, float *dw, float *db, float grad_scale, int precision, void *stream)
{
    return odl::linear_cross_entropy(x, w, b, labels, labels_are_int64, ignore_index, M, N, K, w_layout, loss, lse, dx, dw, db,
                                     grad_scale, precision, static_cast<cudaStream_t>(stream));
}
