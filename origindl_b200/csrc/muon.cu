// Orthogonalised updates of weight matrices: the quintic Newton-Schulz iteration and the momentum step around it.
//   X_0 = u / max(|u|_F, eps);   X <- a X + (b A + c A^2) X,  A = X X^T  (X^T X for tall matrices: the smaller side)
// with (a, b, c) = (3.4445, -4.7750, 2.0315) drives the singular values of X towards 1.
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
constexpr float kNsA = 3.4445f, kNsB = -4.7750f, kNsC = 2.0315f;
constexpr int kNormBlocks = 256;

inline size_t a256(size_t x)
{
    return (x + 255) & ~size_t(255);
}

struct MomentumArgs
{
    float momentum, hook_wd, grad_scale;
    int nesterov;
};

// buf = momentum * buf + g, u = nesterov ? g + momentum * buf : buf (the order of the SGD step); squares summed in double
__global__ void __launch_bounds__(256) muon_momentum_kernel(const float *p, float *g, float *buf, float *u, int64_t n, MomentumArgs a,
                                                            double *partial)
{
    double s           = 0;
    const bool write_g = p && (a.hook_wd > 0.f || a.grad_scale != 1.f);
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256)
    {
        float v = g[i];
        if (a.grad_scale != 1.f)
            v = __fmul_rn(v, a.grad_scale);
        if (p && a.hook_wd > 0.f)
            v = __fadd_rn(v, __fmul_rn(p[i], a.hook_wd));
        if (write_g)
            g[i] = v;
        if (buf)
        {
            const float m = __fadd_rn(__fmul_rn(buf[i], a.momentum), v);
            buf[i]        = m;
            v             = a.nesterov ? __fadd_rn(v, __fmul_rn(m, a.momentum)) : m;
        }
        u[i] = v;
        s += static_cast<double>(v) * v;
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
        partial[blockIdx.x] = s;
    }
}

__global__ void __launch_bounds__(256) muon_scale_kernel(float *u, int64_t n, const double *partial, float eps)
{
    double s = 0;
    for (int i = 0; i < kNormBlocks; ++i)
        s += partial[i];
    const double norm = sqrt(s);
    const double inv  = 1.0 / (norm > eps ? norm : static_cast<double>(eps));
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256)
        u[i] = static_cast<float>(u[i] * inv);
}

// S = a I + b A + c A^2, in place of A^2
__global__ void muon_poly_kernel(float *s, const float *a, int m)
{
    const int64_t n = static_cast<int64_t>(m) * m;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256)
        s[i] = kNsC * s[i] + kNsB * a[i] + (i / m == i % m ? kNsA : 0.f);
}

__global__ void muon_update_kernel(float *p, const float *x, float *p_small, int64_t n, float keep, float rate)
{
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256)
    {
        const float v = __fsub_rn(__fmul_rn(p[i], keep), __fmul_rn(rate, x[i]));
        p[i]          = v;
        if (p_small)
            p_small[i] = tf32_small(v);
    }
}

int orthogonalise(const float *p, float *g, float *buf, const MomentumArgs &a, float *out, float *param, float *param_small,
                  float keep, float rate, int64_t batch, int64_t rows, int64_t cols, int steps, float eps, int precision,
                  cudaStream_t stream)
{
    const int64_t n = rows * cols, m = rows < cols ? rows : cols;
    const bool tall = rows > cols;
    auto padded     = [&](int64_t r, int64_t c) { return 2 * a256(static_cast<size_t>(r) * ((c + 3) & ~int64_t(3)) * 4); };
    int rc          = kOk;
    for (int64_t i = 0; i < batch; ++i)
    {
        if ((rc = arena_begin(2 * a256(n * 4) + 2 * a256(m * m * 4) + a256(kNormBlocks * 8) +
                                  steps * (4 * padded(rows, cols) + 6 * padded(m, m)),
                              stream)))
            return rc;
        float *x        = static_cast<float *>(arena_alloc(n * 4));
        float *y        = static_cast<float *>(arena_alloc(n * 4));
        float *A        = static_cast<float *>(arena_alloc(m * m * 4));
        float *S        = static_cast<float *>(arena_alloc(m * m * 4));
        double *partial = static_cast<double *>(arena_alloc(kNormBlocks * 8));
        muon_momentum_kernel<<<kNormBlocks, 256, 0, stream>>>(p ? p + i * n : nullptr, g + i * n, buf ? buf + i * n : nullptr, x, n, a, partial);
        muon_scale_kernel<<<592, 256, 0, stream>>>(x, n, partial, eps);
        g_launch_count += 2;
        for (int k = 0; k < steps; ++k)
        {
            rc = tall ? gemm_dispatch(1, 0, m, m, rows, x, nullptr, cols, x, nullptr, cols, A, nullptr, m, nullptr, nullptr, 0, nullptr, 0,
                                      precision, stream, false)
                      : gemm_dispatch(0, 1, m, m, cols, x, nullptr, cols, x, nullptr, cols, A, nullptr, m, nullptr, nullptr, 0, nullptr, 0,
                                      precision, stream, false);
            if (rc || (rc = gemm_dispatch(0, 0, m, m, m, A, nullptr, m, A, nullptr, m, S, nullptr, m, nullptr, nullptr, 0, nullptr, 0,
                                          precision, stream, false)))
                return rc;
            muon_poly_kernel<<<592, 256, 0, stream>>>(S, A, (int)m);
            ++g_launch_count;
            rc = tall ? gemm_dispatch(0, 0, rows, cols, m, x, nullptr, cols, S, nullptr, m, y, nullptr, cols, nullptr, nullptr, 0, nullptr,
                                      0, precision, stream, false)
                      : gemm_dispatch(0, 0, rows, cols, m, S, nullptr, m, x, nullptr, cols, y, nullptr, cols, nullptr, nullptr, 0, nullptr,
                                      0, precision, stream, false);
            if (rc)
                return rc;
            float *t = x;
            x = y, y = t;
        }
        if (param)
        {
            muon_update_kernel<<<592, 256, 0, stream>>>(param + i * n, x, param_small ? param_small + i * n : nullptr, n, keep, rate);
            ++g_launch_count;
        }
        else
            ODL_CUDA_TRY(cudaMemcpyAsync(out + i * n, x, n * 4, cudaMemcpyDeviceToDevice, stream));
        ODL_CUDA_TRY(cudaGetLastError());
        if ((rc = arena_end(stream)))
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
    return orthogonalise(nullptr, const_cast<float *>(g), nullptr, a, out, nullptr, nullptr, 1.f, 0.f, batch, rows, cols, steps, eps,
                         precision, static_cast<cudaStream_t>(stream));
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
    return orthogonalise(param, grad, momentum > 0.f ? momentum_buf : nullptr, a, nullptr, param, param_small,
                         static_cast<float>(1.0 - static_cast<double>(lr) * weight_decay), static_cast<float>(lr * s), batch, rows,
                         cols, steps, eps, precision, static_cast<cudaStream_t>(stream));
}
