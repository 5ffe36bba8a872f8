// What the two forms of the Newton-Schulz iteration share (muon.cu: any size; muon_small.cu: one side of at most 128).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "gemm_tc.cuh"

namespace odl
{

constexpr float kNsA = 3.4445f, kNsB = -4.7750f, kNsC = 2.0315f;
// b s + c s^2 = c s (s + h)
constexpr float kNsH = static_cast<float>(-4.7750 / 2.0315);
constexpr float kSx = 16384.f, kSa = 16384.f, kSs = 8192.f;  // halves hold value * this

struct MomentumArgs
{
    float momentum, hook_wd, grad_scale;
    int nesterov;
};

// where the result goes: written out, or the parameters' update
struct NsOut
{
    float *out;      // result, or parameters (param != 0)
    float *small;    // low part of the parameters, may be null
    float keep, rate;
    int param;
};

#ifdef __CUDACC__
// buf = momentum * buf + g, u = nesterov ? g + momentum * buf : buf (operation by operation as in the SGD step)
__device__ __forceinline__ float momentum_one(float &g, float &buf, float p, bool has_buf, const MomentumArgs &a)
{
    if (a.grad_scale != 1.f)
        g = __fmul_rn(g, a.grad_scale);
    if (a.hook_wd > 0.f)
        g = __fadd_rn(g, __fmul_rn(p, a.hook_wd));
    if (!has_buf)
        return g;
    buf = __fadd_rn(__fmul_rn(buf, a.momentum), g);
    return a.nesterov ? __fadd_rn(g, __fmul_rn(buf, a.momentum)) : buf;
}

// Sum of the squares of N values, in double, whatever their size.  Conversions to double are slow (a few a cycle and SM): the
// values are scaled by the power of two of the largest, their squares added in fp32, and the one sum converted.
template <int N>
__device__ __forceinline__ double square_sum(const float (&u)[N])
{
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
        top = fmaxf(top, fabsf(u[i]));
    const int e   = max(1, min(253, static_cast<int>(__float_as_uint(top) >> 23)));  // biased exponent
    const float f = __int_as_float((254 - e) << 23);                                 // 2^(127 - e)
    float q       = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
        q = fmaf(u[i] * f, u[i] * f, q);
    return static_cast<double>(q) * __hiloint2double((1023 + 2 * (e - 127)) << 20, 0);
}

// u / norm as floats without a double per element: 1 / norm as the sum of two floats, and a power of two in front where the
// first alone would leave the normal range
struct InverseNorm
{
    float pre, hi, lo;
    __device__ __forceinline__ float times(float u) const
    {
        const float v = u * pre;
        return fmaf(v, hi, v * lo);
    }
};
__device__ __forceinline__ InverseNorm inverse_norm(double norm, double eps, double scale)
{
    const double d = norm > eps || !(norm == norm) ? norm : eps;
    InverseNorm r;
    r.pre            = d > 1e30 ? 1.f / 1099511627776.f : 1.f;  // 2^-40
    const double inv = scale / (d * r.pre);
    r.hi             = static_cast<float>(inv);
    r.lo             = static_cast<float>(inv - r.hi);
    return r;
}

__device__ __forceinline__ float ns_result(const NsOut &o, float x, float was)
{
    return o.param ? __fsub_rn(__fmul_rn(was, o.keep), __fmul_rn(o.rate, x)) : x;
}
#endif

bool muon_small_eligible(int64_t rows, int64_t cols, int steps);
// p: parameters for the weight-decay hook (null: none); buf null: u = g
int muon_small(const float *p, float *g, float *buf, const MomentumArgs &a, const NsOut &out, int64_t batch, int64_t rows, int64_t cols, int steps,
               float eps, int terms, cudaStream_t stream);

}  // namespace odl
