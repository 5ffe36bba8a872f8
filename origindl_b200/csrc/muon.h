// What the two forms of the Newton-Schulz iteration share (muon.cu: any size; muon_small.cu: one side of at most 128).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "gemm_tc.cuh"

namespace odl
{

constexpr float kNsA = 3.4445f, kNsB = -4.7750f, kNsC = 2.0315f;
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
