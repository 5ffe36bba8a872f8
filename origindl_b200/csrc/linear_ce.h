// The forms of odl_linear_cross_entropy behind its argument checks (linear_ce.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace odl
{

// Loss and log-sum-exp of few rows, straight from the fp32 weights (linear_ce_few.cu).
bool linear_ce_few_eligible(int64_t M, int64_t N, int64_t K, const float *w, int w_layout);
int linear_ce_few(const float *x, const float *w, const float *b, const void *labels, int is64, int64_t ignore_index, int64_t M, int64_t N,
                  int64_t K, int w_layout, float *loss, float *lse_out, int precision, cudaStream_t stream);

}  // namespace odl
