// Splitting a fp32 matrix into the two-halves form of gemm_split16.cuh.
#pragma once
#include <cuda_runtime.h>

#include "gemm_split16.cuh"

namespace odl
{
namespace s16
{

// out (rows x cols, tile scales in `scale`, [ceil(rows / 128)][cols_pad / 64]) = src, row-major with pitch ld, or its transpose
// (element (r, c) at src[c * ld + r]).  gather (not with transposed): row r of out is row gather[r] of src, r < *count; the rows
// behind, up to a multiple of 128, become zeros (out holds that many).
int split16_encode(const float *src, int64_t ld, int transposed, int rows, int cols, const int *gather, const int *count, const Split16 &out,
                   float *scale, cudaStream_t stream);

}  // namespace s16
}  // namespace odl
