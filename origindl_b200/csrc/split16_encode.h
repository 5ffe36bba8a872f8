// Splitting fp32 matrices into the two-halves form of gemm_split16.cuh.
#pragma once
#include <cuda_runtime.h>

#include "gemm_split16.cuh"

namespace odl
{
namespace s16
{

// out (rows x cols, tile scales in `scale`, [ceil(rows / 128)][ceil(cols_pad / 128)]) = src, row-major with pitch ld, or its transpose
// (element (r, c) at src[c * ld + r]).  gather (not with transposed): row r of out is row gather[r] of src, r < *count; the rows
// behind, up to a multiple of 128, become zeros (out holds that many).
struct EncodeJob
{
    const float *src;
    const int *gather, *count;
    __half *out;
    float *scale;
    int64_t ld, pitch, blocks;
    int transposed, rows, cols, cols_pad, blocks_c;
};
EncodeJob encode_job(const float *src, int64_t ld, int transposed, int rows, int cols, const int *gather, const int *count, const Split16 &out, float *scale);

// Rows of `matrix` (rows x cols, may be null) and words of `words` (may be null) with pos_of[row] < 0 become zero.
struct ZeroRows
{
    const int *pos_of;
    float *matrix, *words;
    int rows, cols, blocks;
};

int split16_encode(const EncodeJob &a, const EncodeJob &b, const ZeroRows &z, cudaStream_t stream);

}  // namespace s16
}  // namespace odl
