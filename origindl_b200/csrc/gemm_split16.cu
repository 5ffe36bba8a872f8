// Host side of the split-fp16 GEMM: tensor maps and how many CTAs of a kernel the GPU holds; and the pass that splits a
// fp32 matrix tile by tile.
#include "gemm_split16.cuh"

#include "internal.h"
#include "split16_encode.h"

namespace odl
{
namespace s16
{

int make_tmap_split16(CUtensorMap *out, const Split16 &m, int box_rows)
{
    return make_tmap_half3d(out, m.data, 2 * static_cast<int64_t>(m.cols_pad), m.rows, m.batch, m.pitch, m.batch_stride, kBK, box_rows);
}

int sm_count()
{
    static int n = 0;
    if (n == 0)
    {
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
            n = 148;
    }
    return n;
}

// CTAs (cluster == 1) or CTA pairs of `kernel` the device holds at once; 0 with the error text set on failure.
int resident_ctas(const void *kernel, int cluster, int smem)
{
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess)
    {
        set_last_error("cudaFuncSetAttribute(smem=%d) failed: %s", smem, cudaGetErrorString(e));
        return 0;
    }
    if (cluster == 1)
        return sm_count();
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim          = dim3(static_cast<unsigned>(sm_count() & ~1), 1, 1);
    cfg.blockDim         = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id               = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs                = attr;
    cfg.numAttrs             = 1;
    int n                    = 0;
    e                        = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
    if (e != cudaSuccess || n <= 0)
    {
        set_last_error("no CTA pair of the split-fp16 GEMM fits: %s", cudaGetErrorString(e));
        return 0;
    }
    return n;
}

Plan plan_tiles(int64_t M, int64_t N, int64_t K, int terms, int batch, bool may_split, bool sym)
{
    // Times in units of a K-block of the pair's tile (1536 cycles with three products): a 128 x 128 tile's products take 0.5 of
    // that on its SM, a 128 x 64 tile's 0.375 (shared-memory reads: 192 bytes a cycle for full rate, 128 there).  What the
    // L2 -> SM fabric delivers, 10 MB a unit over all SMs, bounds the small tiles once many SMs run them: on 4096^3 the
    // 128 x 128 tile kept the tensor pipe 57 % busy at 11 TB/s and took 386 us, the pair's tile 87 % and 309 us.
    struct Kind
    {
        int cg, bn;
        double per_kb, bytes, fixed;  // of a tile: a K-block's products and bytes, filling the ring + storing
    };
    const double parts  = terms == 3 ? 1.0 : 1.0 / 3;  // products; bytes are a half
    const double bytes_ = terms == 3 ? 1.0 : 0.5;
    const Kind kinds[3] = {{2, 256, 1.0, 131072, 4.0}, {1, 128, 0.5, 65536, 3.0}, {1, 64, 0.375, 49152, 2.5}};
    const int64_t n_kb  = (K + kBK - 1) / kBK;
    Plan best;
    double best_t = 1e300;
    for (const Kind &k : kinds)
    {
        const int bm = 128 * k.cg;
        if (sym && bm != k.bn)
            continue;  // (a symmetric output needs square tiles)
        if (g_bn_override && (sym && g_bn_override == 64 ? 128 : g_bn_override) != k.bn)
            continue;
        const int64_t slots = sm_count() / k.cg;
        const int64_t tn = (N + k.bn - 1) / k.bn, tm = (M + bm - 1) / bm;
        const int64_t tiles = (sym ? tn * (tn + 1) / 2 : tm * tn) * batch;
        for (int s = 1; s <= (may_split ? 16 : 1); ++s)
        {
            const int64_t kb = (n_kb + s - 1) / s;
            if (may_split && g_split_k > 0 ? s != g_split_k : s > 1 && kb < 8)
                continue;
            const int64_t units = tiles * s, waves = (units + slots - 1) / slots, full = units / slots;
            const double busy = static_cast<double>(units < slots ? units : slots), rest = static_cast<double>(units - full * slots);
            auto kb_time = [&](double active) {
                const double fabric = active * k.bytes * bytes_ / 10e6;
                return k.per_kb * parts > fabric ? k.per_kb * parts : fabric;
            };
            // slices are written and read once more: M N s floats there and back
            const double t = (full * kb_time(busy) + (rest > 0 ? kb_time(rest) : 0.0)) * kb + waves * k.fixed +
                             (s > 1 ? 4.0 + static_cast<double>(M) * N * batch * s * 8 / 5e6 : 0.0);
            if (t < best_t)
                best_t = t, best.cg = k.cg, best.bn = k.bn, best.splits = s;
        }
    }
    return best;
}

namespace
{
// One 128 x 64 tile per block: read once, its largest finite value gives the tile's power of two, written as halves.
// Bound by memory: 4 bytes in and 4 out per value.  TRANSPOSED: element (r, c) is src[c * ld + r].
template <bool TRANSPOSED>
__global__ void __launch_bounds__(256) split16_tiles_kernel(const float *__restrict__ src, int64_t ld, int rows, int cols, const int *__restrict__ gather,
                                                            const int *__restrict__ count, __half *__restrict__ out, int64_t pitch,
                                                            float *__restrict__ scale, int blocks_c, bool vec)
{
    // neighbouring blocks take neighbouring columns: rows are read in long stretches (DRAM pages), not 256 bytes at a time
    const int block_c = blockIdx.x % blocks_c, block_r = blockIdx.x / blocks_c;
    const int c0 = block_c * 64, r0 = block_r * 128;
    const int live = count ? min(rows, *count) : rows;
    if (r0 >= live)
        return;  // (gathered matrices: nobody reads rows past the last 128 that hold any)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float2 v[16];
    if (TRANSPOSED)
    {
        __shared__ float tile[64][129];
        for (int i = warp; i < 64; i += 8)
        {
            const float *line = src + (c0 + i) * ld + r0;
            for (int j = 0; j < 4; ++j)
            {
                const int r           = lane + 32 * j;
                tile[i][r] = (c0 + i < cols && r0 + r < live) ? __ldg(line + r) : 0.f;
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 16; ++i)
            v[i] = make_float2(tile[2 * lane][warp + 8 * i], tile[2 * lane + 1][warp + 8 * i]);
    }
    else
    {
        const int c = c0 + 2 * lane;
#pragma unroll
        for (int i = 0; i < 16; ++i)
        {
            const int r = r0 + warp + 8 * i;
            v[i]        = make_float2(0.f, 0.f);
            if (r < live)
            {
                const float *line = src + static_cast<int64_t>(gather ? gather[r] : r) * ld;
                if (vec)
                {
                    if (c < cols)
                        v[i] = __ldg(reinterpret_cast<const float2 *>(line + c));
                }
                else
                {
                    if (c < cols)
                        v[i].x = __ldg(line + c);
                    if (c + 1 < cols)
                        v[i].y = __ldg(line + c + 1);
                }
            }
        }
    }
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i)
    {
        // infinities and NaN stay what they are and choose no scale
        const float a = fabsf(v[i].x), b = fabsf(v[i].y);
        top = fmaxf(top, a < INFINITY ? a : 0.f);
        top = fmaxf(top, b < INFINITY ? b : 0.f);
    }
    __shared__ float box[8];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0)
        box[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w)
        top = fmaxf(top, box[w]);
    // s = 2^(e - 14) with 2^e <= top < 2^(e + 1): v / s below 2^15, fp16's largest is just under 2^16
    const int e     = top > 0.f ? max(ilogbf(top), -112) : 0;
    const float s   = __int_as_float((e - 14 + 127) << 23);
    const float inv = __int_as_float((127 - (e - 14)) << 23);
    if (threadIdx.x == 0)
        scale[blockIdx.x] = s;
#pragma unroll
    for (int i = 0; i < 16; ++i)
    {
        const int r = r0 + warp + 8 * i;
        if (r < (gather ? r0 + 128 : rows))
        {
            uint32_t hi, lo;
            split2(v[i].x * inv, v[i].y * inv, hi, lo);
            uint32_t *line = reinterpret_cast<uint32_t *>(out + r * pitch + 2 * c0);
            line[lane]      = hi;
            line[32 + lane] = lo;
        }
    }
}
}  // namespace

int split16_encode(const float *src, int64_t ld, int transposed, int rows, int cols, const int *gather, const int *count, const Split16 &out,
                   float *scale, cudaStream_t stream)
{
    const int blocks_c   = out.cols_pad / 64;
    const int64_t blocks = static_cast<int64_t>((rows + 127) / 128) * blocks_c;
    if (blocks > 0x7fffffff)
    {
        set_last_error("split: %d x %d is too large", rows, cols);
        return kTooLarge;
    }
    const unsigned grid = static_cast<unsigned>(blocks);
    const bool vec = !(cols & 1) && !(ld & 1) && !(reinterpret_cast<uintptr_t>(src) & 7);
    __half *dst    = const_cast<__half *>(out.data);
    if (transposed)
        split16_tiles_kernel<true><<<grid, 256, 0, stream>>>(src, ld, rows, cols, gather, count, dst, out.pitch, scale, blocks_c, vec);
    else
        split16_tiles_kernel<false><<<grid, 256, 0, stream>>>(src, ld, rows, cols, gather, count, dst, out.pitch, scale, blocks_c, vec);
    ++g_launch_count;
    ODL_CUDA_TRY(cudaGetLastError());
    return kOk;
}

}  // namespace s16
}  // namespace odl
