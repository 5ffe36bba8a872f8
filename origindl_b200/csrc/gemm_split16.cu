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
// One 128 x 128 tile per block of 512 threads: read once, its largest finite value gives the tile's power of two, written as
// halves.  Bound by memory: 4 bytes in and 4 out per value.  A launch holds two matrices (x and W of a loss) and a range of blocks
// that put zeros into rows of `zero` (rows without a label: pos_of < 0).
constexpr int kTileThreads = 512;

__device__ __forceinline__ void split16_tile(const EncodeJob &j, int block, float (&box)[16], float (&tile)[64][129])
{
    // neighbouring blocks take neighbouring columns: rows are read in long stretches
    const int block_c = block % j.blocks_c, block_r = block / j.blocks_c;
    const int c0 = block_c * 128, r0 = block_r * 128;
    const int live = j.count ? min(j.rows, *j.count) : j.rows;
    if (r0 >= live)
        return;  // (gathered matrices: nobody reads rows past the last 128 that hold any)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int c = c0 + 4 * lane;  // thread: columns c .. c + 3 of rows warp + 16 i
    float4 v[8];
    if (j.transposed)
    {
        const bool vec = !(j.ld & 3) && !(reinterpret_cast<uintptr_t>(j.src) & 15) && r0 + 128 <= live;
#pragma unroll 1
        for (int h = 0; h < 2; ++h)  // 64 columns at a time through shared memory
        {
            __syncthreads();
            for (int i = warp; i < 64; i += 16)
            {
                const int col     = c0 + 64 * h + i;
                const float *line = j.src + col * j.ld + r0;
                if (vec && col < j.cols)
                {
                    const float4 q = __ldg(reinterpret_cast<const float4 *>(line) + lane);
                    tile[i][4 * lane] = q.x, tile[i][4 * lane + 1] = q.y, tile[i][4 * lane + 2] = q.z, tile[i][4 * lane + 3] = q.w;
                }
                else
                    for (int k = 0; k < 4; ++k)
                    {
                        const int r = lane + 32 * k;
                        tile[i][r]  = (col < j.cols && r0 + r < live) ? __ldg(line + r) : 0.f;
                    }
            }
            __syncthreads();
            if ((lane >> 4) == h)
            {
                const int cc = 4 * (lane & 15);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                {
                    const int r = warp + 16 * i;
                    v[i]        = make_float4(tile[cc][r], tile[cc + 1][r], tile[cc + 2][r], tile[cc + 3][r]);
                }
            }
        }
    }
    else
    {
        const bool vec = !(j.ld & 3) && !(j.cols & 3) && !(reinterpret_cast<uintptr_t>(j.src) & 15);
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            const int r = r0 + warp + 16 * i;
            v[i]        = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < live)
            {
                const float *line = j.src + static_cast<int64_t>(j.gather ? j.gather[r] : r) * j.ld + c;
                if (vec)
                {
                    if (c < j.cols)
                        v[i] = __ldg(reinterpret_cast<const float4 *>(line));
                }
                else
                {
                    if (c < j.cols)
                        v[i].x = __ldg(line);
                    if (c + 1 < j.cols)
                        v[i].y = __ldg(line + 1);
                    if (c + 2 < j.cols)
                        v[i].z = __ldg(line + 2);
                    if (c + 3 < j.cols)
                        v[i].w = __ldg(line + 3);
                }
            }
        }
    }
    float top = 0.f;
    // infinities and NaN stay what they are and choose no scale
    auto see = [&](float x) {
        x   = fabsf(x);
        top = fmaxf(top, x < INFINITY ? x : 0.f);
    };
#pragma unroll
    for (int i = 0; i < 8; ++i)
        see(v[i].x), see(v[i].y), see(v[i].z), see(v[i].w);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0)
        box[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 16; ++w)
        top = fmaxf(top, box[w]);
    // s = 2^(e - 14) with 2^e <= top < 2^(e + 1): v / s below 2^15, fp16's largest is just under 2^16
    const int e     = top > 0.f ? max(ilogbf(top), -112) : 0;
    const float s   = __int_as_float((e - 14 + 127) << 23);
    const float inv = __int_as_float((127 - (e - 14)) << 23);
    if (threadIdx.x == 0)
        j.scale[block] = s;
    if (c >= j.cols_pad)
        return;
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        const int r = r0 + warp + 16 * i;
        if (r < (j.gather ? r0 + 128 : j.rows))
        {
            uint2 hi, lo;
            split2(v[i].x * inv, v[i].y * inv, hi.x, lo.x);
            split2(v[i].z * inv, v[i].w * inv, hi.y, lo.y);
            __half *line = j.out + r * j.pitch + (c >> 6) * 128 + (c & 63);
            *reinterpret_cast<uint2 *>(line)      = hi;
            *reinterpret_cast<uint2 *>(line + 64) = lo;
        }
    }
}

__global__ void __launch_bounds__(kTileThreads) split16_tiles_kernel(const __grid_constant__ EncodeJob a, const __grid_constant__ EncodeJob b, const ZeroRows z)
{
    __shared__ float box[16];
    __shared__ float tile[64][129];
    let_next_in();
    after_previous();
    int block = blockIdx.x;
    if (block < a.blocks)
        return split16_tile(a, block, box, tile);
    block -= a.blocks;
    if (block < b.blocks)
        return split16_tile(b, block, box, tile);
    block -= b.blocks;
    const int lane = threadIdx.x & 31;
    constexpr int kWarps = kTileThreads / 32;
    for (int row = block * kWarps + (threadIdx.x >> 5); row < z.rows; row += z.blocks * kWarps)
    {
        if (z.pos_of[row] >= 0)
            continue;
        if (z.words && lane == 0)
            z.words[row] = 0.f;
        if (z.matrix)
            for (int c = lane; c < z.cols; c += 32)
                z.matrix[static_cast<int64_t>(row) * z.cols + c] = 0.f;
    }
}
}  // namespace

EncodeJob encode_job(const float *src, int64_t ld, int transposed, int rows, int cols, const int *gather, const int *count, const Split16 &out, float *scale)
{
    EncodeJob j;
    j.src = src, j.ld = ld, j.transposed = transposed, j.rows = rows, j.cols = cols, j.gather = gather, j.count = count;
    j.out = const_cast<__half *>(out.data), j.pitch = out.pitch, j.scale = scale;
    j.cols_pad = out.cols_pad;
    j.blocks_c = (out.cols_pad + 127) / 128;
    j.blocks   = static_cast<int64_t>((rows + 127) / 128) * j.blocks_c;
    return j;
}

int split16_encode(const EncodeJob &a, const EncodeJob &b, const ZeroRows &z, cudaStream_t stream)
{
    const int64_t blocks = a.blocks + b.blocks + z.blocks;
    if (blocks > 0x7fffffff)
    {
        set_last_error("split: %lld tiles are too many", (long long)blocks);
        return kTooLarge;
    }
    return launch_after(split16_tiles_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kTileThreads), 0, stream, a, b, z);
}

}  // namespace s16
}  // namespace odl
