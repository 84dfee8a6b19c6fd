// fp4_gemm.cu - products of microscaled 4-bit operands: tensor maps, choice of tile, launch (loop: fp4_gemm.cuh).
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/hcomm_fp4.h"
#include "../core/log.h"
#include "../core/per_device.h"
#include "fp4_gemm.cuh"
#include "fp4_gemm_pair.cuh"
#include "gemm_api.h"

namespace {
using namespace hcfp4;

// Set when a bounded wait expired; part of the device image, so no call has to allocate it.
__device__ uint32_t g_error;

template <bool GLU>
__global__ void __launch_bounds__(kGemmThreads, 1) Fp4GemmKernel(const __grid_constant__ Maps maps, const __grid_constant__ Shape shape)
{
    GemmLoop<GLU>(&maps, shape);
}

template <bool GLU>
__global__ void __launch_bounds__(kGemmThreads, 1) Fp4GemmPairKernel(const __grid_constant__ Maps maps, const __grid_constant__ Shape shape)
{
    GemmLoopPair<GLU>(&maps, shape);
}

// pairs: clusters of two CTAs of the pair loop that fit at once; clusters: of the other loop's, of 2, 4 and 8 CTAs
struct Device { int sms, pairs, clusters[3]; uint32_t *error; };
template <typename Kernel> bool AllowShared(Kernel *kernel)
{
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) == cudaSuccess) return true;
    cudaGetLastError();
    return false;
}
cudaLaunchConfig_t LaunchConfig(cudaLaunchAttribute *at, int ctas, int clusterCtas, int smem, void *stream)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, 1, 1);
    cfg.blockDim = dim3(kGemmThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = clusterCtas; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = clusterCtas > 1 ? 2 : 1;
    return cfg;
}
bool CurrentDevice(Device *d)
{
    static hc::PerDevice<Device> devices;
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); return false; }
    bool good = true;
    *d = devices.Get(dev, [&](Device *v) {
        good = cudaDeviceGetAttribute(&v->sms, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && cudaGetSymbolAddress((void **)&v->error, g_error) == cudaSuccess &&
               AllowShared(Fp4GemmKernel<false>) && AllowShared(Fp4GemmKernel<true>) && AllowShared(Fp4GemmPairKernel<false>) && AllowShared(Fp4GemmPairKernel<true>);
        cudaLaunchAttribute at[2];
        const cudaLaunchConfig_t cfg = LaunchConfig(at, v->sms / 2 * 2, 2, PairSmemBytes(kMaxExperts), nullptr);
        good = good && cudaOccupancyMaxActiveClusters(&v->pairs, Fp4GemmPairKernel<true>, &cfg) == cudaSuccess;
        for (int i = 0; i < 3 && good; ++i) {
            const cudaLaunchConfig_t c = LaunchConfig(at, v->sms / (2 << i) * (2 << i), 2 << i, 227 * 1024, nullptr);
            good = cudaOccupancyMaxActiveClusters(&v->clusters[i], Fp4GemmKernel<true>, &c) == cudaSuccess;
        }
        if (!good) cudaGetLastError();
        return good;
    });
    return good;
}

struct Operand { const void *values, *scales; };
constexpr int kMost = INT32_MAX - 256;         // rows, columns and depth: rounded up to a tile or a stage still a 32-bit number

// boxRows rows x 256 columns of values; `matrices` of them one behind the other.
HcclResult ValueMap(CUtensorMap *m, const void *values, int64_t matrices, int64_t rows, int64_t K, int boxRows)
{
    const uint64_t dims[3] = {(uint64_t)K / 2, (uint64_t)rows, (uint64_t)matrices}, pitches[2] = {(uint64_t)K / 2, (uint64_t)(rows * (K / 2))};
    const uint32_t box[3] = {128, (uint32_t)boxRows, 1};
    return hc::EncodeTensorMap(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, values, 3, dims, pitches, box, true);
}
// Two tiles of scales that follow one another along K.
HcclResult ScaleMap(CUtensorMap *m, const void *scales, int64_t tiles)
{
    const uint64_t dims[2] = {kTileBytes / 4, (uint64_t)tiles}, pitches[1] = {kTileBytes};
    const uint32_t box[2] = {kTileBytes / 4, 2};
    return hc::EncodeTensorMap(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, scales, 2, dims, pitches, box, false);
}

template <typename Kernel> cudaError_t Launch(Kernel *kernel, int ctas, int clusterCtas, int smem, void *stream, const Maps &maps, const Shape &shape)
{
    cudaLaunchAttribute at[2];
    const cudaLaunchConfig_t cfg = LaunchConfig(at, ctas, clusterCtas, smem, stream);
    return cudaLaunchKernelEx(&cfg, kernel, maps, shape);
}

// Whether a product goes by pairs of CTAs (tiles of 256 rows x 256 columns, or 128 of a gated product) or by single CTAs (up to 128 rows x
// 128 columns): the less of two estimates, in us.
//   * tiles come in waves of what fits at once; of grouped rows, which are known on the device only, every expert is taken to have the
//     average of all rows that the operand has room for, and a tile that it fills half: where a step fills little of a long buffer, as an expert layer made for more
//     tokens does, the rule plans for rows that are not there (a layer of 32 experts, 7168 and 2048, on 64 tokens: made for 64 185 us, for 4096 213);
//   * single: a stage of 256 columns of K takes 0.19 us to issue, or its bytes at 112 a ns; a tile at least 0.4 us and 1.6 a 128 rows, in which
//     the tile in front is stored;
//   * pair: 0.34 us a stage, and 1.5 in which nothing overlaps the reading of the tile's accumulator;
//   * nothing is faster than its bytes at 6.5 TB/s, pairs at 4.6: they have less of B under way.
// us, single / pair: 500 x 3584 x 8192 13.7 / 15.1, 777 x 3584 x 8192 21.5 / 16.0, 256 x 8192 x 28672 34.8 / 41.1, 1024 x 1024 x 4096 9.0 / 10.0,
// 2048 x 4096 x 1024 11.5 / 10.5, 4096 x 4096 x 4096 36 / 29, 8192 x 28672 x 8192 862 / 642; 32 experts, 7168 and 2048, gated and down: 64 rows
// 67 / 81 and 37 / 54, 3000 94 / 111 and 55 / 66, 5003 106 / 123 and 69 / 76, 8000 138 / 137 and 91 / 88, 16000 234 / 215 and 153 / 142.
//
// Single CTAs share a tile along K, as clusters of 2, 4 or 8, where the clusters of all tiles that there can be fit at once (by expert: of any split of the operand's
// rows, so of a few rows only) and that is estimated to be faster: exchanging sums takes 0.9 us, 0.2 a CTA and 12 ns a row.  us, alone / 2 / 4 / 8 of them: 1 x 4096 x 14336 15.0 / 10.6 / 9.5 / -,
// 16 x 8192 x 28672 28.1 / 24.7 / - / -, 128 x 1024 x 4096 8.4 / 8.5 / 7.0 / 7.1, 16 x 8192 x 3584 6.8 / 7.6 / - / -, 16 x 4096 x 1024 3.8 / 4.5 / 5.2 / -.
struct Costs { double single, pair; int split; };
Costs Estimate(int64_t M, int64_t N, int64_t K, int experts, bool glu, int sms, int pairs, const int (&clusters)[3])
{
    const double stages = (double)((K + kStageCols - 1) / kStageCols), matrices = experts > 0 ? std::min<double>((double)M, experts) : 1, rows = M / matrices;
    auto tiles = [&](double tall, double wide) {
        const double down = experts > 0 ? std::max(1.0, rows / tall + 0.5) : std::ceil(rows / tall);
        return matrices * down * std::ceil(N / wide);
    };
    const double hbm = (17.0 / 32 * (M * K + matrices * (glu ? 2 : 1) * N * K) + 2.0 * M * N) / 6.5e6;
    const double used = std::min(rows, 128.0), stage = std::max(0.19, ((glu ? 2 : 1) * 17408 + 1024 + 128 * used) / 112e3);
    const double pair = std::ceil(tiles(256, glu ? 128 : 256) / std::max(pairs, 1)) * (stages * 0.34 + 1.5);
    Costs c = {std::ceil(tiles(128, 128) / sms) * std::max(stages * stage, 0.4 + 1.6 * used / 128), pair, 1};
    c.single = 3.0 + std::max(c.single, hbm) + 0.5;
    c.pair = 3.0 + std::max(c.pair, 1.4 * hbm) + 0.5;
    const double most = (double)(experts > 0 ? GroupedTileRows(M, experts) : (M + 127) / 128) * std::ceil(N / 128.0);
    for (int i = 0; i < 3; ++i) {
        const int split = 2 << i;
        if (most > clusters[i] || stages < split) continue;
        const double us = 3.0 + std::max(std::ceil(stages / split) * stage, hbm) + 0.9 + 0.2 * split + 0.012 * used;
        if (us < c.single) { c.single = us; c.split = split; }
    }
    return c;
}

// b[1] is the up projection of a gated product, else NULL.
HcclResult Gemm(const char *what, Operand a, const Operand (&b)[2], bool glu, void *out, int M, int N, int K, int64_t ldOut, const int32_t *offsets, int experts, void *stream)
{
    if (M < 0 || N < 0 || K < 0 || M > kMost || N > kMost || K > kMost || K % kBlock || ldOut < N || experts < 0 || experts > kMaxExperts || (experts > 0) != (offsets != nullptr)) {
        RPT_ERR("EI0003", "%s: M %d, N %d, K %d (a multiple of %d; at most %d each), rows of the result %lld apart, %d experts (at most %d, with offsets)", what, M, N, K, kBlock, kMost,
                (long long)ldOut, experts, kMaxExperts);
        return HCCL_E_PARA;
    }
    if (M == 0 || N == 0) return HCCL_SUCCESS;
    if (!out) return HCCL_E_PTR;
    if ((uintptr_t)out & 1) { RPT_ERR("EI0003", "%s: misaligned result", what); return HCCL_E_PARA; }
    if (K == 0) { RPT_ERR("EI0003", "%s: no columns to multiply", what); return HCCL_E_PARA; }
    const Operand all[3] = {a, b[0], glu ? b[1] : b[0]};
    for (const Operand &o : all) {
        if (!o.values || !o.scales) return HCCL_E_PTR;
        if (((uintptr_t)o.values & 15) || ((uintptr_t)o.scales & 15)) { RPT_ERR("EI0003", "%s: operands must be 16-byte aligned", what); return HCCL_E_PARA; }
    }
    Device dev;
    if (!CurrentDevice(&dev)) { HCCL_ERROR("%s: the current device cannot run it", what); return HCCL_E_RUNTIME; }
    Shape g = {};
    g.M = M; g.N = N; g.K = K;
    g.experts = experts; g.offsets = offsets;
    g.tileCols = (K + kTileCols - 1) / kTileCols;
    g.tileRowsB = (N + kTileRows - 1) / kTileRows;
    g.ldOut = ldOut; g.out = (__nv_bfloat16 *)out;
    g.error = dev.error;
    const int matrices = std::max(experts, 1);
    const int64_t rowTiles = experts > 0 ? GroupedTileRows(M, experts) : (M + 127) / 128;
    const Costs costs = Estimate(M, N, K, experts, glu, dev.sms, dev.pairs, dev.clusters);
    const bool pairs = dev.pairs > 0 && M > 128 && costs.pair < costs.single;
    g.tilesN = pairs && !glu ? (N + 255) / 256 : (N + 127) / 128;
    g.group = pairs ? 8 : 16;
    if (rowTiles * g.tilesN > INT32_MAX / 2 || (int64_t)matrices * g.tileRowsB * g.tileCols > INT32_MAX / 2 || rowTiles * g.tileCols > INT32_MAX / 2) {
        RPT_ERR("EI0003", "%s: %d x %d x %d is more than a launch can count", what, M, N, K);
        return HCCL_E_PARA;
    }
    // A SM's loads take some 55 bytes a cycle, rows outside the matrix as long as others: 16 x 18944 x 8192 with boxes of 128 rows
    // 20.6 us, of 16 16.4.  Rows of an expert, which are known on the device only, come in boxes of 32 where there are few of them.
    g.boxRows = 128;
    if (!pairs) {
        const int likely = experts > 0 ? M / experts : M;
        while (g.boxRows > 8 && g.boxRows / 2 >= likely) g.boxRows /= 2;
        if (experts > 0) g.boxRows = likely >= 96 ? 128 : 32;
    }
    g.aSlot = Config<128>::ASlot(g.boxRows, experts > 0);
    g.stages = glu ? Config<256>::Stages(g.aSlot, experts) : Config<128>::Stages(g.aSlot, experts);
    Maps maps;
    CHK_RET(ValueMap(&maps.a, a.values, 1, M, K, g.boxRows));
    CHK_RET(ScaleMap(&maps.sa, a.scales, rowTiles * g.tileCols));
    for (int h = 0; h < 2; ++h) {
        if (h == 1 && !glu) { maps.b[1] = maps.b[0]; maps.sb[1] = maps.sb[0]; break; }
        CHK_RET(ValueMap(&maps.b[h], b[h].values, matrices, N, K, 128));
        CHK_RET(ScaleMap(&maps.sb[h], b[h].scales, (int64_t)matrices * g.tileRowsB * g.tileCols));
    }
    g.split = pairs ? 1 : costs.split;
    const int ctas = g.split > 1 ? (int)(rowTiles * g.tilesN) * g.split : (int)std::min<int64_t>(dev.sms, rowTiles * g.tilesN);
    cudaError_t e;
    if (pairs) {
        const int both = 2 * (int)std::min<int64_t>(dev.pairs, rowTiles * g.tilesN);
        e = glu ? Launch(Fp4GemmPairKernel<true>, both, 2, PairSmemBytes(experts), stream, maps, g) : Launch(Fp4GemmPairKernel<false>, both, 2, PairSmemBytes(experts), stream, maps, g);
    } else {
        e = glu ? Launch(Fp4GemmKernel<true>, ctas, g.split, Config<256>::SmemBytes(g.aSlot, g.stages, experts), stream, maps, g)
                : Launch(Fp4GemmKernel<false>, ctas, g.split, Config<128>::SmemBytes(g.aSlot, g.stages, experts), stream, maps, g);
    }
    if (e != cudaSuccess) {
        cudaGetLastError();
        HCCL_ERROR("%s launch failed: %s", what, cudaGetErrorString(e));
        return HCCL_E_RUNTIME;
    }
    return HCCL_SUCCESS;
}

}  // namespace

extern "C" int HcommFp4Gemm(const void *aValues, const void *aScales, const void *bValues, const void *bScales, void *out, int M, int N, int K, int64_t ldOut,
                            const int32_t *offsets, int experts, void *stream)
{
    return Gemm("HcommFp4Gemm", {aValues, aScales}, {{bValues, bScales}, {nullptr, nullptr}}, false, out, M, N, K, ldOut, offsets, experts, stream);
}
extern "C" int HcommFp4GemmSwiglu(const void *aValues, const void *aScales, const void *gValues, const void *gScales, const void *uValues, const void *uScales, void *out,
                                  int M, int N, int K, int64_t ldOut, const int32_t *offsets, int experts, void *stream)
{
    return Gemm("HcommFp4GemmSwiglu", {aValues, aScales}, {{gValues, gScales}, {uValues, uScales}}, true, out, M, N, K, ldOut, offsets, experts, stream);
}
extern "C" int HcommFp4TakeError(void)
{
    uint32_t v = 0;
    const uint32_t zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_error, sizeof(v)) != cudaSuccess) { cudaGetLastError(); return -1; }
    if (v) cudaMemcpyToSymbol(g_error, &zero, sizeof(zero));
    return (int)v;
}
// What the rule makes of a product on a device that holds so many SMs, pairs of CTAs and clusters of 2, 4 and 8 CTAs at once: us by single
// CTAs and by pairs.  Returns how many single CTAs share a tile.
extern "C" int HcommToolFp4Estimate(int M, int N, int K, int experts, int gated, int sms, int pairs, const int *clusters, double *us)
{
    const int held[3] = {clusters[0], clusters[1], clusters[2]};
    const Costs c = Estimate(M, N, K, experts, gated != 0, sms, pairs, held);
    us[0] = c.single; us[1] = c.pair;
    return c.split;
}
