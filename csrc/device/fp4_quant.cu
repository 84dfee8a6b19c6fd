// fp4_quant.cu - quantisation to microscaled 4-bit values and back (format: include/hcomm_fp4.h).
//
// For each block of 32 values x of a row, with m = max |x|:   e = max(floor(log2 m) - 2, -127),   q = round_e2m1(x / 2^e).
// Division by a power of two is exact, the conversion instruction rounds to the nearest (even) and saturates at 6, so every
// result is that of the definition, bit for bit.  The maximum is taken over the magnitudes' bits: integers order like the
// floats they are, infinities and NaN above everything, which is how such a block is found.
//
// Memory is what bounds it: 2 bytes read and 17/32 written a value (bf16).  Sixteen lanes take 128 columns of a row - 16 bytes a
// lane, four lanes a block - and end with one 32-bit word of scales, so neither shared memory nor a second pass is needed.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/hcomm_fp4.h"
#include "../core/log.h"
#include "fp4.cuh"
#include "sm100_ptx.cuh"

namespace {
using namespace hcfp4;

constexpr int kThreads = 256;
constexpr int kHalfWarps = kThreads / 16;

struct Rows {
    int64_t rows, cols;                     // of one matrix
    int64_t batch;
    int tileCols;                           // ceil(cols / 128)
    const int32_t *offsets;                 // grouped rows, else NULL
    int experts;
};

// Walks the chunks (row, 128 columns) of a half warp: chunk c, c + step, c + 2 step ...
struct Walk {
    int64_t row;
    int col;
    int64_t rowStep;
    int colStep, tileCols;
    __device__ Walk(int64_t first, int64_t step, int cols) : tileCols(cols)
    {
        row = first / cols; col = (int)(first % cols);
        rowStep = step / cols; colStep = (int)(step % cols);
    }
    __device__ void Next()
    {
        row += rowStep; col += colStep;
        if (col >= tileCols) { col -= tileCols; ++row; }
    }
};

// The rows that a block works on: all of the batch's, or those that the offsets cover.
struct Range { int64_t first, last; };
__device__ __forceinline__ Range RowsOf(const Rows &r, int *start, int *tile)
{
    if (!r.offsets) return {0, r.batch * r.rows};
    if (threadIdx.x < 32) BuildGroups(r.offsets, r.experts, (int)r.rows, start, tile);
    __syncthreads();
    return {start[0], start[r.experts]};
}
// Address of a row's bytes in tile column 0.
__device__ __forceinline__ int64_t ScaleAt(const Rows &r, const int *start, const int *tile, int64_t row)
{
    int64_t tileRow;
    uint32_t in;
    if (r.offsets) {
        const int e = GroupOf(start, r.experts, (int)row), local = (int)row - start[e];
        tileRow = tile[e] + local / kTileRows;
        in = local % kTileRows;
    } else if (r.batch > 1) {
        const int64_t b = row / r.rows, local = row - b * r.rows;
        tileRow = b * ((r.rows + kTileRows - 1) / kTileRows) + local / kTileRows;
        in = (uint32_t)(local % kTileRows);
    } else {
        tileRow = row / kTileRows;
        in = (uint32_t)(row % kTileRows);
    }
    return tileRow * r.tileCols * kTileBytes + ScaleByte(in);
}

template <typename T> struct Eight {};      // eight consecutive values as they lie in memory
template <> struct Eight<float> { uint4 a, b; };
template <> struct Eight<__half> { uint4 a; };
template <> struct Eight<__nv_bfloat16> { uint4 a; };
template <> struct Eight<__nv_fp8_e4m3> { uint2 a; };

__device__ __forceinline__ float ToFloat(float v) { return v; }
__device__ __forceinline__ float ToFloat(__half v) { return __half2float(v); }
__device__ __forceinline__ float ToFloat(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float ToFloat(__nv_fp8_e4m3 v) { return (float)v; }

// aligned: every row starts on a boundary of eight values' size (16 bytes for fp32), else value by value
template <typename T> __device__ __forceinline__ void Load(Eight<T> *v, const T *p, bool aligned)
{
    if (aligned) {
        if constexpr (sizeof(T) == 1) *(uint2 *)v = __ldg((const uint2 *)p);
        else {
            ((uint4 *)v)[0] = __ldg((const uint4 *)p);
            if constexpr (sizeof(T) == 4) ((uint4 *)v)[1] = __ldg((const uint4 *)p + 1);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) ((T *)v)[i] = p[i];
    }
}

// {even column in the low half of byte i, odd in the high half} for pairs i = 0 .. 3
__device__ __forceinline__ uint32_t PackE2m1(const float (&v)[8])
{
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

struct Source { const void *x; const float *xScales; int64_t batchPitch, rowPitch, scalePitch; bool aligned; };

template <typename T>
__global__ void __launch_bounds__(kThreads) QuantizeKernel(Rows r, Source s, uint8_t *values, uint8_t *scales)
{
    __shared__ int start[kMaxExperts + 1], tile[kMaxExperts + 1];
    sm100::GridDependencyWait();
    sm100::GridDependentsLaunch();
    const Range range = RowsOf(r, start, tile);
    const int lane = threadIdx.x & 15;
    const int64_t half = (int64_t)blockIdx.x * kHalfWarps + (threadIdx.x >> 4), halves = (int64_t)gridDim.x * kHalfWarps;
    constexpr int U = sizeof(T) == 4 ? 2 : 4;           // loads of that many chunks are under way at once
    Walk w(half, halves, r.tileCols);
    w.row += range.first;
    // both halves of a warp go round together: the shuffles below are the whole warp's
    for (int64_t c = half & ~(int64_t)1; c < (range.last - range.first) * r.tileCols; c += halves * U) {
        Eight<T> in[U];
        float mul[U];
        int64_t row[U];
        int col[U];
        bool real[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            row[u] = w.row; col[u] = w.col * kTileCols + lane * 8;
            real[u] = w.row < range.last && col[u] < r.cols;
            in[u] = Eight<T>();
            mul[u] = 1.f;
            if (real[u]) {
                int64_t at = row[u] * s.rowPitch;
                if (r.batch > 1) { const int64_t b = row[u] / r.rows; at = b * s.batchPitch + (row[u] - b * r.rows) * s.rowPitch; }
                Load(&in[u], (const T *)s.x + at + col[u], s.aligned);
                if constexpr (sizeof(T) == 1) {
                    int64_t sat = row[u] * s.scalePitch;        // of a batch: pitches count rows through all matrices
                    mul[u] = __ldg(s.xScales + sat + w.col);
                }
            }
            w.Next();
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float v[8];
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[i] = ToFloat(((const T *)&in[u])[i]);
                if constexpr (sizeof(T) == 1) v[i] = __fmul_rn(v[i], mul[u]);
                top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
            }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // the exponent field less two, or 255 where the block holds something that is no number
            const uint32_t scale = top >= 0x7f800000u ? 255u : (uint32_t)max((int)(top >> 23) - 2, 0);
            const float inverse = __uint_as_float((scale == 255u ? 127u : 254u - scale) << 23);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= inverse;
            if (real[u]) *(uint32_t *)(values + (row[u] * r.cols + col[u]) / 2) = PackE2m1(v);
            uint32_t word = (col[u] < r.cols ? scale : 0u) << (lane >> 2) * 8;
            word |= __shfl_xor_sync(0xffffffffu, word, 4);
            word |= __shfl_xor_sync(0xffffffffu, word, 8);
            if (lane == 0 && row[u] < range.last) *(uint32_t *)(scales + ScaleAt(r, start, tile, row[u]) + (int64_t)(col[u] / kTileCols) * kTileBytes) = word;
        }
    }
}

__device__ __forceinline__ float ScaleOf(uint32_t byte)
{
    return byte == 255u ? __uint_as_float(0x7fc00000u) : byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}
__device__ __forceinline__ void UnpackE2m1(uint32_t word, float (&v)[8])
{
    uint32_t h[4];
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(word));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*(const __half2 *)&h[i]);
        v[2 * i] = f.x; v[2 * i + 1] = f.y;
    }
}
template <typename T> __device__ __forceinline__ T FromFloat(float v);
template <> __device__ __forceinline__ float FromFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ __half FromFloat<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 FromFloat<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T>
__global__ void __launch_bounds__(kThreads) DequantizeKernel(Rows r, const uint8_t *values, const uint8_t *scales, T *out)
{
    __shared__ int start[kMaxExperts + 1], tile[kMaxExperts + 1];
    sm100::GridDependencyWait();
    sm100::GridDependentsLaunch();
    const Range range = RowsOf(r, start, tile);
    const int lane = threadIdx.x & 15;
    const int64_t half = (int64_t)blockIdx.x * kHalfWarps + (threadIdx.x >> 4), halves = (int64_t)gridDim.x * kHalfWarps;
    constexpr int U = 4;
    Walk w(half, halves, r.tileCols);
    w.row += range.first;
    for (int64_t c = half; c < (range.last - range.first) * r.tileCols; c += halves * U) {
        uint32_t word[U], byte[U];
        int64_t at[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int col = w.col * kTileCols + lane * 8;
            at[u] = w.row < range.last && col < r.cols ? w.row * r.cols + col : -1;
            if (at[u] >= 0) {
                word[u] = *(const uint32_t *)(values + at[u] / 2);
                byte[u] = scales[ScaleAt(r, start, tile, w.row) + (int64_t)w.col * kTileBytes + (lane >> 2)];
            }
            w.Next();
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (at[u] < 0) continue;
            float v[8];
            UnpackE2m1(word[u], v);
            const float scale = ScaleOf(byte[u]);
            __align__(16) T o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = FromFloat<T>(v[i] * scale);
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) ((uint4 *)(out + at[u]))[i] = ((const uint4 *)o)[i];
        }
    }
}

HcclResult CheckRows(const char *what, int64_t batch, int64_t rows, int64_t cols, const int32_t *offsets, int experts)
{
    if (batch < 0 || rows < 0 || cols < 0 || cols % kBlock || rows > INT32_MAX || cols > INT32_MAX || (batch && rows > INT64_MAX / 4096 / batch)) {
        RPT_ERR("EI0003", "%s: %lld x %lld x %lld, columns must be a multiple of 32", what, (long long)batch, (long long)rows, (long long)cols);
        return HCCL_E_PARA;
    }
    if (experts < 0 || experts > kMaxExperts || (experts > 0) != (offsets != nullptr) || (experts > 0 && batch != 1)) {
        RPT_ERR("EI0003", "%s: grouped rows need offsets, 1 to %d experts and a single matrix (experts %d)", what, kMaxExperts, experts);
        return HCCL_E_PARA;
    }
    return HCCL_SUCCESS;
}

// Programmatic launch: set-up overlaps the end of the kernel in front, which the kernel waits for before it touches memory.
template <typename... Params, typename... Args> HcclResult Launch(const char *what, void (*kernel)(Params...), int64_t chunks, void *stream, Args... args)
{
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    cudaLaunchConfig_t cfg = {};
    // small operands: a chunk to each half warp, so that all loads are under way at once; large ones: eight blocks a SM
    cfg.gridDim = dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>((chunks + kHalfWarps - 1) / kHalfWarps, (int64_t)sms * 8)), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at; cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e != cudaSuccess) {
        cudaGetLastError();
        HCCL_ERROR("%s launch failed: %s", what, cudaGetErrorString(e));
        return HCCL_E_RUNTIME;
    }
    return HCCL_SUCCESS;
}
template <typename T>
HcclResult LaunchQuantize(const Rows &r, const Source &s, void *values, void *scales, void *stream)
{
    return Launch("HcommFp4Quantize", QuantizeKernel<T>, r.batch * r.rows * r.tileCols, stream, r, s, (uint8_t *)values, (uint8_t *)scales);
}
template <typename T> HcclResult LaunchDequantize(const Rows &r, const void *values, const void *scales, void *out, void *stream)
{
    return Launch("HcommFp4Dequantize", DequantizeKernel<T>, r.batch * r.rows * r.tileCols, stream, r, (const uint8_t *)values, (const uint8_t *)scales, (T *)out);
}

}  // namespace

extern "C" uint64_t HcommFp4ScaleBytes(int64_t batch, int64_t rows, int64_t cols, int experts)
{
    if (batch < 0 || rows < 0 || cols < 0 || experts < 0) return 0;
    const int64_t tileRows = experts > 0 ? GroupedTileRows(rows, experts) : batch * ((rows + kTileRows - 1) / kTileRows);
    return (uint64_t)tileRows * ((cols + kTileCols - 1) / kTileCols) * kTileBytes;
}

extern "C" int HcommFp4Quantize(const void *x, int dataType, const float *xScales, int64_t batch, int64_t rows, int64_t cols, int64_t batchPitch, int64_t rowPitch,
                                int64_t scalePitch, const int32_t *offsets, int experts, void *values, void *scales, void *stream)
{
    CHK_RET(CheckRows("HcommFp4Quantize", batch, rows, cols, offsets, experts));
    const bool fp8 = dataType == HCCL_DATA_TYPE_FP8E4M3;
    if (batch * rows * cols == 0) return HCCL_SUCCESS;
    if (!x || !values || !scales || (fp8 && !xScales)) return HCCL_E_PTR;
    if (rowPitch < cols || batchPitch < 0 || ((uintptr_t)values & 15) || ((uintptr_t)scales & 15) || (fp8 && (cols % 128 || scalePitch < cols / 128 || batch != 1))) {
        RPT_ERR("EI0003", "HcommFp4Quantize: row pitch %lld of %lld columns, scale pitch %lld; outputs must be 16-byte aligned, fp8 rows a multiple of 128 wide and one matrix",
                (long long)rowPitch, (long long)cols, (long long)scalePitch);
        return HCCL_E_PARA;
    }
    const int64_t wide = dataType == HCCL_DATA_TYPE_FP32 ? 4 : 8;           // values in the widest load
    const uintptr_t boundary = fp8 ? 8 : 16;
    const Rows r{rows, cols, batch, (int)((cols + kTileCols - 1) / kTileCols), offsets, experts};
    const Source s{x, xScales, batchPitch, rowPitch, scalePitch, ((uintptr_t)x % boundary) == 0 && rowPitch % wide == 0 && (batch == 1 || batchPitch % wide == 0)};
    switch (dataType) {
        case HCCL_DATA_TYPE_FP32: return LaunchQuantize<float>(r, s, values, scales, stream);
        case HCCL_DATA_TYPE_FP16: return LaunchQuantize<__half>(r, s, values, scales, stream);
        case HCCL_DATA_TYPE_BFP16: return LaunchQuantize<__nv_bfloat16>(r, s, values, scales, stream);
        case HCCL_DATA_TYPE_FP8E4M3: return LaunchQuantize<__nv_fp8_e4m3>(r, s, values, scales, stream);
        default:
            RPT_ERR("EI0003", "HcommFp4Quantize: data type %d is not FP32, FP16, BFP16 or FP8E4M3", dataType);
            return HCCL_E_PARA;
    }
}

extern "C" int HcommFp4Dequantize(const void *values, const void *scales, int64_t batch, int64_t rows, int64_t cols, const int32_t *offsets, int experts, void *out,
                                  int dataType, void *stream)
{
    CHK_RET(CheckRows("HcommFp4Dequantize", batch, rows, cols, offsets, experts));
    if (batch * rows * cols == 0) return HCCL_SUCCESS;
    if (!values || !scales || !out) return HCCL_E_PTR;
    if (((uintptr_t)values & 15) || ((uintptr_t)scales & 15) || ((uintptr_t)out & 15)) {
        RPT_ERR("EI0003", "HcommFp4Dequantize: buffers must be 16-byte aligned");
        return HCCL_E_PARA;
    }
    const Rows r{rows, cols, batch, (int)((cols + kTileCols - 1) / kTileCols), offsets, experts};
    switch (dataType) {
        case HCCL_DATA_TYPE_FP32: return LaunchDequantize<float>(r, values, scales, out, stream);
        case HCCL_DATA_TYPE_FP16: return LaunchDequantize<__half>(r, values, scales, out, stream);
        case HCCL_DATA_TYPE_BFP16: return LaunchDequantize<__nv_bfloat16>(r, values, scales, out, stream);
        default:
            RPT_ERR("EI0003", "HcommFp4Dequantize: data type %d is not FP32, FP16 or BFP16", dataType);
            return HCCL_E_PARA;
    }
}
