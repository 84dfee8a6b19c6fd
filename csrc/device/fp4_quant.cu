// fp4_quant.cu - quantisation to microscaled 4-bit values and back (format: include/hcomm_fp4.h).
//
// For each block of 32 values x of a row, with m = max |x|:   e = max(floor(log2 m) - 2, -127),   q = round_e2m1(x / 2^e).
// Division by a power of two is exact, the conversion instruction rounds to the nearest (even) and saturates at 6, so every
// result is that of the definition, bit for bit.  The maximum is taken over the magnitudes' bits: integers order like the
// floats they are, infinities and NaN above everything, which is how such a block is found.
//
// Memory is what bounds it: 2 bytes read and 17/32 written a value (bf16).  A lane takes 16 values (32 of fp8) of a row, two (one) a block
// of 32, and stays in its columns from row to row, so that neither shared memory nor a second pass nor address arithmetic is in the way.
// 8192 x 28672 bf16: 99 us, 6.0 TB/s (eight values a lane and addresses by division: 281 us); back to bf16 101.
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
constexpr int64_t kMostRows = INT32_MAX - (1 << 20);       // a step behind the last row is still a 32-bit number

struct Rows {
    int64_t rows, cols;                     // of one matrix
    int64_t batch;
    int tileCols;                           // ceil(cols / 128)
    int across, most;                       // rows that all teams of lanes take at a time; and, without groups, how often
    const int32_t *offsets;                 // grouped rows, else NULL
    int experts;
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

// A row's number, unsigned: all teams of a warp go round as often as the busiest, and one of the few that are left over begins behind the last row
// and goes on by as much again and some steps, which is below 2^32 (2 kMostRows and 5 x 28416), where a signed number came back as one of a
// row in front of the last (1.08 G rows of 288 columns).  A step that is 0 for those teams takes a register too many: 8192 x 28672 108 us for 100.
using RowNumber = uint32_t;

// What a team of lanes works on: 128 columns of some rows.  Of grouped rows it takes `most` in a row, so that the expert hardly ever
// changes from one to the next (32768 x 2048 bf16 rows of 256 experts: 49 us with rows a grid apart, 38 so); of others rows a grid apart, which
// memory takes better (8192 x 28672 fp32: 156 us, in a row 176).
struct Walk {
    RowNumber row, end;
    int step, most, col;
    int segment;
    RowNumber segmentRow, segmentEnd;   // of a batch: its matrix; of grouped rows: the expert
    int64_t tileBase;                   // bytes to the segment's tiles of this column
    __device__ Walk(int lanes, const Range &range, const Rows &r, const int *start, const int *tile)
    {
        const int mine = (blockIdx.x * kThreads + threadIdx.x) / lanes, lane = mine / r.tileCols;         // lane: of those that take rows
        const int rows = (int)(range.last - range.first);
        col = mine - lane * r.tileCols;
        most = r.offsets ? (rows + r.across - 1) / r.across : r.most;
        step = r.offsets ? 1 : r.across;
        const int64_t first = lane >= r.across ? rows : r.offsets ? (int64_t)lane * most : lane;         // the few teams that are left over have nothing to do
        row = (RowNumber)(range.first + min(first, (int64_t)rows)); end = r.offsets ? (RowNumber)min((int64_t)row + most, range.last) : (RowNumber)range.last;
        segment = 0; segmentRow = 0; segmentEnd = end;
        tileBase = (int64_t)col * kTileBytes;
        if (row < end && (r.offsets || r.batch > 1)) {
            segment = r.offsets ? GroupOf(start, r.experts, row) : (int)(row / r.rows);
            Enter(r, start, tile);
        }
    }
    __device__ void Enter(const Rows &r, const int *start, const int *tile)
    {
        int64_t tileRow;
        if (r.offsets) { segmentRow = start[segment]; segmentEnd = start[segment + 1]; tileRow = tile[segment]; }
        else { segmentRow = segment * (RowNumber)r.rows; segmentEnd = segmentRow + (RowNumber)r.rows; tileRow = segment * ((r.rows + kTileRows - 1) / kTileRows); }
        tileBase = (tileRow * r.tileCols + col) * kTileBytes;
    }
    __device__ void Next(const Rows &r, const int *start, const int *tile)
    {
        row += step;
        while (row < end && row >= segmentEnd) {
            segment = r.offsets ? segment + 1 : (int)(row / r.rows);
            Enter(r, start, tile);
        }
    }
    __device__ int64_t Scales(const Rows &r) const
    {
        const uint32_t local = row - segmentRow;
        return tileBase + (int64_t)(local / kTileRows) * (r.tileCols * kTileBytes) + ScaleByte(local % kTileRows);
    }
};

// Sixteen consecutive values as they lie in memory: 16, 32 or 64 bytes.
template <typename T> struct __align__(16) Sixteen { uint4 q[sizeof(T)]; };
// aligned: every row starts on a 16-byte boundary, else value by value
template <typename T> __device__ __forceinline__ void Load(Sixteen<T> *v, const T *p, bool aligned)
{
    if (aligned) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T); ++i) v->q[i] = ((const uint4 *)p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) ((T *)v)[i] = p[i];
    }
}
__device__ __forceinline__ float MaxNan(float a, float b)       // a NaN if one of them is
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// The values in 32 bits, and the largest magnitude as they lay in memory (exact in 32 bits; NaN if there is one): two at a time where
// the type has such an instruction.
__device__ __forceinline__ void Widen(const Sixteen<float> &in, float (&v)[16], float *top)
{
    *top = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) { v[i] = ((const float *)&in)[i]; *top = MaxNan(*top, fabsf(v[i])); }
}
__device__ __forceinline__ void Widen(const Sixteen<__nv_bfloat16> &in, float (&v)[16], float *top)
{
    const __nv_bfloat162 *p = (const __nv_bfloat162 *)&in;
    __nv_bfloat162 m = __habs2(p[0]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t w = ((const uint32_t *)&in)[i];
        v[2 * i] = __uint_as_float(w << 16); v[2 * i + 1] = __uint_as_float(w & 0xffff0000u);
        if (i) m = __hmax2_nan(m, __habs2(p[i]));
    }
    *top = __bfloat162float(__hmax_nan(__low2bfloat16(m), __high2bfloat16(m)));
}
__device__ __forceinline__ void WidenHalves(const __half2 (&p)[8], float (&v)[16], float *top)
{
    __half2 m = __habs2(p[0]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 f = __half22float2(p[i]);
        v[2 * i] = f.x; v[2 * i + 1] = f.y;
        if (i) m = __hmax2_nan(m, __habs2(p[i]));
    }
    *top = __half2float(__hmax_nan(__low2half(m), __high2half(m)));
}
__device__ __forceinline__ void Widen(const Sixteen<__half> &in, float (&v)[16], float *top)
{
    __half2 p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = ((const __half2 *)&in)[i];
    WidenHalves(p, v, top);
}
__device__ __forceinline__ void Widen(const Sixteen<__nv_fp8_e4m3> &in, float (&v)[16], float *top)
{
    __half2 p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(((const uint16_t *)&in)[i], __NV_E4M3);
        p[i] = *(const __half2 *)&h;
    }
    WidenHalves(p, v, top);
}

// {even column in the low half of byte i, odd in the high half} for eight values
__device__ __forceinline__ uint32_t PackE2m1(const float *v)
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

// Values that a lane takes at a time: 16, or a whole block of fp8, where the work around the values weighs more than the values
// (32768 x 7168 grouped: 111 us with 16, 73 with 32).
template <typename T> constexpr int kPieces = sizeof(T) == 1 ? 2 : 1;
template <typename T> constexpr int kLanes = 8 / kPieces<T>;
template <typename T> constexpr int kBlocks = sizeof(T) == 1 ? 3 : 5;           // that fit on a SM

template <typename T>
__global__ void __launch_bounds__(kThreads, kBlocks<T>) QuantizeKernel(Rows r, Source s, uint8_t *values, uint8_t *scales)
{
    extern __shared__ int start[];          // with grouped rows: where each expert's start, then where its tiles do
    int *const tile = start + r.experts + 1;
    sm100::GridDependencyWait();
    sm100::GridDependentsLaunch();
    const Range range = RowsOf(r, start, tile);
    constexpr int P = kPieces<T>, L = kLanes<T>;
    const int lane = threadIdx.x & (L - 1);
    constexpr int U = 4 / (int)sizeof(T) / P;           // 64 bytes a lane are under way at once
    Walk w(L, range, r, start, tile);
    const int at = w.col * kTileCols + lane * 16 * P;
    const bool inside = at < r.cols;
    // the lanes of a warp go round together: the shuffle below is the whole warp's
    for (int left = w.most; left > 0; left -= U) {
        Sixteen<T> in[U][P];
        float mul[U];
        uint8_t *to[U], *scaleTo[U];            // NULL: nothing to store
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int h = 0; h < P; ++h) in[u][h] = Sixteen<T>();
            mul[u] = 1.f;
            to[u] = scaleTo[u] = nullptr;
            if (w.row < w.end) {
                scaleTo[u] = scales + w.Scales(r) + (lane * P >> 1);
                if (inside) {
                    const int64_t from = r.batch > 1 ? w.segment * s.batchPitch + (w.row - w.segmentRow) * s.rowPitch : w.row * s.rowPitch;
#pragma unroll
                    for (int h = 0; h < P; ++h) Load(&in[u][h], (const T *)s.x + from + at + 16 * h, s.aligned);
                    if constexpr (sizeof(T) == 1) mul[u] = s.xScales[w.row * s.scalePitch + w.col];
                    to[u] = values + (w.row * r.cols + at) / 2;
                }
            }
            w.Next(r, start, tile);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float v[P][16], top = 0;
#pragma unroll
            for (int h = 0; h < P; ++h) {
                float t;
                Widen(in[u][h], v[h], &t);
                top = MaxNan(top, t);
            }
            // rounding keeps order: the largest product is that of the largest value
            if constexpr (sizeof(T) == 1) top = __fmul_rn(top, mul[u]);
            uint32_t bits = __float_as_uint(top) & 0x7fffffffu;
            if constexpr (P == 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 1));
            // the exponent field less two, or 255 where the block holds something that is no number
            const uint32_t scale = bits >= 0x7f800000u ? 255u : (uint32_t)max((int)(bits >> 23) - 2, 0);
            float inverse = __uint_as_float((scale == 255u ? 127u : 254u - scale) << 23);
            if constexpr (sizeof(T) == 1) {
                // round(q m) 2^-e = round(q (m 2^-e)), as long as neither side leaves the range of ordinary numbers: products below it, of
                // which only some in a block with a large one, become 0 either way
                if (scale < 64) {
#pragma unroll
                    for (int i = 0; i < 16 * P; ++i) v[i / 16][i % 16] = __fmul_rn(v[i / 16][i % 16], mul[u]);
                } else inverse *= mul[u];
            }
#pragma unroll
            for (int i = 0; i < 16 * P; ++i) v[i / 16][i % 16] *= inverse;
            if (to[u]) {
                if constexpr (P == 1) *(uint2 *)to[u] = make_uint2(PackE2m1(v[0]), PackE2m1(v[0] + 8));
                else *(uint4 *)to[u] = make_uint4(PackE2m1(v[0]), PackE2m1(v[0] + 8), PackE2m1(v[P - 1]), PackE2m1(v[P - 1] + 8));
            }
            if ((P == 2 || (lane & 1) == 0) && scaleTo[u]) *scaleTo[u] = to[u] ? (uint8_t)scale : 0;
        }
    }
}

__device__ __forceinline__ float ScaleOf(uint32_t byte)
{
    return byte == 255u ? __uint_as_float(0x7fc00000u) : byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}
__device__ __forceinline__ void UnpackE2m1(uint32_t word, float *v)
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

// 32 bytes in one store: two of 16 at this stride reach the lines half by half (8192 x 28672 to bf16: 144 us instead of 103).
__device__ __forceinline__ void Store32(void *p, const uint4 &a, const uint4 &b)
{
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w) : "memory");
}

constexpr int kBlocksBack = 4;

template <typename T>
__global__ void __launch_bounds__(kThreads, kBlocksBack) DequantizeKernel(Rows r, const uint8_t *values, const uint8_t *scales, T *out)
{
    extern __shared__ int start[];          // with grouped rows: where each expert's start, then where its tiles do
    int *const tile = start + r.experts + 1;
    sm100::GridDependencyWait();
    sm100::GridDependentsLaunch();
    const Range range = RowsOf(r, start, tile);
    const int lane = threadIdx.x & 7;
    constexpr int U = 2;
    Walk w(8, range, r, start, tile);
    const int col = w.col * kTileCols + lane * 16;
    if (col >= r.cols) return;
    while (w.row < w.end) {
        uint2 word[U];
        uint32_t byte[U];
        int64_t at[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            at[u] = w.row < w.end ? w.row * r.cols + col : -1;
            if (at[u] >= 0) {
                word[u] = *(const uint2 *)(values + at[u] / 2);
                byte[u] = scales[w.Scales(r) + (lane >> 1)];
            }
            w.Next(r, start, tile);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (at[u] < 0) continue;
            float v[16];
            UnpackE2m1(word[u].x, v);
            UnpackE2m1(word[u].y, v + 8);
            const float scale = ScaleOf(byte[u]);
            Sixteen<T> o;
#pragma unroll
            for (int i = 0; i < 16; ++i) ((T *)&o)[i] = FromFloat<T>(v[i] * scale);
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) Store32(out + at[u] + i * (32 / sizeof(T)), o.q[2 * i], o.q[2 * i + 1]);
        }
    }
}

HcclResult CheckRows(const char *what, int64_t batch, int64_t rows, int64_t cols, const int32_t *offsets, int experts)
{
    if (batch < 0 || rows < 0 || cols < 0 || cols % kBlock || rows > INT32_MAX || cols > INT32_MAX || (batch && rows > kMostRows / batch)) {
        RPT_ERR("EI0003", "%s: %lld x %lld x %lld, columns must be a multiple of 32 and rows no more than 2^31 - 2^20 in all", what, (long long)batch, (long long)rows, (long long)cols);
        return HCCL_E_PARA;
    }
    if (experts < 0 || experts > kMaxExperts || (experts > 0) != (offsets != nullptr) || (experts > 0 && batch != 1)) {
        RPT_ERR("EI0003", "%s: grouped rows need offsets, 1 to %d experts and a single matrix (experts %d)", what, kMaxExperts, experts);
        return HCCL_E_PARA;
    }
    return HCCL_SUCCESS;
}

// small operands: a chunk to every team of lanes, so that all loads are under way at once; large ones: as many blocks as fit
// at once, since each builds the table of groups first (5003 x 2048 by 32 experts, eight blocks a SM: 12.5 us, five 10.0)
int64_t SetGrid(Rows *r, int lanes, int blocks, int sms)
{
    const int teams = kThreads / lanes;
    const int64_t rows = r->batch * r->rows, chunks = rows * r->tileCols;
    const int64_t least = ((int64_t)r->tileCols + teams - 1) / teams;          // a row at a time needs so many
    const int64_t grid = std::max(least, std::min<int64_t>((chunks + teams - 1) / teams, (int64_t)sms * blocks));
    r->across = (int)(grid * teams / r->tileCols);
    r->most = (int)((rows + r->across - 1) / r->across);
    return grid;
}

// Programmatic launch: set-up overlaps the end of the kernel in front, which the kernel waits for before it touches memory.
template <typename... Params, typename... Args> HcclResult Launch(const char *what, void (*kernel)(Rows, Params...), int lanes, int blocks, Rows r, void *stream, Args... args)
{
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)SetGrid(&r, lanes, blocks, sms), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = r.experts > 0 ? 8 * (r.experts + 1) : 0;         // no more, so that a product behind finds room beside the last blocks
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at; cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, r, args...);
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
    return Launch("HcommFp4Quantize", QuantizeKernel<T>, kLanes<T>, kBlocks<T>, r, stream, s, (uint8_t *)values, (uint8_t *)scales);
}
template <typename T> HcclResult LaunchDequantize(const Rows &r, const void *values, const void *scales, void *out, void *stream)
{
    return Launch("HcommFp4Dequantize", DequantizeKernel<T>, 8, kBlocksBack, r, stream, (const uint8_t *)values, (const uint8_t *)scales, (T *)out);
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
    if (rowPitch < 0 || batchPitch < 0 || ((uintptr_t)values & 15) || ((uintptr_t)scales & 15) || (fp8 && (cols % 128 || scalePitch < 0 || batch != 1))) {
        RPT_ERR("EI0003", "HcommFp4Quantize: row pitch %lld of %lld columns, scale pitch %lld (none negative); outputs must be 16-byte aligned, fp8 rows a multiple of 128 wide and one matrix",
                (long long)rowPitch, (long long)cols, (long long)scalePitch);
        return HCCL_E_PARA;
    }
    const int64_t wide = dataType == HCCL_DATA_TYPE_FP32 ? 4 : fp8 ? 16 : 8;         // values in 16 bytes
    const Rows r{rows, cols, batch, (int)((cols + kTileCols - 1) / kTileCols), 0, 0, offsets, experts};
    const Source s{x, xScales, batchPitch, rowPitch, scalePitch, ((uintptr_t)x & 15) == 0 && rowPitch % wide == 0 && (batch == 1 || batchPitch % wide == 0)};
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
    if (((uintptr_t)values & 15) || ((uintptr_t)scales & 15) || ((uintptr_t)out & 31)) {
        RPT_ERR("EI0003", "HcommFp4Dequantize: values and scales must be 16-byte aligned, the result 32");
        return HCCL_E_PARA;
    }
    const Rows r{rows, cols, batch, (int)((cols + kTileCols - 1) / kTileCols), 0, 0, offsets, experts};
    switch (dataType) {
        case HCCL_DATA_TYPE_FP32: return LaunchDequantize<float>(r, values, scales, out, stream);
        case HCCL_DATA_TYPE_FP16: return LaunchDequantize<__half>(r, values, scales, out, stream);
        case HCCL_DATA_TYPE_BFP16: return LaunchDequantize<__nv_bfloat16>(r, values, scales, out, stream);
        default:
            RPT_ERR("EI0003", "HcommFp4Dequantize: data type %d is not FP32, FP16 or BFP16", dataType);
            return HCCL_E_PARA;
    }
}

// Whether a team of the quantiser's lanes takes its rows and no others, on a device of so many SMs and of rows without groups: followed in 64 bits
// beside the kernel's own numbers for as long as it goes round.  Returns how many teams there are, of which the last ones may be left over; -1: no
// such call, -2: it takes a row that is not its own.
extern "C" int64_t HcommToolFp4Walk(int64_t rows, int64_t cols, int dataType, int sms, int64_t team)
{
    if (rows < 1 || cols < kBlock || CheckRows("HcommToolFp4Walk", 1, rows, cols, nullptr, 0) != HCCL_SUCCESS) return -1;
    const bool fp8 = dataType == HCCL_DATA_TYPE_FP8E4M3;
    const int lanes = fp8 ? kLanes<__nv_fp8_e4m3> : kLanes<float>, blocks = fp8 ? kBlocks<__nv_fp8_e4m3> : kBlocks<float>, together = 4;
    Rows r{rows, cols, 1, (int)((cols + kTileCols - 1) / kTileCols), 0, 0, nullptr, 0};
    const int64_t teams = SetGrid(&r, lanes, blocks, sms) * (kThreads / lanes), lane = team / r.tileCols;
    int64_t at = lane < r.across ? std::min(lane, rows) : rows;
    RowNumber row = (RowNumber)at;
    const RowNumber end = (RowNumber)rows;
    for (int left = r.most; left > 0; left -= together)
        for (int u = 0; u < together; ++u) {
            if (row < end && ((int64_t)row != at || at < 0)) return -2;
            row = (RowNumber)((uint32_t)row + r.across);
            at += r.across;
        }
    return teams;
}
