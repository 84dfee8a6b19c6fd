/* hcomm_fp4.h - microscaled 4-bit floating point: quantisation, and products on the tensor cores' block-scaled path.
 *
 * A value is e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two to a byte, the even column in the low half.  Every 32
 * consecutive values of a row share a power of two, 2^(byte - 127); byte 255 makes the whole block NaN.  This is the MXFP4 format of the Open
 * Compute Project's microscaling specification.
 *
 * Scale bytes lie in tiles of 128 rows x 4 blocks (128 columns), 512 bytes each: tile (r / 128, c / 128) is number
 * (r / 128) * ceil(cols / 128) + c / 128 and holds the byte of row r, column c at (r % 32) * 16 + (r % 128) / 32 * 4 + c % 128 / 32.
 * Bytes of columns beyond the last are 0.
 *
 * Rows grouped by expert: with `offsets` (int32 [experts + 1] on the device, as the expert-parallel exchange delivers
 * them) expert e owns rows offsets[e] .. offsets[e + 1]; rows behind the last are neither read nor written.  The values of the rows stay
 * where the rows are; scale tiles start anew with every expert, at tile row sum over e' < e of ceil(rows of e' / 128).
 *
 * `stream` is a cudaStream_t.  Functions launch on the current device and return an HcclResult.  The reference library
 * has no compute operators.
 */
#ifndef HCOMM_FP4_H
#define HCOMM_FP4_H

#include <stdint.h>

#include "hccl/hccl_types.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of the scale tiles of `batch` matrices of rows x cols; experts > 0: of one matrix whose rows are grouped (batch must be 1). */
uint64_t HcommFp4ScaleBytes(int64_t batch, int64_t rows, int64_t cols, int experts);

/* x [batch][rows][cols] of dataType FP32, FP16, BFP16, or FP8E4M3 with xScales f32 [batch][rows][cols / 128] (a value is then the product
 * of the two, rounded to fp32).  Pitches count elements.  Scale of a block: 2^(floor(log2(largest magnitude)) - 2), at least
 * 2^-127; values are rounded to the nearest, the even one of two, at most 6.  A block that holds an infinity or a NaN is NaN.
 * cols a multiple of 32 (of 128 for FP8E4M3).  values [batch][rows][cols / 2]; 16-byte aligned, like scales.
 * experts > 0: offsets as above, batch 1.  1024 experts at most. */
int HcommFp4Quantize(const void *x, int dataType, const float *xScales, int64_t batch, int64_t rows, int64_t cols, int64_t batchPitch, int64_t rowPitch,
                     int64_t scalePitch, const int32_t *offsets, int experts, void *values, void *scales, void *stream);
/* The values that a quantised tensor stands for, contiguous, rounded to dataType (FP32, FP16, BFP16); 32-byte aligned. */
int HcommFp4Dequantize(const void *values, const void *scales, int64_t batch, int64_t rows, int64_t cols, const int32_t *offsets, int experts, void *out,
                       int dataType, void *stream);

/* out[M][N] (bf16) = A[M][K] * B[N][K]^T, accumulated in fp32.  With experts > 0 the rows of A are grouped as above and B holds `experts`
 * matrices: rows of expert e are multiplied with matrix e; rows of out behind the last expert's are left as they were.
 * K a multiple of 32; M, N and K at most 2^31 - 257; rows of out ldOut elements apart.  out may not overlap an operand. */
int HcommFp4Gemm(const void *aValues, const void *aScales, const void *bValues, const void *bScales, void *out, int M, int N, int K, int64_t ldOut,
                 const int32_t *offsets, int experts, void *stream);
/* out[M][N] = silu(A * G^T) * (A * U^T): the gate and up projections of a gated feed-forward layer in one pass over A, the
 * product taken from the fp32 accumulators.  silu is taken as 0 where its argument is below -87.3 (magnitudes below 2^-119). */
int HcommFp4GemmSwiglu(const void *aValues, const void *aScales, const void *gValues, const void *gScales, const void *uValues, const void *uScales, void *out,
                       int M, int N, int K, int64_t ldOut, const int32_t *offsets, int experts, void *stream);
/* Reads and clears the "a bounded wait expired inside a product" flag of the current device (0 = none). */
int HcommFp4TakeError(void);

#ifdef __cplusplus
}
#endif
#endif
