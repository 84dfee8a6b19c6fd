/* hcomm_moe.h - expert-parallel exchange for mixture-of-experts layers: dispatch (tokens to the ranks that own their
 * experts, quantised to fp8 e4m3 with one fp32 scale per 128 values on the way) and combine (expert outputs back to the
 * token's rank with the gate-weighted sum fused).  The reference library offers AlltoAll(V/VC) for this
 * (pkg_inc/legacy/hccl/hccl_inner.h:55-66); routing, quantisation and the weighted sum are fused here.
 * `stream` is a cudaStream_t; functions return an HcclResult value. */
#pragma once
#include <stdint.h>

#include "hccl/hccl_types.h"

#ifdef __cplusplus
extern "C" {
#endif
// Offsets are relative to the start of each rank's buffer; the layout is identical on all ranks.
struct MoeLayout {
    int32_t numExperts, topk, hidden, maxTokens, maxRecvRows, reserved;
    uint64_t offCounts;          // u32 [nRanks][expertsPerRank]      rows each source sends to each local expert
    uint64_t offExpertOffsets;   // u32 [expertsPerRank + 1]          start row of every local expert, last = total
    uint64_t offOrigin;          // u64 [maxRecvRows]                 (source rank << 32) | (token * topk + k)
    uint64_t offScales;          // f32 [maxRecvRows][hidden / 128]
    uint64_t offRows;            // fp8 e4m3 [maxRecvRows][hidden]
    uint64_t offCombine;         // bf16 [maxTokens][topk][hidden]    landing area of the combine step: rows from other ranks, from all
                                 //                                   once HcommMoeGetBuffers has been asked for its address
    uint64_t totalBytes;
    uint64_t offValid;           // u8 [maxTokens][topk]              1 = dispatch sent this (token, k), 0 = masked or dropped
};
#ifndef __cplusplus
typedef struct MoeLayout MoeLayout;
#endif

/* Collective: every rank allocates the same symmetric buffer (capacityFactor x maxTokens x topk receive rows; <= 0 means 2)
 * and maps its peers'.  numExperts a multiple of the rank count (<= 1024), topk <= 16, hidden a multiple of 512 (<= 8192). */
int HcommMoeCreate(HcclComm comm, int numExperts, int topk, int hidden, int maxTokens, float capacityFactor, void **handle, MoeLayout *layoutOut);
int HcommMoeDestroy(void *handle);
/* Local addresses of the receive-side arrays (valid after a dispatch on the same stream; any may be NULL).  Asking for
 * `combine` makes every later HcommMoeCombine place the row of each (token, k) that was sent in that area, those of this
 * rank's own experts as well; until then these are summed where y holds them, which is faster. */
int HcommMoeGetBuffers(void *handle, void **rows, void **scales, void **origin, void **expertOffsets, void **combine);
/* x: bf16 [numTokens][hidden]; topkIdx: int32 [numTokens][topk], an index outside [0, numExperts) masks that choice. */
int HcommMoeDispatch(void *handle, const void *x, const int32_t *topkIdx, int numTokens, void *stream);
/* y: bf16 expert outputs in receive-row order; gates: f32 [numTokens][topk]; out: bf16 [numTokens][hidden], which may lie
 * inside y.  HcommMoeCombineRows is told how many rows the memory at y has room for; HcommMoeCombine assumes the receive
 * capacity, and takes a result that starts behind a shorter y for one inside it (same result, a pass more). */
int HcommMoeCombine(void *handle, const void *y, const float *gates, void *out, int numTokens, void *stream);
int HcommMoeCombineRows(void *handle, const void *y, uint64_t yRows, const float *gates, void *out, int numTokens, void *stream);
/* HcommMoeCombineRows with the gates of HcommMoeRoute, which gives a token whose logits are no numbers choices of -1 and gates of NaN: a token with a
 * gate of NaN comes back as NaN, also where no row was sent for it (the other two leave such a gate out, whatever it holds). */
int HcommMoeCombineRouted(void *handle, const void *y, uint64_t yRows, const float *gates, void *out, int numTokens, void *stream);
/* Rows dropped because a rank received more than its capacity since the last call (clears the counter). */
int HcommMoeTakeOverflow(void *handle);

// HcommMoeDispatch with the kernel's per-expert counters kept in an array built into the library's device image
// rather than in allocated memory: the call allocates nothing, on the device or through any library.  Same
// arguments and results as HcommMoeDispatch.  This entry point has no counterpart in the reference library.
// Up to 256 experts (1 KB of built-in scratch per process and GPU); larger exchanges return HCCL_E_PARA, with a single
// rank too, which needs no counters in memory.
// All calls on one GPU share the array: it is cleared at the start of every call, and calls that overlap in time
// race on it (not those of a single rank).  The array's address is resolved by HcommMoeCreate (set-up time); the call must be made with the
// exchange's GPU current and is refused with HCCL_E_PARA otherwise.
int HcommMoeDispatchStaticScratch(void *handle, const void *x, const int32_t *topkIdx, int numTokens, void *stream);

/* Routing: what dispatch and combine take, from the router's logits.  No communicator is involved.
 *
 * logits [tokens][experts] (FP32, FP16, BFP16; rows ldLogits elements apart).  A token's k largest logits - with `bias` (f32 [experts],
 * HCOMM_MOE_SIGMOID only): its k largest sigmoid(logit) + bias, compared in 64 bits - are its choices, largest first, of equal ones
 * the lowest index.  p is the softmax of the logits, or the sigmoids divided by their sum.
 *   topkIdx i32 [tokens][topk]   expert, or -1: nothing left to choose
 *   gates   f32 [tokens][topk]   scale * score of the choice, softmax probability or sigmoid; renormalize: divided by the sum over the token's
 *                                choices.  0 where topkIdx is -1
 *   counts  i32 [experts + 1]    tokens that chose the expert; last: tokens counted (T)
 *   probSums f32 [experts]       sum of p over the tokens, or NULL
 *   loss    f32                  balance * experts * sum over e of counts[e] / (T topk) * probSums[e] / T, or NULL
 * A logit of -inf takes the expert out for the token.  Tokens whose `valid` byte (NULL: all) is 0 choose -1, have gates of 0 and are not counted.
 * A row that holds a NaN (or, of a softmax, +inf) chooses -1 with gates of NaN, and makes sums and loss NaN.
 * Sums are added up in an order that depends on the sizes and the device alone.  experts <= 1024, topk <= 16.
 * scratch: HcommMoeRouteScratchBytes, 4-byte aligned, whatever it holds; free again once the stream has passed the call. */
#define HCOMM_MOE_SOFTMAX 0
#define HCOMM_MOE_SIGMOID 1
uint64_t HcommMoeRouteScratchBytes(int tokens, int experts);
int HcommMoeRoute(const void *logits, int dataType, int64_t ldLogits, int tokens, int experts, int topk, int scoring, int renormalize, float scale, const float *bias,
                  const uint8_t *valid, int32_t *topkIdx, float *gates, int32_t *counts, float *probSums, float balance, float *loss, void *scratch, void *stream);
/* The loss alone, from counts and probSums that were summed over ranks. */
int HcommMoeBalanceLoss(const int32_t *counts, const float *probSums, int experts, int topk, float balance, float *loss, void *stream);
/* dlogits [tokens][experts] in the logits' type (rows ldGrad apart) from dgates f32 [tokens][topk] and dloss f32 (either may be NULL), with the
 * arguments of the call in front and its topkIdx and counts (summed over ranks, where the loss was).  Rows that are not valid get 0. */
int HcommMoeRouteBackward(const void *logits, int dataType, int64_t ldLogits, int tokens, int experts, int topk, int scoring, int renormalize, float scale, const uint8_t *valid,
                          const int32_t *topkIdx, const float *dgates, const int32_t *counts, float balance, const float *dloss, void *dlogits, int64_t ldGrad, void *stream);
#ifdef __cplusplus
}
#endif
