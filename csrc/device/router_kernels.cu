// router_kernels.cu - top-k routing for mixture-of-experts layers with per-expert counts and a balance loss, forward and
// backward (entry points: include/hcomm_moe.h).  It makes the choices and gates that dispatch and combine take.
//
// With x a token's logits, z = x (softmax) or log sigmoid(x), p = softmax(z) over the experts:
//   choice   the k largest x (or sigmoid(x) + bias), of equal ones the lowest index
//   gate     s * softmax of z over the chosen, or s p, or s sigmoid(x)
//   counts   n_e = tokens that chose e;  f_e = n_e / (T k),  P_e = sum_t p_te / T,  loss = c E sum_e f_e P_e
// Backward, with w_e = dloss c E f_e / T (the choices are constants):
//   softmax gates not renormalised join w:  u_e = w_e + s dgate_e;  dz_e = p_e (u_e - sum_j p_j u_j)
//   renormalised, g the gates / s:          dz_e += g_e s (dgate_e - sum_j g_j dgate_j)
//   sigmoid gates not renormalised:         dz_e += s dgate_e sigmoid(x_e)
//   dx = dz (softmax) or dz sigmoid(-x)
// An x of -inf is an expert that is off: p = 0, never chosen.  A row in which nothing is left chooses -1 and has gates of 0.
//
// One warp takes a token: lane l holds the V experts l V .. l V + V - 1 in registers, so that the row is read once, the lowest
// lane among equals is the lowest index, and the k rounds of the choice are a maximum in the lane, one warp-wide integer
// maximum (redux) and a ballot.  Sums over tokens stay in registers for as long as a warp works, then go to shared memory and, a
// row for each block, to scratch; they are added up in a fixed order, so results do not depend on which block was first.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/hcomm_moe.h"
#include "../core/log.h"
#include "sm100_ptx.cuh"

namespace {

constexpr int kMaxExperts = 1024, kMaxTopk = 16;
constexpr uint32_t kAll = 0xffffffffu;
constexpr int kFinishThreads = 1024;

struct Params {
    const void *logits;
    int64_t ld;
    int tokens, experts, topk;
    bool sigmoid, renormalize, vectors;     // vectors: rows may be read V values at a time
    float scale, balance;
    const float *bias;
    const uint8_t *valid;
    int32_t *idx;
    float *gates;
    int32_t *counts;                        // [experts + 1], the last one counts the tokens
    float *sums, *loss;                     // sums [experts]: of p over the tokens
    float *partSums;                        // scratch: [blocks][experts], then the counts likewise
    int32_t *partCounts;                    // [blocks][experts + 1]
    // backward
    const float *dgates, *dloss;
    void *dlogits;
    int64_t ldGrad;
};

template <typename T> __device__ __forceinline__ float ToFloat(T v);
template <> __device__ __forceinline__ float ToFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ float ToFloat<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float ToFloat<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T FromFloat(float v);
template <> __device__ __forceinline__ float FromFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ __half FromFloat<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 FromFloat<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <int Bytes> struct Word {};
template <> struct Word<2> { using type = uint16_t; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<16> { using type = uint4; };

// This lane's V values of a row; -inf behind the last expert.
template <typename T, int V> __device__ __forceinline__ void LoadRow(float (&x)[V], const T *row, int experts, int first, bool vectors)
{
    constexpr int kBytes = V * (int)sizeof(T), kWord = kBytes > 16 ? 16 : kBytes;
    using W = typename Word<kWord>::type;
    __align__(16) T raw[V];
    if (vectors) {
        if (first < experts) {
#pragma unroll
            for (int i = 0; i < kBytes / kWord; ++i) ((W *)raw)[i] = __ldg((const W *)(row + first) + i);
#pragma unroll
            for (int j = 0; j < V; ++j) x[j] = ToFloat(raw[j]);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) x[j] = -INFINITY;
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = first + j < experts ? ToFloat(row[first + j]) : -INFINITY;
    }
}
template <typename T, int V> __device__ __forceinline__ void StoreRow(const float (&x)[V], T *row, int experts, int first, bool vectors)
{
    constexpr int kBytes = V * (int)sizeof(T), kWord = kBytes > 16 ? 16 : kBytes;
    using W = typename Word<kWord>::type;
    __align__(16) T raw[V];
#pragma unroll
    for (int j = 0; j < V; ++j) raw[j] = FromFloat<T>(x[j]);
    if (vectors) {
        if (first < experts) {
#pragma unroll
            for (int i = 0; i < kBytes / kWord; ++i) ((W *)(row + first))[i] = ((const W *)raw)[i];
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (first + j < experts) row[first + j] = raw[j];
    }
}

__device__ __forceinline__ float WarpSum(float v)
{
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(kAll, v, d);
    return v;
}
__device__ __forceinline__ float WarpMax(float v)
{
#pragma unroll
    for (int d = 16; d; d >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, d));
    return v;
}

// Integers that order like the floats they are made of, 0 for "not a candidate" (below every float).  Both zeros are one value.
__device__ __forceinline__ uint32_t Key(float x)
{
    const uint32_t b = __float_as_uint(x + 0.f);
    return x == -INFINITY ? 0u : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t Key(double x)
{
    const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
    return x == -INFINITY ? 0u : b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ uint32_t WarpMaxKey(uint32_t k) { return __reduce_max_sync(kAll, k); }
__device__ __forceinline__ uint64_t WarpMaxKey(uint64_t k)
{
    const uint32_t hi = __reduce_max_sync(kAll, (uint32_t)(k >> 32));
    const uint32_t lo = __reduce_max_sync(kAll, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
    return (uint64_t)hi << 32 | lo;
}

// log sigmoid(x), also where the sigmoid itself is next to nothing
__device__ __forceinline__ float LogSigmoid(float x) { return fminf(x, 0.f) - log1pf(expf(-fabsf(x))); }

// The k largest keys of the warp: lane i gets the i-th, its expert and its x; experts of -1 where no candidate is left.
template <int V, typename K> __device__ __forceinline__ void TopK(K (&key)[V], const float (&x)[V], int topk, int lane, int *expert, float *value)
{
    *expert = -1; *value = 0.f;
    for (int i = 0; i < topk; ++i) {
        K best = key[0];
        int at = 0;
        float bx = x[0];
#pragma unroll
        for (int j = 1; j < V; ++j)
            if (key[j] > best) { best = key[j]; at = j; bx = x[j]; }
        const K top = WarpMaxKey(best);
        if (top == 0) break;
        const int winner = __ffs(__ballot_sync(kAll, best == top)) - 1;
        const int e = __shfl_sync(kAll, lane * V + at, winner);
        const float v = __shfl_sync(kAll, bx, winner);
        if (lane == i) { *expert = e; *value = v; }
        if (lane == winner) {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j == at) key[j] = 0;
        }
    }
}

// The row as probabilities: x becomes p; the row's maximum must not be -inf in all lanes.
template <int V> __device__ __forceinline__ void Softmax(float (&x)[V], bool sigmoid)
{
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (sigmoid && x[j] != -INFINITY) x[j] = LogSigmoid(x[j]);
        top = fmaxf(top, x[j]);
    }
    top = WarpMax(top);
    if (top == -INFINITY) top = 0.f;            // nothing left: all of them become 0
    float sum = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) { x[j] = expf(x[j] - top); sum += x[j]; }
    sum = WarpSum(sum);
    const float inverse = sum > 0 ? 1.f / sum : 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] *= inverse;
}

// A row without a defined softmax (or sum of sigmoids): it holds a NaN, or +inf under softmax.
template <int V> __device__ __forceinline__ bool Undefined(const float (&x)[V], bool sigmoid)
{
    bool bad = false;
#pragma unroll
    for (int j = 0; j < V; ++j) bad |= x[j] != x[j] || (!sigmoid && x[j] == INFINITY);
    return __any_sync(kAll, bad);
}

// Share of the chosen: lanes below topk with an expert hold its x.
__device__ __forceinline__ float ChosenShare(float x, bool chosen, bool sigmoid)
{
    const float z = chosen ? (sigmoid ? LogSigmoid(x) : x) : -INFINITY;
    const float top = WarpMax(z);
    const float e = chosen ? expf(z - top) : 0.f;
    const float sum = WarpSum(e);
    return chosen ? e / sum : 0.f;
}

// Adds up the blocks' rows of scratch (or takes the only block's sums), writes counts, sums and loss.  All threads of one block.
__device__ void Finish(const Params &p, int blocks, const float *sums, const int32_t *counts, float *warpSum)
{
    const int E = p.experts, threads = blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __shared__ float total;
    // the count of tokens lies behind those of the experts
    if (warp == 0) {
        int n = 0;
        for (int b = lane; b < blocks; b += 32) n += counts[(size_t)b * (E + 1) + E];
        n = __reduce_add_sync(kAll, n);
        if (lane == 0) { p.counts[E] = n; total = (float)max(n, 1); }
    }
    float loss = 0;
    for (int e = threadIdx.x; e < E; e += threads) {
        int n = 0;
        float s = 0;
#pragma unroll 8
        for (int b = 0; b < blocks; ++b) {
            n += counts[(size_t)b * (E + 1) + e];
            if (sums) s += sums[(size_t)b * E + e];
        }
        p.counts[e] = n;
        if (p.sums) p.sums[e] = s;
        loss += (float)n * s;
    }
    loss = WarpSum(loss);
    if (lane == 0) warpSum[warp] = loss;
    __syncthreads();
    if (threadIdx.x == 0 && p.loss) {
        float all = 0;
        for (int w = 0; w < threads / 32; ++w) all += warpSum[w];
        *p.loss = p.balance * E * (all / (total * p.topk) / total);
    }
}

template <int V> constexpr int Threads() { return V >= 16 ? 512 : 1024; }      // 128 or 64 registers a thread

template <typename T, int V>
__global__ void __launch_bounds__(Threads<V>()) RouteKernel(const __grid_constant__ Params p)
{
    constexpr int kWarps = Threads<V>() / 32;
    extern __shared__ float shared[];           // counts of the block, then one row of sums for each warp in use
    __shared__ float warpSum[32];
    int32_t *counts = (int32_t *)shared;
    float *rows = shared + p.experts + 1;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, E = p.experts, first = lane * V;
    sm100::GridDependencyWait();
    sm100::GridDependentsLaunch();
    for (int e = threadIdx.x; e <= E; e += Threads<V>()) counts[e] = 0;
    __syncthreads();
    const bool stats = p.partSums != nullptr;           // sums of the probabilities are wanted
    float sum[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = 0;
    int seen = 0;
    for (int64_t t = (int64_t)blockIdx.x * kWarps + warp; t < p.tokens; t += (int64_t)gridDim.x * kWarps) {
        const bool counted = !p.valid || p.valid[t];
        int expert = -1;
        float gate = 0;
        if (counted) {
            ++seen;
            float x[V];
            LoadRow<T, V>(x, (const T *)p.logits + t * p.ld, E, first, p.vectors);
            bool bad = Undefined(x, p.sigmoid);
            float value = 0;
            if (p.bias) {
                uint64_t key[V];
                bool none = false;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    // in 64 bits: a choice between two scores that 32 bits cannot tell apart must not hang on the way they were rounded
                    const double s = x[j] == -INFINITY ? -INFINITY : 1.0 / (1.0 + exp(-(double)x[j])) + (double)p.bias[first + j < E ? first + j : 0];
                    none |= s != s;
                    key[j] = Key(s);
                }
                bad = bad || __any_sync(kAll, none);
                if (!bad) TopK<V, uint64_t>(key, x, p.topk, lane, &expert, &value);
            } else {
                uint32_t key[V];
#pragma unroll
                for (int j = 0; j < V; ++j) key[j] = Key(x[j]);
                if (!bad) TopK<V, uint32_t>(key, x, p.topk, lane, &expert, &value);
            }
            const bool chosen = expert >= 0;
            if (p.renormalize) gate = ChosenShare(value, chosen, p.sigmoid);
            else if (p.sigmoid) gate = chosen ? expf(LogSigmoid(value)) : 0.f;
            if (stats || (!p.renormalize && !p.sigmoid)) {
                float top = 0, whole = 0;
                if (!p.renormalize && !p.sigmoid) {
                    // the chosen one's probability from its own x, by the same steps as the row's
                    top = -INFINITY;
#pragma unroll
                    for (int j = 0; j < V; ++j) top = fmaxf(top, x[j]);
                    top = WarpMax(top);
#pragma unroll
                    for (int j = 0; j < V; ++j) whole += x[j] == -INFINITY ? 0.f : expf(x[j] - top);
                    whole = WarpSum(whole);
                    gate = chosen ? expf(value - top) / whole : 0.f;
                }
                if (stats) {
                    Softmax(x, p.sigmoid);
#pragma unroll
                    for (int j = 0; j < V; ++j) sum[j] += bad ? NAN : x[j];
                }
            }
            gate = bad ? NAN : gate * p.scale;
            if (chosen) atomicAdd(&counts[expert], 1);
        }
        if (lane < p.topk) {
            p.idx[t * p.topk + lane] = expert;
            p.gates[t * p.topk + lane] = gate;
        }
    }
    if (lane == 0) atomicAdd(&counts[E], seen);
    if (stats) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (first + j < E) rows[warp * E + first + j] = sum[j];
    }
    __syncthreads();
    if (stats) {
        for (int e = threadIdx.x; e < E; e += Threads<V>()) {
            float s = 0;
            for (int w = 0; w < kWarps; ++w) s += rows[w * E + e];
            rows[e] = s;                    // only this thread reads or writes column e
            if (gridDim.x > 1) p.partSums[(size_t)blockIdx.x * E + e] = s;
        }
    }
    if (gridDim.x > 1) {
        for (int e = threadIdx.x; e <= E; e += Threads<V>()) p.partCounts[(size_t)blockIdx.x * (E + 1) + e] = counts[e];
    } else {
        __syncthreads();
        Finish(p, 1, stats ? rows : nullptr, counts, warpSum);
    }
}

__global__ void __launch_bounds__(kFinishThreads) FinishKernel(const __grid_constant__ Params p, int blocks)
{
    __shared__ float warpSum[32];
    sm100::GridDependencyWait();
    sm100::GridDependentsLaunch();
    Finish(p, blocks, p.partSums, p.partCounts, warpSum);
}

// The loss from counts and sums that were added up over ranks: one warp.
__global__ void BalanceLossKernel(const int32_t *counts, const float *sums, int experts, int topk, float balance, float *loss)
{
    sm100::GridDependencyWait();
    float all = 0;
    for (int e = threadIdx.x; e < experts; e += 32) all += (float)counts[e] * sums[e];
    all = WarpSum(all);
    const float total = (float)max(counts[experts], 1);
    if (threadIdx.x == 0) *loss = balance * experts * (all / (total * topk) / total);
}

template <typename T, int V>
__global__ void __launch_bounds__(Threads<V>()) RouteBackwardKernel(const __grid_constant__ Params p)
{
    constexpr int kWarps = Threads<V>() / 32;
    extern __shared__ float shared[];           // a row for each warp: what comes to the chosen experts alone
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, E = p.experts, first = lane * V;
    float *mine = shared + warp * 32 * V;
    sm100::GridDependencyWait();
    sm100::GridDependentsLaunch();
#pragma unroll
    for (int j = 0; j < V; ++j) mine[first + j] = 0;
    const bool balanced = p.dloss != nullptr, joined = !p.renormalize && !p.sigmoid;
    float w[V];                                 // of the loss: the same for every token
    if (balanced) {
        const float total = (float)max(p.counts[E], 1), c = *p.dloss * p.balance * E / (total * p.topk) / total;
#pragma unroll
        for (int j = 0; j < V; ++j) w[j] = first + j < E ? c * (float)p.counts[first + j] : 0.f;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) w[j] = 0;
    }
    __syncwarp();
    for (int64_t t = (int64_t)blockIdx.x * kWarps + warp; t < p.tokens; t += (int64_t)gridDim.x * kWarps) {
        float d[V];
        if (p.valid && !p.valid[t]) {
#pragma unroll
            for (int j = 0; j < V; ++j) d[j] = 0;
        } else {
            const T *row = (const T *)p.logits + t * p.ld;
            float x[V];
            LoadRow<T, V>(x, row, E, first, p.vectors);
            const bool bad = Undefined(x, p.sigmoid);
            int expert = -1;
            float dg = 0, value = 0;
            if (p.dgates && lane < p.topk) {
                expert = p.idx[t * p.topk + lane];
                if (expert >= 0 && expert < E) {
                    dg = p.dgates[t * p.topk + lane] * p.scale;
                    value = ToFloat(row[expert]);
                } else expert = -1;
            }
            const bool chosen = expert >= 0;
            float to = dg;                      // to the chosen expert alone
            if (p.renormalize) {
                const float share = ChosenShare(value, chosen, p.sigmoid);
                to = share * (dg - WarpSum(share * dg));
            } else if (p.sigmoid) to = chosen ? dg * expf(LogSigmoid(value)) : 0.f;
            if (chosen) mine[expert] = to;
            __syncwarp();
            float own[V];
#pragma unroll
            for (int j = 0; j < V; ++j) own[j] = mine[first + j];
            __syncwarp();
            if (chosen) mine[expert] = 0;
            if (balanced || joined) {
                float q[V];
#pragma unroll
                for (int j = 0; j < V; ++j) q[j] = x[j];
                Softmax(q, p.sigmoid);
                float mean = 0;
#pragma unroll
                for (int j = 0; j < V; ++j) mean += q[j] * (joined ? w[j] + own[j] : w[j]);
                mean = WarpSum(mean);
#pragma unroll
                for (int j = 0; j < V; ++j) d[j] = joined ? q[j] * (w[j] + own[j] - mean) : q[j] * (w[j] - mean) + own[j];
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) d[j] = own[j];
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (p.sigmoid) d[j] = d[j] / (1.f + expf(x[j]));
                if (bad) d[j] = NAN;
            }
        }
        StoreRow<T, V>(d, (T *)p.dlogits + t * p.ldGrad, E, first, p.vectors);
    }
}

int SmCount()
{
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms;
}
int ValuesOf(int experts)           // V: experts a lane holds, a power of two
{
    int v = 1;
    while (32 * v < experts) v *= 2;
    return v;
}
int WarpsOf(int v) { return v >= 16 ? 16 : 32; }
// A block for every round of warps, one a SM at most: each leaves a row of sums behind.
int BlocksOf(int tokens, int experts, int sms)
{
    const int warps = WarpsOf(ValuesOf(experts));
    return std::max(1, std::min(sms, (tokens + warps - 1) / warps));
}
constexpr int kMostBlocks = 256;        // of scratch, whatever the device

template <typename Kernel, typename... Args> HcclResult Launch(const char *what, Kernel *kernel, int grid, int threads, int smem, void *stream, const Args &...args)
{
    if (smem > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
        HCCL_ERROR("%s: %d bytes of shared memory: %s", what, smem, cudaGetErrorString(cudaGetLastError()));
        return HCCL_E_RUNTIME;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
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
template <typename T, bool BACKWARD> HcclResult LaunchRows(const char *what, const Params &p, int grid, void *stream)
{
    const int v = ValuesOf(p.experts), warps = WarpsOf(v);
    const int smem = BACKWARD ? warps * 32 * v * 4 : 4 * (p.experts + 1 + (p.partSums ? warps * p.experts : 0));
    switch (v) {
#define HCOMM_CASE(V) case V: return Launch(what, BACKWARD ? RouteBackwardKernel<T, V> : RouteKernel<T, V>, grid, warps * 32, smem, stream, p);
        HCOMM_CASE(1) HCOMM_CASE(2) HCOMM_CASE(4) HCOMM_CASE(8) HCOMM_CASE(16) HCOMM_CASE(32)
#undef HCOMM_CASE
    }
    return HCCL_E_PARA;
}
template <bool BACKWARD> HcclResult LaunchTyped(const char *what, const Params &p, int dataType, int grid, void *stream)
{
    switch (dataType) {
        case HCCL_DATA_TYPE_FP32: return LaunchRows<float, BACKWARD>(what, p, grid, stream);
        case HCCL_DATA_TYPE_FP16: return LaunchRows<__half, BACKWARD>(what, p, grid, stream);
        case HCCL_DATA_TYPE_BFP16: return LaunchRows<__nv_bfloat16, BACKWARD>(what, p, grid, stream);
        default: return HCCL_E_PARA;
    }
}
int BytesOf(int dataType) { return dataType == HCCL_DATA_TYPE_FP32 ? 4 : 2; }
HcclResult CheckShape(const char *what, int dataType, int64_t ld, int tokens, int experts, int topk, int scoring, const float *bias)
{
    if ((dataType != HCCL_DATA_TYPE_FP32 && dataType != HCCL_DATA_TYPE_FP16 && dataType != HCCL_DATA_TYPE_BFP16) || tokens < 0 || experts < 1 || experts > kMaxExperts || topk < 1 ||
        topk > kMaxTopk || topk > experts || ld < experts || (scoring != HCOMM_MOE_SOFTMAX && scoring != HCOMM_MOE_SIGMOID) || (bias && scoring != HCOMM_MOE_SIGMOID)) {
        RPT_ERR("EI0003", "%s: type %d (FP32, FP16, BFP16), %d tokens, %d experts (<= %d) %lld apart, %d of them chosen (<= %d), scoring %d%s", what, dataType, tokens, experts, kMaxExperts,
                (long long)ld, topk, kMaxTopk, scoring, bias ? " with a bias, which only the sigmoid takes" : "");
        return HCCL_E_PARA;
    }
    return HCCL_SUCCESS;
}
bool Vectors(const void *base, int64_t ld, int experts, int dataType)
{
    const int v = ValuesOf(experts), word = std::min(16, v * BytesOf(dataType));
    return experts % v == 0 && (uintptr_t)base % word == 0 && ld * BytesOf(dataType) % word == 0;
}

}  // namespace

extern "C" uint64_t HcommMoeRouteScratchBytes(int tokens, int experts)
{
    if (tokens < 0 || experts < 1 || experts > kMaxExperts) return 0;
    const int blocks = BlocksOf(tokens, experts, kMostBlocks);
    return blocks == 1 ? 0 : (uint64_t)blocks * (2 * experts + 1) * 4;
}

extern "C" int HcommMoeRoute(const void *logits, int dataType, int64_t ldLogits, int tokens, int experts, int topk, int scoring, int renormalize, float scale, const float *bias,
                             const uint8_t *valid, int32_t *topkIdx, float *gates, int32_t *counts, float *probSums, float balance, float *loss, void *scratch, void *stream)
{
    CHK_RET(CheckShape("HcommMoeRoute", dataType, ldLogits, tokens, experts, topk, scoring, bias));
    const int blocks = BlocksOf(tokens, experts, std::min(kMostBlocks, SmCount()));
    if (!counts || (tokens > 0 && (!logits || !topkIdx || !gates)) || (blocks > 1 && !scratch)) return HCCL_E_PTR;
    if (((uintptr_t)scratch & 3) || (uintptr_t)logits % BytesOf(dataType)) {
        RPT_ERR("EI0003", "HcommMoeRoute: misaligned logits or scratch");
        return HCCL_E_PARA;
    }
    Params p = {};
    p.logits = logits; p.ld = ldLogits;
    p.tokens = tokens; p.experts = experts; p.topk = topk;
    p.sigmoid = scoring == HCOMM_MOE_SIGMOID; p.renormalize = renormalize != 0;
    p.vectors = Vectors(logits, ldLogits, experts, dataType);
    p.scale = scale; p.balance = balance;
    p.bias = bias; p.valid = valid;
    p.idx = topkIdx; p.gates = gates; p.counts = counts; p.sums = probSums; p.loss = loss;
    const bool stats = probSums || loss;
    // a single block needs no scratch: any address that is not NULL says that sums are wanted
    p.partSums = stats ? (blocks > 1 ? (float *)scratch : (float *)counts) : nullptr;
    p.partCounts = (int32_t *)scratch + (blocks > 1 ? (size_t)blocks * experts : 0);
    CHK_RET(LaunchTyped<false>("HcommMoeRoute", p, dataType, blocks, stream));
    if (blocks > 1) return Launch("HcommMoeRoute", FinishKernel, 1, kFinishThreads, 0, stream, p, blocks);
    return HCCL_SUCCESS;
}

extern "C" int HcommMoeBalanceLoss(const int32_t *counts, const float *probSums, int experts, int topk, float balance, float *loss, void *stream)
{
    if (experts < 1 || experts > kMaxExperts || topk < 1 || topk > kMaxTopk) {
        RPT_ERR("EI0003", "HcommMoeBalanceLoss: %d experts (<= %d), %d of them chosen (<= %d)", experts, kMaxExperts, topk, kMaxTopk);
        return HCCL_E_PARA;
    }
    if (!counts || !probSums || !loss) return HCCL_E_PTR;
    return Launch("HcommMoeBalanceLoss", BalanceLossKernel, 1, 32, 0, stream, counts, probSums, experts, topk, balance, loss);
}

extern "C" int HcommMoeRouteBackward(const void *logits, int dataType, int64_t ldLogits, int tokens, int experts, int topk, int scoring, int renormalize, float scale, const uint8_t *valid,
                                     const int32_t *topkIdx, const float *dgates, const int32_t *counts, float balance, const float *dloss, void *dlogits, int64_t ldGrad, void *stream)
{
    CHK_RET(CheckShape("HcommMoeRouteBackward", dataType, ldLogits, tokens, experts, topk, scoring, nullptr));
    if (ldGrad < experts) {
        RPT_ERR("EI0003", "HcommMoeRouteBackward: rows of the gradient overlap");
        return HCCL_E_PARA;
    }
    if (tokens == 0) return HCCL_SUCCESS;
    if (!logits || !dlogits || (dgates && !topkIdx) || (dloss && !counts)) return HCCL_E_PTR;
    if ((uintptr_t)logits % BytesOf(dataType) || (uintptr_t)dlogits % BytesOf(dataType)) {
        RPT_ERR("EI0003", "HcommMoeRouteBackward: misaligned logits or gradient");
        return HCCL_E_PARA;
    }
    Params p = {};
    p.logits = logits; p.ld = ldLogits;
    p.tokens = tokens; p.experts = experts; p.topk = topk;
    p.sigmoid = scoring == HCOMM_MOE_SIGMOID; p.renormalize = renormalize != 0;
    p.vectors = Vectors(logits, ldLogits, experts, dataType) && Vectors(dlogits, ldGrad, experts, dataType);
    p.scale = scale; p.balance = balance;
    p.valid = valid;
    p.idx = const_cast<int32_t *>(topkIdx); p.counts = const_cast<int32_t *>(counts);
    p.dgates = dgates; p.dloss = dloss;
    p.dlogits = dlogits; p.ldGrad = ldGrad;
    const int warps = WarpsOf(ValuesOf(experts));
    const int64_t blocks = std::min<int64_t>((tokens + warps - 1) / warps, 2 * (int64_t)SmCount());
    return LaunchTyped<true>("HcommMoeRouteBackward", p, dataType, (int)blocks, stream);
}
