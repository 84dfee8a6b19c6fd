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
//
// What bounds it beyond some ten thousand tokens is instructions: 65003 x 64 and 65536 x 256 use 84 and 83 % of the issue slots forward, 69 and 71 backward,
// with HBM at 6 to 24 %; one block of 64 registers a SM keeps two to three warps ready in each cycle.  Below that it is the latency of a token's chain -
// maximum after maximum, then exponentials and sums across lanes - and the launches: 4096 x 256, one token a warp, 62 and 49 %.
// us forward with counts and loss / backward, floor by bytes: 4096 x 256 bf16 11.7 / 6.3 (0.4, 0.7), 65003 x 64 fp32 34 / 19 (3, 6), 65536 x 256 fp32
// 70 / 45 (11, 21); 16 x 256 with a bias 5.9.  A token's row is asked for one token ahead (65536 x 256 fp32 backward 62 -> 47).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/hcomm_moe.h"
#include "../core/log.h"
#include "../core/per_device.h"
#include "gemm_sm100_2sm.cuh"
#include "sm100_ptx.cuh"

namespace {

constexpr int kMaxExperts = 1024, kMaxTopk = 16;
constexpr int kMostTokens = INT32_MAX - 32;      // rounded up to a block's tokens still a 32-bit number
constexpr uint32_t kAll = 0xffffffffu;
constexpr int kFinishThreads = 1024, kFinishCtas = 8;

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

// This lane's V values of a row as they lie in memory, asked for one token ahead of their use.
template <typename T, int V> struct __align__(16) Raw { T v[V]; };
template <typename T, int V> __device__ __forceinline__ void AskRow(Raw<T, V> &raw, const T *row, int experts, int first, bool vectors)
{
    constexpr int kBytes = V * (int)sizeof(T), kWord = kBytes > 16 ? 16 : kBytes;
    using W = typename Word<kWord>::type;
    if (vectors) {
        if (first < experts) {
#pragma unroll
            for (int i = 0; i < kBytes / kWord; ++i) ((W *)raw.v)[i] = ((const W *)(row + first))[i];
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (first + j < experts) raw.v[j] = row[first + j];
    }
}
// -inf behind the last expert
template <typename T, int V> __device__ __forceinline__ void TakeRow(float (&x)[V], const Raw<T, V> &raw, int experts, int first)
{
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = first + j < experts ? ToFloat(raw.v[j]) : -INFINITY;
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
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
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
// The same in the 16 bits of the type that x came from.
template <typename T> __device__ __forceinline__ uint32_t Key16(float x);
template <> __device__ __forceinline__ uint32_t Key16<__nv_bfloat16>(float x) { return Key(x) >> 16; }
template <> __device__ __forceinline__ uint32_t Key16<__half>(float x)
{
    const uint32_t b = __half_as_ushort(__float2half_rn(x + 0.f));
    return x == -INFINITY ? 0u : (b & 0x8000u ? ~b & 0xffffu : b | 0x8000u);
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

__device__ __forceinline__ float Unkey(uint32_t k) { return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu)); }
// Whether a <= b might be the other way round, see ChooseBiased.
__device__ __forceinline__ bool Close(uint32_t upper, uint32_t lower)
{
    const float a = Unkey(upper), b = Unkey(lower);
    return !(a - b > 0x1p-20f * (1.f + fabsf(a) + fabsf(b)));
}
__device__ __forceinline__ bool Close(uint64_t, uint64_t) { return false; }

// One step of the order inside a lane: the larger key first, of equal ones the one that stood in front.
template <typename K> __device__ __forceinline__ void Order(K &a, K &b, uint32_t &ia, uint32_t &ib)
{
    const bool swap = b > a;
    const K k = swap ? a : b;
    const uint32_t i = swap ? ia : ib;
    a = swap ? b : a; ia = swap ? ib : ia;
    b = k; ib = i;
}
// The k largest keys of the warp: lane i gets the i-th's expert, -1 where no candidate is left; returns the largest key.  With close
// it looks at one more and says whether two neighbours are.
// Up to eight keys a lane are put in order first (by steps that keep equal ones in place), so that a round looks at one key a lane
// and the winner moves its list up; places within the lane are four bits each of a word, which moves up with it.
template <int V, typename K> __device__ __forceinline__ K TopK(K (&key)[V], int topk, int lane, int *expert, bool *close = nullptr)
{
    constexpr bool kSorted = V <= 8;
    *expert = -1;
    K largest = 0, before = 0;
    uint32_t places = 0;
    if constexpr (kSorted) {
        uint32_t at[V];
#pragma unroll
        for (int j = 0; j < V; ++j) at[j] = j;
#pragma unroll
        for (int pass = 0; pass < V; ++pass)
#pragma unroll
            for (int j = pass & 1; j + 1 < V; j += 2) Order(key[j], key[j + 1], at[j], at[j + 1]);
#pragma unroll
        for (int j = 0; j < V; ++j) places |= at[j] << 4 * j;
    }
    const int rounds = close ? topk + 1 : topk;
    for (int i = 0; i < rounds; ++i) {
        K best = key[0];
        int at = (int)(places & 15);
        if constexpr (!kSorted) {
            at = 0;
#pragma unroll
            for (int j = 1; j < V; ++j)
                if (key[j] > best) { best = key[j]; at = j; }
        }
        const K top = WarpMaxKey(best);
        if (i == 0) largest = top;
        if (top == 0) break;
        if (close && i) *close |= Close(before, top);
        before = top;
        const int winner = __ffs(__ballot_sync(kAll, best == top)) - 1, e = __shfl_sync(kAll, lane * V + at, winner);
        if (lane == i && i < topk) *expert = e;
        if (lane == winner) {
            if constexpr (kSorted) {
#pragma unroll
                for (int j = 0; j + 1 < V; ++j) key[j] = key[j + 1];
                key[V - 1] = 0;
                places >>= 4;
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (j == at) key[j] = 0;
            }
        }
    }
    return largest;
}
// The same of 16-bit keys, which share a word with the expert (the lower one is the larger word): no two words are equal, so that one
// maximum says who it is.  (4096 tokens of 256 experts, bf16, choice alone: 10.0 us with keys of 32 bits, 9.6 so; 65536 of 128 experts 31 and 28.)
template <int V> __device__ __forceinline__ uint32_t TopKPacked(uint32_t (&word)[V], int topk, int lane, int *expert)
{
    *expert = -1;
    uint32_t largest = 0;
    if constexpr (V <= 8) {
#pragma unroll
        for (int pass = 0; pass < V; ++pass)
#pragma unroll
            for (int j = pass & 1; j + 1 < V; j += 2) {
                const uint32_t a = max(word[j], word[j + 1]), b = min(word[j], word[j + 1]);
                word[j] = a; word[j + 1] = b;
            }
    }
    for (int i = 0; i < topk; ++i) {
        uint32_t best = word[0];
        if constexpr (V > 8) {
#pragma unroll
            for (int j = 1; j < V; ++j) best = max(best, word[j]);
        }
        const uint32_t top = __reduce_max_sync(kAll, best);
        if (i == 0) largest = top >> 16;
        if (top >> 16 == 0) break;
        if (lane == i) *expert = 0xffff - (int)(top & 0xffff);
        if (best == top) {
            if constexpr (V <= 8) {
#pragma unroll
                for (int j = 0; j + 1 < V; ++j) word[j] = word[j + 1];
                word[V - 1] = 0;
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (word[j] == top) word[j] = 0;
            }
        }
    }
    return largest;
}

// The row as probabilities: x becomes p.  Logarithm of the largest score and 1 / sum, for a single score's own.
template <int V> __device__ __forceinline__ float2 Softmax(float (&x)[V], bool sigmoid)
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
    return {top, inverse};
}

// A row without a defined softmax (or sum of sigmoids): it holds a NaN, or +inf under softmax.
template <int V> __device__ __forceinline__ bool Undefined(const float (&x)[V], bool sigmoid)
{
    bool bad = false;
#pragma unroll
    for (int j = 0; j < V; ++j) bad |= x[j] != x[j] || (!sigmoid && x[j] == INFINITY);
    return __any_sync(kAll, bad);
}

// The choice by sigmoid(x) + bias; true where a value is no number.  A choice between two scores that 32 bits cannot tell apart must not
// hang on the way they were rounded, so it is made in 64 bits - but only for rows that need it, since an exponential in 64 bits costs as much as
// everything else (65536 tokens, 256 experts: 124 us with all rows, 87 so).  In 32 bits a score is off by less than 2^-22, and by 2^-24 of the
// sum with its bias: a row whose k + 1 best lie further apart than twice that has its order.
template <int V> __device__ __forceinline__ bool ChooseBiased(const float (&x)[V], const Params &p, int first, int lane, int *expert)
{
    uint32_t quick[V];
    float bias[V];
    bool none = false, close = false;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        bias[j] = p.bias[first + j < p.experts ? first + j : 0];
        const float s = x[j] == -INFINITY ? -INFINITY : 1.f / (1.f + expf(-x[j])) + bias[j];
        none |= s != s;
        quick[j] = Key(s);
    }
    if (__any_sync(kAll, none)) return true;
    TopK<V, uint32_t>(quick, p.topk, lane, expert, &close);
    if (!close) return false;
    uint64_t key[V];
#pragma unroll
    for (int j = 0; j < V; ++j) key[j] = Key(x[j] == -INFINITY ? (double)-INFINITY : 1.0 / (1.0 + exp(-(double)x[j])) + (double)bias[j]);
    TopK<V, uint64_t>(key, p.topk, lane, expert);
    return false;
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

__device__ __forceinline__ float Loss(const Params &p, float products, float tokens) { return p.balance * p.experts * (products / (tokens * p.topk) / tokens); }

// A single block's sums are all there is: counts, sums and loss from shared memory.
__device__ void FinishAlone(const Params &p, const float *sums, const int32_t *counts, float *warpSum)
{
    const int E = p.experts, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float products = 0;
    for (int e = threadIdx.x; e <= E; e += blockDim.x) {
        p.counts[e] = counts[e];
        if (e < E && sums) {
            if (p.sums) p.sums[e] = sums[e];
            products += (float)counts[e] * sums[e];
        }
    }
    products = WarpSum(products);
    if (lane == 0) warpSum[warp] = products;
    __syncthreads();
    if (threadIdx.x == 0 && p.loss) {
        float all = 0;
        for (int w = 0; w < (int)blockDim.x / 32; ++w) all += warpSum[w];
        *p.loss = Loss(p, all, (float)max(counts[E], 1));
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
    const int64_t step = (int64_t)gridDim.x * kWarps;
    int64_t t = (int64_t)blockIdx.x * kWarps + warp;
    Raw<T, V> next;
    bool nextCounted = false;
    auto ask = [&](int64_t t) {
        if (t >= p.tokens) return;
        AskRow<T, V>(next, (const T *)p.logits + t * p.ld, E, first, p.vectors);
        nextCounted = !p.valid || p.valid[t];
    };
    ask(t);
    for (; t < p.tokens; t += step) {
        const bool counted = nextCounted;
        float x[V];
        TakeRow<T, V>(x, next, E, first);
        ask(t + step);
        int expert = -1;
        float gate = 0;
        if (counted) {
            ++seen;
            const T *row = (const T *)p.logits + t * p.ld;
            bool bad;
            if (p.bias) bad = ChooseBiased<V>(x, p, first, lane, &expert);
            else {
                // a NaN, which an addition makes positive, has a key above that of infinity
                uint32_t key[V], largest, infinity;
                if constexpr (sizeof(T) == 2) {
#pragma unroll
                    for (int j = 0; j < V; ++j) key[j] = Key16<T>(x[j]) << 16 | (0xffff - (uint32_t)(first + j));
                    largest = TopKPacked<V>(key, p.topk, lane, &expert);
                    infinity = Key16<T>(INFINITY);
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j) key[j] = Key(x[j]);
                    largest = TopK<V, uint32_t>(key, p.topk, lane, &expert);
                    infinity = Key(INFINITY);
                }
                bad = p.sigmoid ? largest > infinity : largest >= infinity;
            }
            if (bad) expert = -1;
            const bool chosen = expert >= 0;
            const float value = chosen ? ToFloat(row[expert]) : 0.f;
            if (p.renormalize) gate = ChosenShare(value, chosen, p.sigmoid);
            else if (p.sigmoid) gate = chosen ? expf(LogSigmoid(value)) : 0.f;
            if (stats || (!p.renormalize && !p.sigmoid)) {
                const float2 s = Softmax(x, p.sigmoid);
                if (!p.renormalize && !p.sigmoid) gate = chosen ? expf(value - s.x) * s.y : 0.f;
#pragma unroll
                for (int j = 0; j < V; ++j) sum[j] += bad ? NAN : x[j];
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
        FinishAlone(p, stats ? rows : nullptr, counts, warpSum);
    }
}

// Adds up the blocks' rows of scratch (one CTA and a thread for each expert took 10 us of 23 at 4096 tokens): a cluster of eight CTAs, each with an eighth of the experts and as many groups of threads as
// there is room for, each with some of the blocks.  Every sum goes through its blocks, then its groups, then its CTAs in order.
__global__ void __launch_bounds__(kFinishThreads) FinishKernel(const __grid_constant__ Params p, int blocks)
{
    __shared__ float groupSum[kFinishThreads], products[kFinishThreads / 32], mine;
    __shared__ int32_t groupCount[kFinishThreads];
    sm100::GridDependencyWait();
    sm100::GridDependentsLaunch();
    const int E = p.experts, rank = (int)hcgemm::pair::ClusterCtaRank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int width = (E + 1 + kFinishCtas - 1) / kFinishCtas, groups = kFinishThreads / width, group = threadIdx.x / width, in = threadIdx.x % width, e = rank * width + in;
    int n = 0;
    float s = 0;
    if (group < groups && e <= E) {
#pragma unroll 8
        for (int b = group; b < blocks; b += groups) {
            n += p.partCounts[(size_t)b * (E + 1) + e];
            if (p.partSums && e < E) s += p.partSums[(size_t)b * E + e];
        }
    }
    groupCount[threadIdx.x] = n; groupSum[threadIdx.x] = s;
    __syncthreads();
    float product = 0;
    if (threadIdx.x < width && e <= E) {
        for (int g = 1; g < groups; ++g) { n += groupCount[g * width + in]; s += groupSum[g * width + in]; }
        p.counts[e] = n;
        if (e < E) {
            if (p.sums) p.sums[e] = s;
            product = (float)n * s;
        } else groupCount[0] = n;           // of tokens: the last CTA's, no other thread of which still reads its group's first entry
    }
    product = WarpSum(product);
    if (lane == 0) products[warp] = product;
    __syncthreads();
    if (threadIdx.x == 0) {
        mine = 0;
        for (int w = 0; w < kFinishThreads / 32; ++w) mine += products[w];
    }
    hcgemm::pair::ClusterSync();
    if (rank == E / width && threadIdx.x == 0 && p.loss) {
        float all = 0;
        for (int r = 0; r < kFinishCtas; ++r) {
            float v;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(hcgemm::pair::MapToCta(&mine, r)) : "memory");
            all += v;
        }
        *p.loss = Loss(p, all, (float)max(groupCount[0], 1));
    }
    hcgemm::pair::ClusterSync();            // nobody leaves while his sum is read
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
    const int64_t step = (int64_t)gridDim.x * kWarps;
    int64_t t = (int64_t)blockIdx.x * kWarps + warp;
    Raw<T, V> next;
    bool nextCounted = false;
    int nextExpert = -1;
    float nextGrad = 0;
    auto ask = [&](int64_t t) {
        if (t >= p.tokens) return;
        AskRow<T, V>(next, (const T *)p.logits + t * p.ld, E, first, p.vectors);
        nextCounted = !p.valid || p.valid[t];
        if (p.dgates && lane < p.topk) {
            nextExpert = p.idx[t * p.topk + lane];
            nextGrad = p.dgates[t * p.topk + lane];
        }
    };
    ask(t);
    for (; t < p.tokens; t += step) {
        const bool counted = nextCounted;
        int expert = nextExpert < E ? nextExpert : -1;
        const float grad = nextGrad;
        float x[V], d[V];
        TakeRow<T, V>(x, next, E, first);
        ask(t + step);
        if (!counted) {
#pragma unroll
            for (int j = 0; j < V; ++j) d[j] = 0;
        } else {
            const bool bad = Undefined(x, p.sigmoid);
            const float dg = expert >= 0 ? grad * p.scale : 0.f, value = expert >= 0 ? ToFloat(((const T *)p.logits)[t * p.ld + expert]) : 0.f;
            const bool chosen = expert >= 0;
            float to = dg;                      // to the chosen expert alone
            if (p.renormalize) {
                const float share = ChosenShare(value, chosen, p.sigmoid);
                to = share * (dg - WarpSum(share * dg));
            } else if (p.sigmoid) to = chosen ? dg * expf(LogSigmoid(value)) : 0.f;
            __syncwarp();                       // the token in front has cleared its places, by other lanes
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

template <typename Kernel, typename... Args>
HcclResult Launch(const char *what, Kernel *kernel, int grid, int cluster, int threads, int smem, void *stream, const Args &...args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e != cudaSuccess) {
        cudaGetLastError();
        HCCL_ERROR("%s launch failed: %s", what, cudaGetErrorString(e));
        return HCCL_E_RUNTIME;
    }
    return HCCL_SUCCESS;
}
constexpr int SharedBytes(int v, int experts, bool backward, bool stats)
{
    const int warps = v >= 16 ? 16 : 32;
    return backward ? warps * 32 * v * 4 : 4 * (experts + 1 + (stats ? warps * experts : 0));
}
// A kernel's limit of shared memory is the process's: it is raised once a GPU to the most that any call takes, never set to a call's own, or
// another thread's launch finds it lower than what it asks for.
template <typename T, int V, bool BACKWARD> HcclResult LaunchRows(const char *what, const Params &p, int grid, void *stream)
{
    constexpr auto kernel = BACKWARD ? RouteBackwardKernel<T, V> : RouteKernel<T, V>;
    constexpr int most = SharedBytes(V, 32 * V, BACKWARD, true);
    if constexpr (most > 48 * 1024) {
        static hc::PerDevice<bool> allowed;
        int dev = -1;
        const bool good = cudaGetDevice(&dev) == cudaSuccess && allowed.Get(dev, [](bool *v) {
            return *v = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most) == cudaSuccess;
        });
        if (!good) {
            HCCL_ERROR("%s: %d bytes of shared memory: %s", what, most, cudaGetErrorString(cudaGetLastError()));
            return HCCL_E_RUNTIME;
        }
    }
    return Launch(what, kernel, grid, 1, Threads<V>(), SharedBytes(V, p.experts, BACKWARD, p.partSums != nullptr), stream, p);
}
template <typename T, bool BACKWARD> HcclResult LaunchRows(const char *what, const Params &p, int grid, void *stream)
{
    switch (ValuesOf(p.experts)) {
#define HCOMM_CASE(V) case V: return LaunchRows<T, V, BACKWARD>(what, p, grid, stream);
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
    if ((dataType != HCCL_DATA_TYPE_FP32 && dataType != HCCL_DATA_TYPE_FP16 && dataType != HCCL_DATA_TYPE_BFP16) || tokens < 0 || tokens > kMostTokens || experts < 1 || experts > kMaxExperts || topk < 1 ||
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
    if (tokens < 0 || tokens > kMostTokens || experts < 1 || experts > kMaxExperts) return 0;
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
    if (blocks > 1) return Launch("HcommMoeRoute", FinishKernel, kFinishCtas, kFinishCtas, kFinishThreads, 0, stream, p, blocks);
    return HCCL_SUCCESS;
}

extern "C" int HcommMoeBalanceLoss(const int32_t *counts, const float *probSums, int experts, int topk, float balance, float *loss, void *stream)
{
    if (experts < 1 || experts > kMaxExperts || topk < 1 || topk > kMaxTopk) {
        RPT_ERR("EI0003", "HcommMoeBalanceLoss: %d experts (<= %d), %d of them chosen (<= %d)", experts, kMaxExperts, topk, kMaxTopk);
        return HCCL_E_PARA;
    }
    if (!counts || !probSums || !loss) return HCCL_E_PTR;
    return Launch("HcommMoeBalanceLoss", BalanceLossKernel, 1, 1, 32, 0, stream, counts, probSums, experts, topk, balance, loss);
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
