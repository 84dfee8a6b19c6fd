// fp4_gemm.cuh - products of microscaled 4-bit operands (tcgen05 kind::mxf4, block scaling), and the loop for few rows.
//
//   out[m][n] = sum over blocks b of 32 columns of  2^(sa[m][b] + sb[n][b] - 254) * sum over the block of a[m][c] b[n][c]
//
// The tensor core applies the scales: besides the operand tiles in shared memory (64 columns, 32 bytes a row and
// instruction) it wants the scale bytes in tensor memory, where row r of an operand finds the four bytes of 128 columns in lane
// r % 32, column r / 32 of each quarter - which is how the tiles of scales are laid out in memory, so that one 512-byte
// copy (tcgen05.cp, 32 lanes x 16 bytes, repeated for the four quarters) per operand, 128 rows and 128 columns puts them there.
//
// In the loop of this file the operands change places: 128 rows of B, the weights, are the instruction's M, and up to 128 rows of A,
// the tokens, its N, which is rounded up to 16 from what there is.  A product of 128 x 64 by 16 x 64 reads 4.5 KB of shared memory where
// the other way round it would read 8 KB for 128 rows of which 16 are real (one rank's 32 experts while decoding, gate and up: 83.8 us, so 81.7).
// Many rows go to the loop of fp4_gemm_pair.cuh.
//
// Warp roles:
//   warp 0      TMA producer: 256 columns a stage - rows of both operands (128-byte swizzle) and their tiles of scales
//   warp 1      issuer: copies a stage's scales to tensor memory, then four products of 64 columns; one thread
//   warps 4-11  epilogue: first the whole accumulator as bf16 into registers, which hands it back to the issuer after a few hundred
//               cycles, then out
// Each stage of the ring has its own columns for scales in tensor memory, so that the barrier that frees the stage frees them too.
//
// Rows of A may be grouped by expert, with a matrix of B for each: tiles never cross a group; what a tile holds behind its
// group's last row are other rows' values, which no stored value depends on.
//
// Where there are fewer tiles than SMs, the CTAs of a cluster share a tile along K.  Each leaves its sums in its own shared memory, where
// all of them then read: every CTA adds up some of the tokens, over the CTAs in order, and stores them.
//
// A gated product (GLU) loads 128 rows of each of two matrices and keeps two accumulators, gate and up of the same element in the
// same lane and thread, and stores silu(gate) * up.
#pragma once
#include <cuda_bf16.h>

#include "fp4.cuh"
#include "gemm_sm100_2sm.cuh"
#include "sm100_ptx.cuh"

namespace hcfp4 {
using namespace sm100;

constexpr int kStageCols = 256;             // columns of K a stage, 128 bytes
constexpr int kUmmaCols = 64;               // of an instruction
constexpr int kStoreWarps = 8;                        // of the epilogue: two for each quarter of the accumulator's rows
constexpr int kGemmThreads = 32 * (4 + kStoreWarps);

struct Maps { CUtensorMap a, sa, b[2], sb[2]; };        // b[1], sb[1]: the second matrix of a gated product, else the first again

struct Shape {
    int M, N, K;
    int tilesN;
    int group;                  // row tiles that are taken together before the next column of tiles
    int boxRows;                // rows of A that a load takes: a tile loads no more than it needs (one CTA a tile)
    int aSlot, stages;          // bytes of A in a stage; stages of the ring
    int split;                  // CTAs of a cluster that share a tile along K
    int experts;                // 0: one matrix
    const int32_t *offsets;
    int tileCols, tileRowsB;    // tiles of scales along K; along N of one matrix
    int64_t ldOut;
    __nv_bfloat16 *out;
    uint32_t *error;
};

constexpr int kMaxStages = 12, kMaxSplit = 8;
constexpr int kRoom = 224 * 1024;           // of shared memory: leaves a small block of the kernel in front its place
struct State {
    uint64_t full[kMaxStages], empty[kMaxStages], accFull[2], accEmpty[2];
    uint32_t tmem;
    volatile uint32_t abort;
};
static_assert(sizeof(State) <= 256, "barriers");

// A CTA's shared memory: the stages' rows of A, then those of B, their tiles of scales, the barriers, and with
// grouped rows where they start.  A stage of A is as large as a load of it, so that few rows leave room for more stages: one
// product after the other takes as long as a load is under way divided by the stages.  The
// tensor core reads 128 rows all the same, those behind from whatever lies there: rows of B at the worst, never behind the allocation.
template <int BN> struct Config {
    static_assert(BN == 128 || BN == 256, "one or two tiles of scales wide");
    static constexpr int kBBytes = BN * 128, kSaBytes = 2 * kTileBytes, kSbBytes = BN / 128 * 2 * kTileBytes;
    static constexpr int kAccumulators = BN == 256 ? 1 : 2;
    static constexpr int kScaleCols = 8 + BN / 128 * 8;             // of a stage, in tensor memory
    static constexpr int kScaleBase = kAccumulators * BN;
    static constexpr int kTail = 256;
    __host__ __device__ static constexpr int ASlot(int boxRows, bool grouped) { return (grouped ? 128 : boxRows) * 128; }
    static constexpr int StageBytes(int aSlot) { return aSlot + kBBytes + kSaBytes + kSbBytes; }
    static constexpr int Stages(int aSlot, int experts)
    {
        const int room = kRoom - 1024 - kTail - (experts > 0 ? 4 * (experts + 1) : 0), fit = room / StageBytes(aSlot), columns = (512 - kScaleBase) / kScaleCols;
        return fit < columns ? (fit < kMaxStages ? fit : kMaxStages) : (columns < kMaxStages ? columns : kMaxStages);
    }
    static constexpr int SmemBytes(int aSlot, int stages, int experts) { return 1024 + stages * StageBytes(aSlot) + kTail + (experts > 0 ? 4 * (experts + 1) : 0); }
};

// kind::mxf4: e2m1 x e2m1 with scales that are powers of two, both operands with K contiguous.  The fields of the scales' byte
// pairs (bits 4-5 for B, 29-30 for A) are set for each instruction: 0 for the first 64 of 128 columns, 2 for the others.
__host__ __device__ constexpr uint32_t InstrDescMxf4(uint32_t M, uint32_t N, uint32_t pair)
{
    return (pair << 4) | (1u << 7) | (1u << 10) | ((N >> 3) << 17) | (1u << 23) | ((M >> 4) << 24) | (pair << 29);
}
// Descriptors of shared memory in two words, so that the issuing thread steps through a ring with 32-bit additions: it has a few
// hundred cycles a stage for eight and more instructions and their operands (with descriptors made anew for each: 27.0 us
// for 16 x 28672 x 8192, so 24.9).  The low word has the address in units of 16 bytes; the high ones say: K contiguous, rows of 128 bytes with
// the 128-byte swizzle, 1024 bytes from eight rows to the next eight; and 32 rows of 16 bytes of scales, eight rows in 128 bytes.
constexpr uint32_t kRowsHigh = (1024 >> 4) | (1u << 14) | (2u << 29), kScalesHigh = (128 >> 4) | (1u << 14);
__device__ __forceinline__ uint32_t DescLow(const void *p) { return ((SmemAddr(p) & 0x3FFFF) >> 4) | (1u << 16); }
__device__ __forceinline__ void CopyScales(uint32_t tmem, uint32_t low)
{
    asm volatile(
        "{\n\t.reg .b64 d;\n\t"
        "mov.b64 d, {%1, %2};\n\t"
        "tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], d;\n\t}" ::"r"(tmem), "r"(low), "r"(kScalesHigh) : "memory");
}
__device__ __forceinline__ void MmaMxf4(uint32_t d, uint32_t aLow, uint32_t bLow, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "mov.b64 a, {%1, %7};\n\t"
        "mov.b64 b, {%2, %7};\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "r"(aLow), "r"(bLow), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate), "r"(kRowsHigh) : "memory");
}
__device__ __forceinline__ void TmaLoad3d(void *dst, const CUtensorMap *m, uint64_t *bar, int32_t x, int32_t y, int32_t z)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(SmemAddr(dst)), "l"(m), "r"(SmemAddr(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}

struct Tile {
    int expert, row, rows;      // first row, rows up to the end of the group (at most 128; none or fewer: nothing to store)
    int column;                 // tile along N
    int scaleTile;              // tile row of A's scales
};
// The tiles of ROWS rows that a CTA (or pair, of which `half` is the CTA) takes, t, t + step, ...: experts in order, inside an expert
// `group` row tiles by all columns of tiles, so that CTAs that run at the same time share rows of both operands in L2.
template <int ROWS> struct Tiles {
    const Shape &g;
    const int *start;           // shared memory, with grouped rows
    int half, step, t, expert = 0, before = 0, scalesBefore = 0;        // before: tiles of ROWS rows (tile rows of scales) of the experts in front
    __device__ Tiles(const Shape &s, const int *st, int first, int stride, int h) : g(s), start(st), half(h), step(stride), t(first) {}
    __device__ bool Next(Tile *out)
    {
        int firstRow = 0, endRow = g.M, rowTiles;
        if (g.experts > 0) {
            for (;; ++expert) {
                if (expert == g.experts) return false;
                firstRow = start[expert]; endRow = start[expert + 1];
                rowTiles = (endRow - firstRow + ROWS - 1) / ROWS;
                if (t < (before + rowTiles) * g.tilesN) break;
                before += rowTiles;
                scalesBefore += (endRow - firstRow + kTileRows - 1) / kTileRows;
            }
        } else {
            rowTiles = (endRow + ROWS - 1) / ROWS;
            if (t >= rowTiles * g.tilesN) return false;
        }
        const int local = t - before * g.tilesN, perGroup = g.group * g.tilesN, group = local / perGroup, in = local - group * perGroup;
        const int wide = min(g.group, rowTiles - group * g.group);
        const int column = in / wide, r = group * g.group + in - column * wide;
        out->expert = expert; out->column = column; out->scaleTile = scalesBefore + r * (ROWS / kTileRows) + half;
        out->row = firstRow + r * ROWS + half * 128; out->rows = min(128, endRow - out->row);
        t += step;
        return true;
    }
};

__device__ __forceinline__ uint32_t Bf16Pair(float a, float b)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *(const uint32_t *)&h;
}
// The quick quotient is off by two units of 2^-23, and 0 where exp(-g) is beyond 2^126 (g below -87.3), where silu's magnitude is below 2^-119.
// An exact one calls a subroutine where a lane's operand is out of the ordinary: 60 us a tile, measured.
__device__ __forceinline__ float SiluTimes(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }

// A warp's part of a finished accumulator, the operands in each other's places: lane l has row 32 q + l of the weights, columns are
// tokens, 64 of them the warp's.  handBack is called once they are in registers; two lanes exchange every other value, so that each
// stores two neighbours.
template <bool GLU, typename HandBack>
__device__ __forceinline__ void StoreTokens(const Shape &g, const Tile &t, uint32_t accumulator, int warp, int lane, bool pairs, HandBack handBack)
{
    const int q = warp & 3, first = (warp >> 2) * 64, tokens = t.rows - first, n = t.column * 128 + q * 32 + lane;
    uint32_t packed[32];            // two tokens each
#pragma unroll
    for (int c = 0; c < 64; c += 32) {
        if (tokens > c) {
            uint32_t v[32];
            const uint32_t from = accumulator + ((uint32_t)(q * 32) << 16) + first + c;
            TmemLoad32x32(from, v);
            if constexpr (GLU) {
                uint32_t u[32];
                TmemLoad32x32(from + 128, u);
                TmemLoadWait();
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    packed[c / 2 + j] = Bf16Pair(SiluTimes(__uint_as_float(v[2 * j]), __uint_as_float(u[2 * j])), SiluTimes(__uint_as_float(v[2 * j + 1]), __uint_as_float(u[2 * j + 1])));
            } else {
                TmemLoadWait();
#pragma unroll
                for (int j = 0; j < 16; ++j) packed[c / 2 + j] = Bf16Pair(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
            }
        }
    }
    TcFenceBefore();
    __syncwarp();
    if (lane == 0) handBack();
    __nv_bfloat16 *out = g.out + (int64_t)(t.row + first) * g.ldOut;
    if (pairs) {
        // the even lane stores token 2 j for both, the odd one token 2 j + 1: an exchange, a selection, a store and a step (with addresses
        // and the matrix's edge worked out in the loop 2048 x 4096 x 1024 took 15.6 us, so 11.5)
        char *at = (char *)(out + (lane & 1) * g.ldOut + (n & ~1));
        const int64_t step = 4 * g.ldOut;           // bytes of two rows
        const uint32_t take = lane & 1 ? 0x3276 : 0x5410;
        const int mine = tokens - (lane & 1), both = (n | 1) < g.N ? mine : 0, last = (n | 1) == g.N ? mine : 0;       // last: a column without a neighbour
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            if (2 * j >= tokens) break;
            const uint32_t v = __byte_perm(packed[j], __shfl_xor_sync(0xffffffffu, packed[j], 1), take);
            if (2 * j < both) *(uint32_t *)at = v;
            if (2 * j < last) *(uint16_t *)at = (uint16_t)v;
            at += step;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            if (2 * j >= tokens) break;
            if (n >= g.N) continue;
            const __nv_bfloat162 both = *(const __nv_bfloat162 *)&packed[j];
            out[(int64_t)(2 * j) * g.ldOut + n] = both.x;
            if (2 * j + 1 < tokens) out[(int64_t)(2 * j + 1) * g.ldOut + n] = both.y;
        }
    }
}

// Of a shared tile: the CTA's sums to shared memory, [gate, up][token][128 rows of weights] in 32 bits.
template <bool GLU> __device__ __forceinline__ void KeepSums(const Tile &t, uint32_t accumulator, int warp, int lane, float *sums)
{
    const int q = warp & 3, first = (warp >> 2) * 64, tokens = t.rows - first;
#pragma unroll
    for (int h = 0; h < (GLU ? 2 : 1); ++h)
#pragma unroll
        for (int c = 0; c < 64; c += 32) {
            if (tokens <= c) break;
            uint32_t v[32];
            TmemLoad32x32(accumulator + ((uint32_t)(q * 32) << 16) + h * 128 + first + c, v);
            TmemLoadWait();
            float *to = sums + ((h * 128 + first + c) * 128 + q * 32 + lane);
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (c + j < tokens) to[j * 128] = __uint_as_float(v[j]);
        }
}
__device__ __forceinline__ float2 LoadCluster(const float *p, int rank)
{
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(hcgemm::pair::MapToCta(p, rank)) : "memory");
    return v;
}
// All threads of all CTAs of the cluster, after everyone's sums are there.
template <bool GLU> __device__ __forceinline__ void AddSums(const Shape &g, const Tile &t, const float *sums, int rank, bool pairs)
{
    const int n = (threadIdx.x & 63) * 2, column = t.column * 128 + n;
    if (column >= g.N) return;
    for (int token = rank + (threadIdx.x >> 6) * g.split; token < t.rows; token += kGemmThreads / 64 * g.split) {
        float2 a[kMaxSplit], b[kMaxSplit];          // asked for all at once
#pragma unroll
        for (int r = 0; r < kMaxSplit; ++r) {
            a[r] = b[r] = {0, 0};
            if (r >= g.split) continue;
            a[r] = LoadCluster(sums + token * 128 + n, r);
            if constexpr (GLU) b[r] = LoadCluster(sums + (128 + token) * 128 + n, r);
        }
        float2 v = a[0], u = b[0];
#pragma unroll
        for (int r = 1; r < kMaxSplit; ++r) {
            v.x += a[r].x; v.y += a[r].y;
            if constexpr (GLU) { u.x += b[r].x; u.y += b[r].y; }
        }
        if constexpr (GLU) { v.x = SiluTimes(v.x, u.x); v.y = SiluTimes(v.y, u.y); }
        __nv_bfloat16 *at = g.out + (int64_t)(t.row + token) * g.ldOut + column;
        if (pairs && column + 1 < g.N) *(uint32_t *)at = Bf16Pair(v.x, v.y);
        else {
            at[0] = __float2bfloat16_rn(v.x);
            if (column + 1 < g.N) at[1] = __float2bfloat16_rn(v.y);
        }
    }
}

template <bool GLU> __device__ __forceinline__ void GemmLoop(const Maps *maps, const Shape &g)
{
    constexpr int BN = GLU ? 256 : 128;         // rows of weights: gate and up take 128 each
    using Cfg = Config<BN>;
    extern __shared__ uint8_t smemRaw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)smemRaw + 1023) & ~(uintptr_t)1023);
    const int ring = g.stages;
    uint8_t *const ringB = smem + ring * g.aSlot, *const ringSa = ringB + ring * Cfg::kBBytes, *const ringSb = ringSa + ring * Cfg::kSaBytes;
    State *st = (State *)(ringSb + ring * Cfg::kSbBytes);
    int *start = (int *)((uint8_t *)st + 256);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // a shared tile is the only one of its cluster
    const int rank = g.split > 1 ? (int)hcgemm::pair::ClusterCtaRank() : 0, firstTile = g.split > 1 ? (int)blockIdx.x / g.split : (int)blockIdx.x;
    const int tileStep = g.split > 1 ? 1 << 30 : (int)gridDim.x;
    const int allStages = (g.K + kStageCols - 1) / kStageCols, firstStage = allStages * rank / g.split, endStage = allStages * (rank + 1) / g.split;
    const bool pairs = g.ldOut % 2 == 0 && ((uintptr_t)g.out & 3) == 0;
    if (threadIdx.x == 0) {
        for (int s = 0; s < ring; ++s) { MbarInit(&st->full[s], 1); MbarInit(&st->empty[s], 1); }
        for (int a = 0; a < 2; ++a) { MbarInit(&st->accFull[a], 1); MbarInit(&st->accEmpty[a], kStoreWarps); }
        st->abort = 0;
        MbarFenceInit();
        TmaPrefetchDescriptor(&maps->a); TmaPrefetchDescriptor(&maps->b[0]);
    }
    if (warp == 1) {
        TmemAlloc(&st->tmem, 512);
        TmemRelinquish();
    }
    if (g.experts > 0 && warp == 2) {
        GridDependencyWait();
        BuildGroups(g.offsets, g.experts, g.M, start, nullptr);
    }
    TcFenceBefore();
    __syncthreads();
    TcFenceAfter();
    const uint32_t tmem = st->tmem;
    GridDependentsLaunch();

    if (warp == 0) {
        // ------------------------------------------------------------------------------- TMA producer
        if (ElectOne()) {
            GridDependencyWait();
            int s = 0;
            uint32_t phase = 0;         // of the ring: flips each time round
            bool alive = true;
            Tiles<128> tiles(g, start, firstTile, tileStep, 0);
            Tile t;
            while (alive && tiles.Next(&t)) {
                const int n = t.column * 128;
                const int boxes = (t.rows + g.boxRows - 1) / g.boxRows, bytes = Cfg::StageBytes(boxes * g.boxRows * 128);
                for (int k = firstStage; k < endStage; ++k) {
                    if (!MbarWait(&st->empty[s], phase ^ 1, &st->abort)) { alive = false; break; }
                    uint8_t *a = smem + s * g.aSlot, *b = ringB + s * Cfg::kBBytes, *sa = ringSa + s * Cfg::kSaBytes, *sb = ringSb + s * Cfg::kSbBytes;
                    MbarExpectTx(&st->full[s], bytes);
                    // as many coordinates as the map has dimensions; rows that are not loaded hold what was there, and are not stored
                    for (int r = 0; r < boxes; ++r) TmaLoad3d(a + r * g.boxRows * 128, &maps->a, &st->full[s], k * 128, t.row + r * g.boxRows, 0);
                    TmaLoad2d(sa, &maps->sa, &st->full[s], 0, t.scaleTile * g.tileCols + 2 * k);
#pragma unroll
                    for (int h = 0; h < BN / 128; ++h) {
                        TmaLoad3d(b + h * 16384, &maps->b[h], &st->full[s], k * 128, n, t.expert);
                        TmaLoad2d(sb + h * 2 * kTileBytes, &maps->sb[h], &st->full[s], 0, (t.expert * g.tileRowsB + t.column) * g.tileCols + 2 * k);
                    }
                    if (++s == ring) { s = 0; phase ^= 1; }
                }
            }
            if (!alive) __nanosleep(500000);        // copies under way still write here: they end long before this does
        }
    } else if (warp == 1) {
        // -------------------------------------------------------------------------------------- issuer
        if (ElectOne()) {
            GridDependencyWait();
            int s = 0;
            uint32_t phase = 0, i = 0;
            const uint32_t lowA = DescLow(smem), lowB = DescLow(ringB), lowSa = DescLow(ringSa), lowSb = DescLow(ringSb);
            bool alive = true;
            Tiles<128> tiles(g, start, firstTile, tileStep, 0);
            Tile t;
            while (alive && tiles.Next(&t)) {
                const uint32_t acc = i % Cfg::kAccumulators, accPhase = (i / Cfg::kAccumulators) & 1;
                ++i;
                if (!MbarWait(&st->accEmpty[acc], accPhase ^ 1, &st->abort)) { alive = false; break; }
                TcFenceAfter();
                const uint32_t d = tmem + acc * BN, tokens = (uint32_t)(t.rows + 15) / 16 * 16;
                const uint32_t idesc[2] = {InstrDescMxf4(128, tokens, 0), InstrDescMxf4(128, tokens, 2)};
                uint32_t more = 0;
                for (int k = firstStage; k < endStage; ++k) {
                    if (!MbarWait(&st->full[s], phase, &st->abort)) { alive = false; break; }
                    TcFenceAfter();
                    const uint32_t a = lowA + s * (g.aSlot >> 4), b = lowB + s * (Cfg::kBBytes >> 4), sa = lowSa + s * (Cfg::kSaBytes >> 4), sb = lowSb + s * (Cfg::kSbBytes >> 4);
                    const uint32_t ta = tmem + Cfg::kScaleBase + s * Cfg::kScaleCols, tb = ta + 8;
                    const int left = g.K - k * kStageCols;
                    // scales of A: columns 0-3 the first 128 of K, 4-7 the second; of B likewise, with four more for each 128 rows
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        if (c * kTileCols >= left) break;
                        CopyScales(ta + c * 4, sa + c * (kTileBytes >> 4));
#pragma unroll
                        for (int h = 0; h < BN / 128; ++h) CopyScales(tb + c * (BN / 32) + h * 4, sb + (h * 2 + c) * (kTileBytes >> 4));
                    }
#pragma unroll
                    for (int u = 0; u < kStageCols / kUmmaCols; ++u) {
                        if (u * kUmmaCols >= left) break;
#pragma unroll
                        for (int h = 0; h < BN / 128; ++h)
                            MmaMxf4(d + h * 128, b + h * (16384 >> 4) + u * 2, a + u * 2, idesc[u & 1], tb + (u >> 1) * (BN / 32) + h * 4, ta + (u >> 1) * 4, more);
                        more = 1;
                    }
                    MmaCommit(&st->empty[s]);
                    if (++s == ring) { s = 0; phase ^= 1; }
                }
                if (alive) MmaCommit(&st->accFull[acc]);
            }
        }
    } else if (warp >= 4) {
        // ------------------------------------------------------------------------------------ epilogue
        GridDependencyWait();
        uint32_t i = 0;
        Tiles<128> tiles(g, start, firstTile, tileStep, 0);
        Tile t;
        while (tiles.Next(&t)) {
            const uint32_t acc = i % Cfg::kAccumulators, phase = (i / Cfg::kAccumulators) & 1;
            ++i;
            if (!MbarWait(&st->accFull[acc], phase, &st->abort)) break;
            __syncwarp();
            TcFenceAfter();
            if (g.split > 1) KeepSums<GLU>(t, tmem, warp - 4, lane, (float *)smem);
            else StoreTokens<GLU>(g, t, tmem + acc * BN, warp - 4, lane, pairs, [&] { MbarArrive(&st->accEmpty[acc]); });
        }
    }
    // ---------------------------------------------------------------------------------------- the end
    TcFenceBefore();
    __syncthreads();
    TcFenceAfter();
    if (g.split > 1) {
        hcgemm::pair::ClusterSync();
        GridDependencyWait();
        Tile t;
        if (Tiles<128>(g, start, firstTile, tileStep, 0).Next(&t)) AddSums<GLU>(g, t, (const float *)smem, rank, pairs);
        hcgemm::pair::ClusterSync();            // nobody leaves while his sums are read
    }
    if (warp == 1) TmemDealloc(tmem, 512);
    if (threadIdx.x == 0 && st->abort) atomicExch(g.error, 1u);
}

}  // namespace hcfp4
