// fp4_gemm.cuh - persistent main loop of products of microscaled 4-bit operands (tcgen05 kind::mxf4, block scaling).
//
//   D[m][n] = sum over blocks b of 32 columns of  2^(sa[m][b] + sb[n][b] - 254) * sum over the block of a[m][c] b[n][c]
//
// The tensor core applies the scales: besides the operand tiles in shared memory (64 columns, 32 bytes a row and
// instruction) it wants the scale bytes in tensor memory, where row r of an operand finds the four bytes of 128 columns in lane
// r % 32, column r / 32 of each quarter - which is how the tiles of scales are laid out in memory, so that one 512-byte
// copy (tcgen05.cp, 32 lanes x 16 bytes, repeated for the four quarters) per operand, 128 rows and 128 columns puts them there.
//
// Warp roles:
//   warp 0      TMA producer: 256 columns a stage - rows of A and B (128-byte swizzle) and their tiles of scales
//   warp 1      issuer: copies a stage's scales to tensor memory, then four products of 64 columns; one thread
//   warps 4-11  epilogue: first the whole accumulator as bf16 into registers, which hands it back to the issuer after a few hundred
//               cycles, then through shared memory out in whole segments of the result's rows
// Each stage of the ring has its own columns for scales in tensor memory, so that the barrier that frees the stage frees them too.
//
// Rows of A may be grouped by expert, with a matrix of B for each: tiles never cross a group; what a tile loads behind its
// group's last row are other rows' values, which no stored row depends on.
//
// A gated product (GLU) loads 128 rows of each of two matrices instead of 256 of one; its epilogue has gate and up of the same
// column in one thread and stores silu(gate) * up.
#pragma once
#include <cuda_bf16.h>

#include "fp4.cuh"
#include "sm100_ptx.cuh"

namespace hcfp4 {
using namespace sm100;

constexpr int kStageCols = 256;             // columns of K a stage, 128 bytes
constexpr int kUmmaCols = 64;               // of an instruction
constexpr int kStoreWarps = 8;                        // of the epilogue: two for each quarter of the accumulator's rows
constexpr int kGemmThreads = 32 * (4 + kStoreWarps);
constexpr int kSlabCols = 32;               // columns that an epilogue warp stages at a time
constexpr int kSlabBytes = 32 * kSlabCols * 2;

struct Maps { CUtensorMap a, sa, b[2], sb[2]; };        // b[1], sb[1]: the second matrix of a gated product, else the first again

struct Shape {
    int M, N, K;
    int tilesN;
    int group;                  // row tiles that are taken together before the next column of tiles
    int boxRows;                // rows of A that a load takes: a tile loads no more than it needs (one CTA a tile)
    int experts;                // 0: one matrix
    const int32_t *offsets;
    int tileCols, tileRowsB;    // tiles of scales along K; along N of one matrix
    int64_t ldOut;
    __nv_bfloat16 *out;
    uint32_t *error;
};

template <int BN> struct Config {
    static_assert(BN == 128 || BN == 256, "one or two tiles of scales wide");
    static constexpr int kABytes = 128 * 128, kBBytes = BN * 128;
    static constexpr int kSaBytes = 2 * kTileBytes, kSbBytes = BN / 128 * 2 * kTileBytes;
    static constexpr int kStageBytes = kABytes + kBBytes + kSaBytes + kSbBytes;
    static constexpr int kStages = BN == 256 ? 4 : 6;
    static constexpr int kAccumulators = BN == 256 ? 1 : 2;
    static constexpr int kScaleCols = 8 + BN / 128 * 8;             // of a stage, in tensor memory
    static constexpr int kScaleBase = kAccumulators * BN;
    static_assert(kScaleBase + kStages * kScaleCols <= 512, "tensor memory");
};

struct State {
    uint64_t full[8], empty[8], accFull[2], accEmpty[2];
    uint32_t tmem;
    volatile uint32_t abort;
};
// Behind the ring: the epilogue's slabs, the barriers, and with grouped rows where they start.
template <int BN> constexpr int SmemBytes(int experts)
{
    return 1024 + Config<BN>::kStages * Config<BN>::kStageBytes + kStoreWarps * kSlabBytes + 256 + (experts > 0 ? 4 * (experts + 1) : 0);
}

// kind::mxf4: e2m1 x e2m1 with scales that are powers of two, both operands with K contiguous.  The fields of the scales' byte
// pairs (bits 4-5 for B, 29-30 for A) are set for each instruction: 0 for the first 64 of 128 columns, 2 for the others.
__host__ __device__ constexpr uint32_t InstrDescMxf4(uint32_t M, uint32_t N, uint32_t pair)
{
    return (pair << 4) | (1u << 7) | (1u << 10) | ((N >> 3) << 17) | (1u << 23) | ((M >> 4) << 24) | (pair << 29);
}
// 32 rows of 16 bytes, no swizzle: groups of eight rows 128 bytes apart.
__device__ __forceinline__ uint64_t ScaleDesc(const void *tile)
{
    return (uint64_t)((SmemAddr(tile) & 0x3FFFF) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}
__device__ __forceinline__ void CopyScales(uint32_t tmem, uint64_t desc)
{
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
__device__ __forceinline__ void MmaMxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, bool accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate ? 1u : 0u) : "memory");
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
// The quick quotient is off by two units of 2^-23 and 0 where exp(-g) is beyond 2^126, as the result then is to any type's smallest
// value.  An exact one calls a subroutine where a lane's operand is out of the ordinary: 60 us a tile, measured.
__device__ __forceinline__ float SiluTimes(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }

// 32 rows x 32 columns of a warp leave through its slab: four lanes write a row's 64 bytes.  Pieces of 16 bytes are exchanged by
// the row so that neither side meets bank conflicts beyond those of the width.
__device__ __forceinline__ void StoreSlab(uint8_t *slab, const uint32_t (&packed)[16], int lane, int rows, __nv_bfloat16 *out, int64_t ld, int cols, bool wide)
{
#pragma unroll
    for (int v = 0; v < 4; ++v)
        *(uint4 *)(slab + lane * 64 + ((v ^ ((lane >> 1) & 3)) << 4)) = make_uint4(packed[4 * v], packed[4 * v + 1], packed[4 * v + 2], packed[4 * v + 3]);
    __syncwarp();
    const int piece = lane & 3;
#pragma unroll
    for (int it = 0; it < 4; ++it) {
        const int row = it * 8 + (lane >> 2);
        if (row >= rows) continue;
        const uint4 v = *(const uint4 *)(slab + row * 64 + ((piece ^ ((row >> 1) & 3)) << 4));
        __nv_bfloat16 *at = out + (int64_t)row * ld + piece * 8;
        if (wide && piece * 8 + 8 <= cols) *(uint4 *)at = v;
        else
            for (int i = 0; i < 8 && piece * 8 + i < cols; ++i) at[i] = ((const __nv_bfloat16 *)&v)[i];
    }
    __syncwarp();
}

// A warp's 32 rows and half of the columns of a finished accumulator.  handBack is called once they are in registers: the next
// tile's products start while these are on their way out (8192 x 28672 x 8192 by pairs of CTAs: BEFORE us with it at the end, AFTER so).
template <int BN, bool GLU, typename HandBack>
__device__ __forceinline__ void StoreTile(const Shape &g, const Tile &t, uint32_t accumulator, int warp, int lane, uint8_t *slab, bool wide, HandBack handBack)
{
    constexpr int kOut = GLU ? BN / 2 : BN, kMine = kOut / 2, kSlabs = kMine / kSlabCols;
    const int q = warp & 3, first = (warp >> 2) * kMine;
    const int rows = t.rows - q * 32, cols = g.N - t.column * kOut - first;
    uint32_t packed[kSlabs][16];
    if (rows > 0) {
        const uint32_t from = accumulator + ((uint32_t)(q * 32) << 16) + first;
#pragma unroll
        for (int c = 0; c < kSlabs; ++c) {
            uint32_t v[32];
            TmemLoad32x32(from + c * kSlabCols, v);
            if constexpr (GLU) {
                uint32_t u[32];
                TmemLoad32x32(from + kOut + c * kSlabCols, u);
                TmemLoadWait();
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    packed[c][j] = Bf16Pair(SiluTimes(__uint_as_float(v[2 * j]), __uint_as_float(u[2 * j])), SiluTimes(__uint_as_float(v[2 * j + 1]), __uint_as_float(u[2 * j + 1])));
            } else {
                TmemLoadWait();
#pragma unroll
                for (int j = 0; j < 16; ++j) packed[c][j] = Bf16Pair(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
            }
        }
    }
    TcFenceBefore();
    __syncwarp();
    if (lane == 0) handBack();
    if (rows > 0) {
        __nv_bfloat16 *out = g.out + (int64_t)(t.row + q * 32) * g.ldOut + t.column * kOut + first;
#pragma unroll
        for (int c = 0; c < kSlabs; ++c)
            if (c * kSlabCols < cols) StoreSlab(slab, packed[c], lane, rows, out + c * kSlabCols, g.ldOut, cols - c * kSlabCols, wide);
    }
}

static_assert(SmemBytes<128>(kMaxExperts) <= 227 * 1024 && SmemBytes<256>(kMaxExperts) <= 227 * 1024, "shared memory");

template <int BN, bool GLU>
__device__ __forceinline__ void GemmLoop(const Maps *maps, const Shape &g)
{
    using Cfg = Config<BN>;
    static_assert(!GLU || BN == 256, "gate and up take 128 rows each");
    extern __shared__ uint8_t smemRaw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)smemRaw + 1023) & ~(uintptr_t)1023);
    uint8_t *slabs = smem + Cfg::kStages * Cfg::kStageBytes;
    State *st = (State *)(slabs + kStoreWarps * kSlabBytes);
    static_assert(sizeof(State) <= 256, "barriers");
    int *start = (int *)((uint8_t *)st + 256);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int stages = (g.K + kStageCols - 1) / kStageCols;
    if (threadIdx.x == 0) {
        for (int s = 0; s < Cfg::kStages; ++s) { MbarInit(&st->full[s], 1); MbarInit(&st->empty[s], 1); }
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
            uint32_t it = 0;
            bool alive = true;
            Tiles<128> tiles(g, start, blockIdx.x, gridDim.x, 0);
            Tile t;
            while (alive && tiles.Next(&t)) {
                const int n = t.column * (GLU ? 128 : BN);
                const int boxes = (t.rows + g.boxRows - 1) / g.boxRows, bytes = Cfg::kStageBytes - Cfg::kABytes + boxes * g.boxRows * 128;
                for (int k = 0; k < stages; ++k, ++it) {
                    const int s = it % Cfg::kStages;
                    if (!MbarWait(&st->empty[s], ((it / Cfg::kStages) & 1) ^ 1, &st->abort)) { alive = false; break; }
                    uint8_t *a = smem + s * Cfg::kStageBytes, *b = a + Cfg::kABytes, *sa = b + Cfg::kBBytes, *sb = sa + Cfg::kSaBytes;
                    MbarExpectTx(&st->full[s], bytes);
                    // as many coordinates as the map has dimensions; rows that are not loaded hold what was there, and are not stored
                    for (int r = 0; r < boxes; ++r) TmaLoad3d(a + r * g.boxRows * 128, &maps->a, &st->full[s], k * 128, t.row + r * g.boxRows, 0);
                    TmaLoad2d(sa, &maps->sa, &st->full[s], 0, t.scaleTile * g.tileCols + 2 * k);
#pragma unroll
                    for (int h = 0; h < BN / 128; ++h) {
                        const int which = GLU ? h : 0, row = GLU ? n : n + h * 128;
                        TmaLoad3d(b + h * 16384, &maps->b[which], &st->full[s], k * 128, row, t.expert);
                        TmaLoad2d(sb + h * 2 * kTileBytes, &maps->sb[which], &st->full[s], 0, (t.expert * g.tileRowsB + row / 128) * g.tileCols + 2 * k);
                    }
                }
            }
            if (!alive) __nanosleep(500000);        // copies under way still write here: they end long before this does
        }
    } else if (warp == 1) {
        // -------------------------------------------------------------------------------------- issuer
        if (ElectOne()) {
            GridDependencyWait();
            uint32_t it = 0, i = 0;
            bool alive = true;
            Tiles<128> tiles(g, start, blockIdx.x, gridDim.x, 0);
            Tile t;
            while (alive && tiles.Next(&t)) {
                const uint32_t acc = i % Cfg::kAccumulators, phase = (i / Cfg::kAccumulators) & 1;
                ++i;
                if (!MbarWait(&st->accEmpty[acc], phase ^ 1, &st->abort)) { alive = false; break; }
                TcFenceAfter();
                const uint32_t d = tmem + acc * BN;
                for (int k = 0; k < stages; ++k, ++it) {
                    const int s = it % Cfg::kStages;
                    if (!MbarWait(&st->full[s], (it / Cfg::kStages) & 1, &st->abort)) { alive = false; break; }
                    TcFenceAfter();
                    uint8_t *a = smem + s * Cfg::kStageBytes, *b = a + Cfg::kABytes, *sa = b + Cfg::kBBytes, *sb = sa + Cfg::kSaBytes;
                    const uint32_t ta = tmem + Cfg::kScaleBase + s * Cfg::kScaleCols, tb = ta + 8;
                    const int left = g.K - k * kStageCols;
                    // scales of A: columns 0-3 the first 128 of K, 4-7 the second; of B likewise, with four more for each 128 rows
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        if (c * kTileCols >= left) break;
                        CopyScales(ta + c * 4, ScaleDesc(sa + c * kTileBytes));
#pragma unroll
                        for (int h = 0; h < BN / 128; ++h) CopyScales(tb + c * (BN / 32) + h * 4, ScaleDesc(sb + (h * 2 + c) * kTileBytes));
                    }
                    const uint64_t da = SmemDescKMajorSw128(a), db = SmemDescKMajorSw128(b);
#pragma unroll
                    for (int u = 0; u < kStageCols / kUmmaCols; ++u) {
                        if (u * kUmmaCols >= left) break;
                        MmaMxf4(d, da + u * 2, db + u * 2, InstrDescMxf4(128, BN, (u & 1) * 2), ta + (u >> 1) * 4, tb + (u >> 1) * (BN / 32), (k | u) != 0);
                    }
                    MmaCommit(&st->empty[s]);
                }
                if (alive) MmaCommit(&st->accFull[acc]);
            }
        }
    } else if (warp >= 4) {
        // ------------------------------------------------------------------------------------ epilogue
        GridDependencyWait();
        uint8_t *slab = slabs + (warp - 4) * kSlabBytes;
        const bool wide = g.ldOut % 8 == 0 && ((uintptr_t)g.out & 15) == 0;
        uint32_t i = 0;
        Tiles<128> tiles(g, start, blockIdx.x, gridDim.x, 0);
        Tile t;
        while (tiles.Next(&t)) {
            const uint32_t acc = i % Cfg::kAccumulators, phase = (i / Cfg::kAccumulators) & 1;
            ++i;
            if (!MbarWait(&st->accFull[acc], phase, &st->abort)) break;
            __syncwarp();
            TcFenceAfter();
            StoreTile<BN, GLU>(g, t, tmem + acc * BN, warp - 4, lane, slab, wide, [&] { MbarArrive(&st->accEmpty[acc]); });
        }
    }
    // ---------------------------------------------------------------------------------------- the end
    TcFenceBefore();
    __syncthreads();
    TcFenceAfter();
    if (warp == 1) TmemDealloc(tmem, 512);
    if (threadIdx.x == 0 && st->abort) atomicExch(g.error, 1u);
}

}  // namespace hcfp4
