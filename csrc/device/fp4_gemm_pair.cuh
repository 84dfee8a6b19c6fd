// fp4_gemm_pair.cuh - the loop of fp4_gemm.cuh on pairs of CTAs (cta_group::2), for many rows.
//
// Two CTAs of a cluster make one tile of 256 rows x 256 columns: each loads 128 rows of A and 128 rows of B, 35 KB a stage of 512 cycles of
// the tensor cores, where a lone CTA would load 52 KB for as many products; L2 delivers some 58 bytes a cycle and SM.  The tensor core of
// each SM reads the other half of B from its neighbour's shared memory.
//
// 8192 x 28672 x 8192 takes 650 us, 5.9 PFLOP/s.  Without the copies of scales (27 cycles of the tensor pipe each, six a stage) it would be 585, with a
// quarter of the products 443: power is what bounds it, at 1.4 - 1.6 GHz.  Of shallow products (8192 x 8192 x 2048, 62 us, 4.5 PFLOP/s) the tensor cores
// are busy for 54 %, copies of scales take 15, the turn of the accumulator 25.
//   * every load of a stage completes on the leader's "full" barrier; the leader's issuer alone copies scales and multiplies,
//     for both (each CTA's scales come from its own shared memory into its own tensor memory);
//   * scales of B are wanted whole in both CTAs, so each loads all of them;
//   * a commit with a mask of both CTAs frees a stage, or publishes the accumulator, on either side.
// A gated product has gate's 128 rows in the leader and up's in the other CTA.
#pragma once
#include "fp4_gemm.cuh"

namespace hcfp4 {

constexpr int kSlabCols = 32;               // columns that an epilogue warp stages at a time
constexpr int kSlabBytes = 32 * kSlabCols * 2;

template <int STAGES> struct PairConfig {
    static constexpr int kStages = STAGES;
    static constexpr int kABytes = 128 * 128, kBBytes = 128 * 128, kSaBytes = 2 * kTileBytes, kSbBytes = 2 * 2 * kTileBytes;
    static constexpr int kStageBytes = kABytes + kBBytes + kSaBytes + kSbBytes;
    static constexpr int kScaleCols = 24, kScaleBase = 256;
    static_assert(kScaleBase + STAGES * kScaleCols <= 512, "tensor memory");
};
constexpr int kPairStages = 5;
constexpr int PairSmemBytes(int experts)
{
    return 1024 + kPairStages * PairConfig<kPairStages>::kStageBytes + kStoreWarps * kSlabBytes + 256 + (experts > 0 ? 4 * (experts + 1) : 0);
}

__device__ __forceinline__ void CopyScalesPair(uint32_t tmem, uint32_t low)
{
    asm volatile(
        "{\n\t.reg .b64 d;\n\t"
        "mov.b64 d, {%1, %2};\n\t"
        "tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], d;\n\t}" ::"r"(tmem), "r"(low), "r"(kScalesHigh) : "memory");
}
__device__ __forceinline__ void MmaMxf4Pair(uint32_t d, uint32_t aLow, uint32_t bLow, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "mov.b64 a, {%1, %7};\n\t"
        "mov.b64 b, {%2, %7};\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "r"(aLow), "r"(bLow), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate), "r"(kRowsHigh) : "memory");
}
__device__ __forceinline__ void TmaLoad3dPair(void *dst, const CUtensorMap *m, uint32_t bar, int32_t x, int32_t y, int32_t z)
{
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(SmemAddr(dst)), "l"(m), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}

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
// tile's products start while these are on their way out (8192 x 28672 x 8192: 718 us by four warps and with it at the end, 663 so).
template <bool GLU, typename HandBack>
__device__ __forceinline__ void StoreTile(const Shape &g, const Tile &t, uint32_t accumulator, int warp, int lane, uint8_t *slab, bool wide, HandBack handBack)
{
    constexpr int kOut = GLU ? 128 : 256, kMine = kOut / 2, kSlabs = kMine / kSlabCols;
    const int q = warp & 3, first = (warp >> 2) * kMine;
    const int rows = t.rows - q * 32, cols = g.N - t.column * kOut - first;
    // A gated product's 64 columns of gate and 64 of up are kept as they are, the exponentials wait until the accumulator is handed back
    // (16000 rows of 32 experts, 7168 to 2048: 230 us before, 222 so); others are rounded between the loads (145 us of those back to 7168; 147 behind them).
    uint32_t v[GLU ? 4 : 1][32], packed[kSlabs][16];
    if (rows > 0) {
        const uint32_t from = accumulator + ((uint32_t)(q * 32) << 16) + first;
        if constexpr (GLU) {
#pragma unroll
            for (int c = 0; c < 4; ++c) TmemLoad32x32(from + (c >= 2 ? kOut - 64 : 0) + c * 32, v[c]);
            TmemLoadWait();
        } else {
#pragma unroll
            for (int c = 0; c < kSlabs; ++c) {
                TmemLoad32x32(from + c * 32, v[0]);
                TmemLoadWait();
#pragma unroll
                for (int j = 0; j < 16; ++j) packed[c][j] = Bf16Pair(__uint_as_float(v[0][2 * j]), __uint_as_float(v[0][2 * j + 1]));
            }
        }
    }
    TcFenceBefore();
    __syncwarp();
    if (lane == 0) handBack();
    if (rows > 0) {
        __nv_bfloat16 *out = g.out + (int64_t)(t.row + q * 32) * g.ldOut + t.column * kOut + first;
#pragma unroll
        for (int c = 0; c < kSlabs; ++c) {
            if (c * kSlabCols >= cols) break;
            if constexpr (GLU) {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    packed[c][j] = Bf16Pair(SiluTimes(__uint_as_float(v[c][2 * j]), __uint_as_float(v[c + 2][2 * j])), SiluTimes(__uint_as_float(v[c][2 * j + 1]), __uint_as_float(v[c + 2][2 * j + 1])));
            }
            StoreSlab(slab, packed[c], lane, rows, out + c * kSlabCols, g.ldOut, cols - c * kSlabCols, wide);
        }
    }
}

template <bool GLU> __device__ __forceinline__ void GemmLoopPair(const Maps *maps, const Shape &g)
{
    using Cfg = PairConfig<kPairStages>;
    using namespace hcgemm::pair;
    extern __shared__ uint8_t smemRaw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)smemRaw + 1023) & ~(uintptr_t)1023);
    uint8_t *slabs = smem + Cfg::kStages * Cfg::kStageBytes;
    State *st = (State *)(slabs + kStoreWarps * kSlabBytes);
    int *start = (int *)((uint8_t *)st + 256);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)ClusterCtaRank(), first = (int)ClusterId(), step = (int)NumClusters();
    const bool leader = rank == 0;
    const int stages = (g.K + kStageCols - 1) / kStageCols;
    if (threadIdx.x == 0) {
        for (int s = 0; s < Cfg::kStages; ++s) { MbarInit(&st->full[s], 1); MbarInit(&st->empty[s], 1); }
        MbarInit(&st->accFull[0], 1); MbarInit(&st->accEmpty[0], 2 * kStoreWarps);          // the epilogue warps of both CTAs
        st->abort = 0;
        MbarFenceInit();
        TmaPrefetchDescriptor(&maps->a); TmaPrefetchDescriptor(&maps->b[0]);
    }
    if (warp == 1) {
        TmemAlloc2(&st->tmem, 512);
        TmemRelinquish2();
    }
    if (g.experts > 0 && warp == 2) {
        GridDependencyWait();
        BuildGroups(g.offsets, g.experts, g.M, start, nullptr);
    }
    TcFenceBefore();
    __syncthreads();
    ClusterSync();          // the other CTA's barriers are there before anything signals them
    TcFenceAfter();
    const uint32_t tmem = st->tmem;
    GridDependentsLaunch();

    if (warp == 0) {
        // ------------------------------------------------------------------ TMA producer (both CTAs)
        if (ElectOne()) {
            GridDependencyWait();
            uint32_t it = 0;
            bool alive = true;
            Tiles<256> tiles(g, start, first, step, rank);
            Tile t;
            while (alive && tiles.Next(&t)) {
                const int n = t.column * (GLU ? 128 : 256);
                const int mine = GLU ? n : n + rank * 128;           // this CTA's rows of B
                for (int k = 0; k < stages; ++k, ++it) {
                    const int s = it % Cfg::kStages;
                    if (!MbarWait(&st->empty[s], ((it / Cfg::kStages) & 1) ^ 1, &st->abort)) { alive = false; break; }
                    uint8_t *a = smem + s * Cfg::kStageBytes, *b = a + Cfg::kABytes, *sa = b + Cfg::kBBytes, *sb = sa + Cfg::kSaBytes;
                    if (leader) MbarExpectTx(&st->full[s], 2 * Cfg::kStageBytes);
                    const uint32_t bar = MapToCta(&st->full[s], 0);
                    TmaLoad3dPair(a, &maps->a, bar, k * 128, t.row, 0);
                    TmaLoad3dPair(b, GLU && !leader ? &maps->b[1] : &maps->b[0], bar, k * 128, mine, t.expert);
                    TmaLoad2dPair(sa, &maps->sa, bar, 0, t.scaleTile * g.tileCols + 2 * k);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        TmaLoad2dPair(sb + h * 2 * kTileBytes, &maps->sb[GLU ? h : 0], bar, 0,
                                      (t.expert * g.tileRowsB + n / 128 + (GLU ? 0 : h)) * g.tileCols + 2 * k);
                }
            }
            if (!alive) __nanosleep(500000);        // copies under way still write here: they end long before this does
        }
    } else if (warp == 1) {
        // -------------------------------------------------------------------- issuer (leader CTA only)
        if (leader && ElectOne()) {
            GridDependencyWait();
            int s = 0;
            uint32_t phase = 0, i = 0;
            const uint32_t low = DescLow(smem);
            bool alive = true;
            Tiles<256> tiles(g, start, first, step, rank);
            Tile t;
            while (alive && tiles.Next(&t)) {
                if (!MbarWait(&st->accEmpty[0], (i & 1) ^ 1, &st->abort)) { alive = false; break; }
                ++i;
                TcFenceAfter();
                uint32_t more = 0;
                for (int k = 0; k < stages; ++k) {
                    if (!MbarWait(&st->full[s], phase, &st->abort)) { alive = false; break; }
                    TcFenceAfter();
                    const uint32_t a = low + s * (Cfg::kStageBytes >> 4), b = a + (Cfg::kABytes >> 4), sa = b + (Cfg::kBBytes >> 4), sb = sa + (Cfg::kSaBytes >> 4);
                    const uint32_t ta = tmem + Cfg::kScaleBase + s * Cfg::kScaleCols, tb = ta + 8;
                    const int left = g.K - k * kStageCols;
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        if (c * kTileCols >= left) break;
                        CopyScalesPair(ta + c * 4, sa + c * (kTileBytes >> 4));
#pragma unroll
                        for (int h = 0; h < 2; ++h) CopyScalesPair(tb + c * 8 + h * 4, sb + (h * 2 + c) * (kTileBytes >> 4));
                    }
#pragma unroll
                    for (int u = 0; u < kStageCols / kUmmaCols; ++u) {
                        if (u * kUmmaCols >= left) break;
                        MmaMxf4Pair(tmem, a + u * 2, b + u * 2, InstrDescMxf4(256, 256, (u & 1) * 2), ta + (u >> 1) * 4, tb + (u >> 1) * 8, more);
                        more = 1;
                    }
                    MmaCommitPair(&st->empty[s]);
                    if (++s == Cfg::kStages) { s = 0; phase ^= 1; }
                }
                if (alive) MmaCommitPair(&st->accFull[0]);
            }
        }
    } else if (warp >= 4) {
        // ---------------------------------------------------------------------- epilogue (both CTAs)
        GridDependencyWait();
        uint8_t *slab = slabs + (warp - 4) * kSlabBytes;
        const bool wide = g.ldOut % 8 == 0 && ((uintptr_t)g.out & 15) == 0;
        uint32_t i = 0;
        Tiles<256> tiles(g, start, first, step, rank);
        Tile t;
        while (tiles.Next(&t)) {
            if (!MbarWait(&st->accFull[0], i & 1, &st->abort)) break;
            ++i;
            __syncwarp();
            TcFenceAfter();
            StoreTile<GLU>(g, t, tmem, warp - 4, lane, slab, wide, [&] {
                if (leader) MbarArrive(&st->accEmpty[0]);
                else RemoteArrive(MapToCta(&st->accEmpty[0], 0));
            });
        }
    }
    // Nobody leaves while the other CTA may still read this one's shared memory or signal its barriers, also after a wait that ran out.
    TcFenceBefore();
    __syncthreads();
    ClusterSync();
    if (warp == 1) TmemDealloc2(tmem, 512);
    if (threadIdx.x == 0 && st->abort) atomicExch(g.error, 1u);
}

}  // namespace hcfp4
