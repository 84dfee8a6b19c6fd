// fp4.cuh - what the microscaled 4-bit kernels share: where scale bytes lie, and the table of row groups.
#pragma once
#include <stdint.h>

namespace hcfp4 {

constexpr int kBlock = 32;              // values that share a scale
constexpr int kTileRows = 128;          // rows and columns of a tile of scales
constexpr int kTileCols = 128;
constexpr int kTileBytes = 512;
constexpr int kMaxExperts = 1024;

// Tile rows that any split of `rows` into `experts` groups needs at most.
inline int64_t GroupedTileRows(int64_t rows, int experts) { return rows / kTileRows + (rows < experts ? rows : experts); }

// Byte of row r (of its tile row) and block 0 inside a tile; block b follows at + b.
__host__ __device__ constexpr uint32_t ScaleByte(uint32_t r) { return (r % 32) * 16 + r / 32 * 4; }

// Where the rows of each expert start, and its tiles of scales, from the offsets in device memory.  Offsets are clamped to
// [0, rows] and made to rise, so that whatever they hold, rows and tiles stay inside their buffers:
// sum of ceil(rows of e / 128) <= GroupedTileRows.  One warp calls it; start and, where it is wanted, tile have experts + 1
// entries in shared memory.
__device__ __forceinline__ void BuildGroups(const int32_t *offsets, int experts, int rows, int *start, int *tile)
{
    const int lane = threadIdx.x & 31;
    int low = 0, before = 0, last = 0;          // last offset so far, tiles so far, the same at the end of the round before
    for (int base = 0; base <= experts; base += 32) {
        const int e = base + lane;
        int v = e <= experts ? min(max(offsets[e], 0), rows) : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, v, d);
            if (lane >= d) v = max(v, o);
        }
        v = max(v, low);
        // tiles of the expert in front of this entry
        int prev = __shfl_up_sync(0xffffffffu, v, 1);
        if (lane == 0) prev = base == 0 ? v : last;
        int t = (v - prev + kTileRows - 1) / kTileRows;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, t, d);
            if (lane >= d) t += o;
        }
        t += before;
        if (e <= experts) {
            start[e] = v;
            if (tile) tile[e] = t;
        }
        low = last = __shfl_sync(0xffffffffu, v, 31);
        before = __shfl_sync(0xffffffffu, t, 31);
    }
}

// The expert whose rows hold `row`, which lies in [start[0], start[experts]).
__device__ __forceinline__ int GroupOf(const int *start, int experts, int row)
{
    int lo = 0, hi = experts;           // start[lo] <= row < start[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= row) lo = mid;
        else hi = mid;
    }
    return lo;
}

}  // namespace hcfp4
