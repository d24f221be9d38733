// Tiles of products whose rows are grouped by expert (expert_offsets [E+1], on the device): which tile a workgroup has, how many
// there can be, and the choice of the tile's kernel.
#pragma once
#include "gemm_layouts_ring.h"
#include "moe_common.h"

namespace hk {

constexpr int kGroupedMaxE = 512;
constexpr long long kMaxWorkgroups = 1ll << 24;   // of 256 threads: a launch has fewer than 2^32

struct GroupedTile { int expert, row0, rows, tile_n; };   // expert < 0: no such tile

// Tile `id` of the list: expert by expert, inside an expert in groups of eight tiles of rows that go over the columns side by
// side, so that an XCD's run of 32 tiles shares its operands (8192 x 8192 x 8192 731 us; with all 32 tiles of rows side by side 1078). Offsets
// are held inside [0, R] and in order whatever they hold (a running maximum: no row is two experts', and there are no more tiles than the
// grid has places for). Each wave scans by itself: lane l holds experts 8 l .. 8 l + 7. Offsets null: one expert with all R rows.
__device__ __forceinline__ GroupedTile grouped_tile(const int32_t* __restrict__ offsets, int E, int R, int tile_m, int tiles_n,
                                                    int in, int out, int id) {
    if (!offsets) {
        int pm, pn;
        const bool banded = 2ll * ((long long)R + out) * in > (320ll << 20);
        banded_raster(id, (R + tile_m - 1) / tile_m, tiles_n, banded ? 4 : 8, banded ? 16 : tiles_n, pm, pn);
        return GroupedTile{0, pm * tile_m, min(R - pm * tile_m, tile_m), pn};
    }
    const int lane = lane_id();
    int lo[8], hi[8], tiles[8], mine = 0;
    bool falls = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int e = 8 * lane + j;
        lo[j] = e < E ? min(max(offsets[e], 0), R) : 0;
        hi[j] = e < E ? min(max(offsets[e + 1], 0), R) : 0;
        falls |= hi[j] < lo[j];
    }
    if (__any(falls)) {   // (not for a table of the sort's; done always, 64 rows of 4 experts of 1024 x 1024 take 9.4 us instead of 9.1)
        int top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, max(lo[j], hi[j]));
        for (int d = 1; d < 64; d <<= 1) {
            const int u = __shfl_up(top, d, 64);
            if (lane >= d) top = max(top, u);
        }
        top = __shfl_up(top, 1, 64);   // of all offsets up to the lane's first
        if (lane == 0) top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            lo[j] = max(top, lo[j]);
            hi[j] = top = max(lo[j], hi[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        tiles[j] = 8 * lane + j < E ? (hi[j] - lo[j] + tile_m - 1) / tile_m * tiles_n : 0;
        mine += tiles[j];
    }
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(upto, d, 64);
        if (lane >= d) upto += u;
    }
    int at = upto - mine;
    GroupedTile t{-1, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (id >= at && id < at + tiles[j]) {
            int pm, pn;
            // bands where the expert's operands do not fit the memory-side cache (raster_band's rule; 8192 rows of 65536 x 4096:
            // 3425 us, with them 3002)
            const bool banded = 2ll * ((long long)(hi[j] - lo[j]) + out) * in > (320ll << 20);
            banded_raster(id - at, tiles[j] / tiles_n, tiles_n, banded ? 4 : 8, banded ? 16 : tiles_n, pm, pn);
            t = GroupedTile{8 * lane + j, lo[j] + pm * tile_m, 0, pn};
            t.rows = min(hi[j] - t.row0, tile_m);
        }
        at += tiles[j];
    }
    const uint64_t holder = __ballot(t.expert >= 0);
    if (!holder) return GroupedTile{-1, 0, 0, 0};
    const int src = __ffsll((unsigned long long)holder) - 1;
    return GroupedTile{__builtin_amdgcn_readlane(t.expert, src), __builtin_amdgcn_readlane(t.row0, src),
                       __builtin_amdgcn_readlane(t.rows, src), __builtin_amdgcn_readlane(t.tile_n, src)};
}

// most tiles of rows there can be: every expert with rows may leave one tile short of `tile` rows by all but one
inline long long grouped_tiles_m(int R, int E, int tile) {
    const long long used = R < E ? R : E;
    return (R + used * (tile - 1)) / tile;
}

// The tile by choose_layout with the tiles of rows that an expert has on average when the rows spread over the experts
// unevenly: one at least, else rows / tile + 0.6. (Forward, us, small / large: N = 4096, K = 7168, 32 experts: 1024 rows 320 / 341,
// 4096 457 / 482, 8192 764 / 539, 65536 4130 / 2873; 128 experts of 5760 x 2880, 16384 rows 1057 / 947; 8 of 1024 x 1024, 4096 rows
// 20 / 27. The rule's one miss there: 32 experts of 64 rows, small 428, large 359.)
inline double grouped_row_tiles(int R, int E, int tile, bool dense) {
    const double used = R < E ? R : E, m = dense ? (R + tile - 1) / tile : R / used / tile + 0.6;
    return used * (m > 1 ? m : 1);
}
inline LayoutChoice grouped_choice(int R, int E, int in, int out, bool dense = false) {
    auto tiles = [&](int tile) { return grouped_row_tiles(R, E, tile, dense) * ((out + tile - 1) / tile); };
    return choose_layout({tiles(256), tiles(128), tiles(64)}, (in + kLayoutStep - 1) / kLayoutStep, moe_num_compute_units());
}

}  // namespace hk
