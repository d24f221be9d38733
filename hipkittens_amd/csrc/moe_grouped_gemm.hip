// The experts' products of a mixture-of-experts layer in bf16, for training: rows in the order of their experts
// (expert_offsets [E+1], on the device) times the experts' weights W [E, N, K], and both gradients.
//
//   forward  y[r]  = x[r] W[e]^T             contraction along the rows of both operands
//   dgrad    dx[r] = dy[r] W[e]              across W's rows
//   wgrad    dW[e] = sum_{r of e} dy[r]^T x[r]   across the rows of both; an expert without rows gets zeros
//
// fp32 accumulation, one rounding. No workspace and one launch: how many tiles of rows an expert has is known on the
// device only, so the grid holds the most there can be, and every workgroup finds its tile by a scan over the offsets.
#include "gemm_layouts_ring.h"
#include "moe_common.h"
#include "../../include/hk355.h"

namespace hk {

constexpr int kGroupedMaxE = 512;
constexpr long long kMaxWorkgroups = 1ll << 24;   // of 256 threads: a launch has fewer than 2^32

struct GroupedTile { int expert, row0, rows, tile_n; };   // expert < 0: no such tile

// Tile `id` of the list: expert by expert, inside an expert in groups of eight tiles of rows that go over the columns side by
// side, so that an XCD's run of 32 tiles shares its operands (8192 x 8192 x 8192 731 us; with all 32 tiles of rows side by side 1078). Offsets
// are held inside [0, R] and in order whatever they hold (a running maximum: no row is two experts', and there are no more tiles than the
// grid has places for). Each wave scans by itself: lane l holds experts 8 l .. 8 l + 7.
__device__ __forceinline__ GroupedTile grouped_tile(const int32_t* __restrict__ offsets, int E, int R, int tile_m, int tiles_n,
                                                    int in, int out, int id) {
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

// x [R, K] W [E, N, K] -> y [R, N]; DGRAD: x [R, N] W [E, N, K] -> y [R, K]
template <typename Tile, bool DGRAD>
__global__ __launch_bounds__(256) void grouped_gemm_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ W,
                                                           const int32_t* __restrict__ offsets, uint16_t* __restrict__ y,
                                                           int R, int E, int N, int K, int tiles_n) {
    extern __shared__ __attribute__((aligned(2048))) uint8_t smem[];
    const int in = DGRAD ? N : K, out = DGRAD ? K : N;
    const GroupedTile t = grouped_tile(offsets, E, R, Tile::kTile, tiles_n, in, out, xcd_chunk_order(blockIdx.x, gridDim.x, kCuPerXcd));
    if (t.expert < 0) return;
    const int col0 = t.tile_n * Tile::kTile;
    const uint16_t* We = W + (size_t)t.expert * N * K;
    v4f acc[Tile::F][Tile::F];
    Tile::template product<false, DGRAD>(smem, operand_along(x, 2ull * in, t.row0, t.row0 + t.rows, in),
                                         DGRAD ? operand_across(We, 2ull * K, col0, N) : operand_along(We, 2ull * K, col0, N, K), in, acc);
    const int w = wave_id(), row = (w >> 1) * Tile::kPatch, col = col0 + (w & 1) * Tile::kPatch;
    store_patch(acc, y + (size_t)(t.row0 + row) * out + col, out, t.rows - row, out - col);
}

template <typename Tile, typename T>
__global__ __launch_bounds__(256) void grouped_wgrad_kernel(const uint16_t* __restrict__ dy, const uint16_t* __restrict__ x,
                                                            const int32_t* __restrict__ offsets, T* __restrict__ dW, int R,
                                                            int E, int N, int K, int tiles_m, int tiles_n) {
    extern __shared__ __attribute__((aligned(2048))) uint8_t smem[];
    const int id = xcd_chunk_order(blockIdx.x, gridDim.x, kCuPerXcd);
    const int e = id / (tiles_m * tiles_n);
    int pm, pn;
    grouped_raster(id - e * tiles_m * tiles_n, tiles_m, tiles_n, 8, pm, pn);
    // the expert's rows as in grouped_tile, from the maximum of the offsets up to its own (0.3 us of a workgroup's start; 128 experts of
    // 2880 x 2880, 128 rows, fp32 984 us without it, 1005 with it)
    const int lane = lane_id();
    int top = offsets[min(lane, e)];
    if (e >= 64) top = max(top, offsets[min(lane + 64, e)]);
    for (int i = 128; i <= e; i += 64) top = max(top, offsets[min(lane + i, e)]);
    int lo = to_sgpr(min(max(offsets[e], 0), R));
    top = min(top, R);
    if (__any(top > lo)) {   // (not for a table of the sort's)
        for (int d = 32; d >= 1; d >>= 1) top = max(top, __shfl_xor(top, d, 64));
        lo = to_sgpr(top);
    }
    const int rows = to_sgpr(min(max(offsets[e + 1], lo), R)) - lo;
    if (rows == 0) {   // zeros, in one run per workgroup
        constexpr int kVec = 16 / sizeof(T);
        const size_t n = (size_t)N * K / kVec, run = (n + tiles_m * tiles_n - 1) / (tiles_m * tiles_n);
        const size_t from = (size_t)(id - e * tiles_m * tiles_n) * run, to = min(n, from + run);
        v4i* out = (v4i*)(dW + (size_t)e * N * K);
        for (size_t i = from + threadIdx.x; i < to; i += 256) out[i] = v4i{0, 0, 0, 0};
        return;
    }
    const int row0 = pm * Tile::kTile, col0 = pn * Tile::kTile;
    v4f acc[Tile::F][Tile::F];
    Tile::template product<true, true>(smem, operand_across(dy + (size_t)lo * N, 2ull * N, row0, rows),
                                       operand_across(x + (size_t)lo * K, 2ull * K, col0, rows), rows, acc);
    const int w = wave_id(), row = row0 + (w >> 1) * Tile::kPatch, col = col0 + (w & 1) * Tile::kPatch;
    store_patch(acc, dW + (size_t)e * N * K + (size_t)row * K + col, K, N - row, K - col);
}

static int grouped_check(const void* a, const void* b, const void* c, const void* offsets, int R, int E, int N, int K) {
    if (!a || !b || !c || !offsets) return HK_ERR_NULL_POINTER;
    // (rows of at most 4 MB: 32-bit offsets inside a K-step's or a tile's rows)
    if (R <= 0 || R >= (1 << 30) || E <= 0 || E > kGroupedMaxE || N <= 0 || K <= 0 || (N % 8) != 0 || (K % 8) != 0 ||
        N > (1 << 21) || K > (1 << 21))
        return HK_ERR_BAD_SHAPE;
    if (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 15u) return HK_ERR_BAD_ALIGNMENT;
    return HK_OK;
}

// most tiles of rows there can be: every expert with rows may leave one tile short of `tile` rows by all but one
static long long grouped_tiles_m(int R, int E, int tile) {
    const long long used = R < E ? R : E;
    return (R + used * (tile - 1)) / tile;
}

template <typename Tile, bool DGRAD>
static int launch_grouped_tile(const void* x, const void* W, const int32_t* offsets, void* y, int R, int E, int N, int K, hipStream_t s) {
    const int tiles_n = ((DGRAD ? K : N) + Tile::kTile - 1) / Tile::kTile;
    const long long grid = grouped_tiles_m(R, E, Tile::kTile) * tiles_n;
    if (grid >= kMaxWorkgroups) return HK_ERR_BAD_SHAPE;
    auto kern = grouped_gemm_kernel<Tile, DGRAD>;
    static DeviceOnce configured;
    if (!set_lds_limit_once((const void*)kern, Tile::kLds, configured)) return HK_ERR_LAUNCH;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(256), Tile::kLds, s, (const uint16_t*)x, (const uint16_t*)W, offsets,
                       (uint16_t*)y, R, E, N, K, tiles_n);
    return hipGetLastError() == hipSuccess ? HK_OK : HK_ERR_LAUNCH;
}

// The tile by choose_layout with the tiles of rows that an expert has on average when the rows spread over the experts
// unevenly: one at least, else rows / tile + 0.6. (Forward, us, small / large: N = 4096, K = 7168, 32 experts: 1024 rows 320 / 341,
// 4096 457 / 482, 8192 764 / 539, 65536 4130 / 2873; 128 experts of 5760 x 2880, 16384 rows 1057 / 947; 8 of 1024 x 1024, 4096 rows
// 20 / 27. The rule's one miss there: 32 experts of 64 rows, small 428, large 359.)
static LayoutChoice grouped_choice(int R, int E, int in, int out) {
    const double used = R < E ? R : E, mean = R / used;
    auto tiles = [&](int tile) {
        const double m = mean / tile + 0.6;
        return used * (m > 1 ? m : 1) * ((out + tile - 1) / tile);
    };
    return choose_layout({tiles(256), tiles(128), tiles(64)}, (in + kLayoutStep - 1) / kLayoutStep, moe_num_compute_units());
}
template <bool DGRAD>
static int launch_grouped(const void* x, const void* W, const int32_t* offsets, void* y, int R, int E, int N, int K, hipStream_t s) {
    switch (grouped_choice(R, E, DGRAD ? N : K, DGRAD ? K : N)) {
        case kLayout256: return launch_grouped_tile<LayoutTile256, DGRAD>(x, W, offsets, y, R, E, N, K, s);
        case kLayout128: return launch_grouped_tile<LayoutTile128, DGRAD>(x, W, offsets, y, R, E, N, K, s);
        case kLayout128Deep: return launch_grouped_tile<LayoutTile128Deep, DGRAD>(x, W, offsets, y, R, E, N, K, s);
        default: return launch_grouped_tile<LayoutTile64Deep, DGRAD>(x, W, offsets, y, R, E, N, K, s);
    }
}

template <typename Tile, typename T>
static int launch_wgrad_tile(const void* dy, const void* x, const int32_t* offsets, void* dW, int R, int E, int N, int K, hipStream_t s) {
    const int tiles_m = (N + Tile::kTile - 1) / Tile::kTile, tiles_n = (K + Tile::kTile - 1) / Tile::kTile;
    const long long grid = (long long)E * tiles_m * tiles_n;
    if (grid >= kMaxWorkgroups) return HK_ERR_BAD_SHAPE;
    auto kern = grouped_wgrad_kernel<Tile, T>;
    static DeviceOnce configured;
    if (!set_lds_limit_once((const void*)kern, Tile::kLds, configured)) return HK_ERR_LAUNCH;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(256), Tile::kLds, s, (const uint16_t*)dy, (const uint16_t*)x, offsets,
                       (T*)dW, R, E, N, K, tiles_m, tiles_n);
    return hipGetLastError() == hipSuccess ? HK_OK : HK_ERR_LAUNCH;
}
template <typename T>
static int launch_wgrad(const void* dy, const void* x, const int32_t* offsets, void* dW, int R, int E, int N, int K, hipStream_t s) {
    const double e = E, n256 = (N + 255) / 256, k256 = (K + 255) / 256, n128 = (N + 127) / 128, k128 = (K + 127) / 128;
    const int cus = moe_num_compute_units();
    const double steps = (double)R / E / kLayoutStep + 0.5;
    // Enough small tiles for four of the single-stage kernel on every CU, whose loads, products and stores then overlap one
    // another's: up to about 300 rows an expert. (us, large / two stages / one: 32 experts of 4096 x 7168, 32 rows each 461 / 447 / 367,
    // 128 634 / 635 / 565, 256 800 / 874 / 784, 384 936 / 1092 / 962; 128 experts of 2880 x 2880, 128 rows, fp32 1090 / 1117 / 1017;
    // fewer tiles, 8 experts of 1024 x 1024: 24 / 14 / 18.)
    if (e * n128 * k128 >= 4.0 * cus) {
        const double large = e * n256 * k256 / cus * (kLargeFixed + kLargeStep * steps), single = e * n128 * k128 / (4.0 * cus) * (3.8 + 2.08 * steps);
        return large < single ? launch_wgrad_tile<LayoutTile256, T>(dy, x, offsets, dW, R, E, N, K, s)
                              : launch_wgrad_tile<LayoutTile128Stages<1>, T>(dy, x, offsets, dW, R, E, N, K, s);
    }
    const double t64 = e * ((N + 63) / 64) * ((K + 63) / 64);
    switch (choose_layout({e * n256 * k256, e * n128 * k128, t64}, steps, cus, kSmallStepAcross)) {
        case kLayout256: return launch_wgrad_tile<LayoutTile256, T>(dy, x, offsets, dW, R, E, N, K, s);
        case kLayout128: return launch_wgrad_tile<LayoutTile128, T>(dy, x, offsets, dW, R, E, N, K, s);
        case kLayout128Deep: return launch_wgrad_tile<LayoutTile128Deep, T>(dy, x, offsets, dW, R, E, N, K, s);
        default: return launch_wgrad_tile<LayoutTile64Deep, T>(dy, x, offsets, dW, R, E, N, K, s);
    }
}

}  // namespace hk

extern "C" int hk_moe_grouped_gemm(const void* x_bf16, const void* w_bf16, const int32_t* expert_offsets, void* y_bf16, int R,
                                   int E, int N, int K, void* stream) {
    if (const int st = hk::grouped_check(x_bf16, w_bf16, y_bf16, expert_offsets, R, E, N, K)) return st;
    return hk::launch_grouped<false>(x_bf16, w_bf16, expert_offsets, y_bf16, R, E, N, K, (hipStream_t)stream);
}

extern "C" int hk_moe_grouped_gemm_dgrad(const void* dy_bf16, const void* w_bf16, const int32_t* expert_offsets, void* dx_bf16,
                                         int R, int E, int N, int K, void* stream) {
    if (const int st = hk::grouped_check(dy_bf16, w_bf16, dx_bf16, expert_offsets, R, E, N, K)) return st;
    return hk::launch_grouped<true>(dy_bf16, w_bf16, expert_offsets, dx_bf16, R, E, N, K, (hipStream_t)stream);
}

extern "C" int hk_moe_grouped_gemm_wgrad(const void* dy_bf16, const void* x_bf16, const int32_t* expert_offsets, void* dw,
                                         int dw_type, int R, int E, int N, int K, void* stream) {
    if (const int st = hk::grouped_check(dy_bf16, x_bf16, dw, expert_offsets, R, E, N, K)) return st;
    if (dw_type != 0 && dw_type != 1) return HK_ERR_UNSUPPORTED;
    return dw_type == 0 ? hk::launch_wgrad<uint16_t>(dy_bf16, x_bf16, expert_offsets, dw, R, E, N, K, (hipStream_t)stream)
                        : hk::launch_wgrad<float>(dy_bf16, x_bf16, expert_offsets, dw, R, E, N, K, (hipStream_t)stream);
}
