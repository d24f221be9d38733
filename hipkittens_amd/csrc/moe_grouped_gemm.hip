// The experts' products of a mixture-of-experts layer in bf16, for training: rows in the order of their experts
// (expert_offsets [E+1], on the device) times the experts' weights W [E, N, K], and both gradients.
//
//   forward  y[r]  = x[r] W[e]^T             contraction along the rows of both operands
//   dgrad    dx[r] = dy[r] W[e]              across W's rows
//   wgrad    dW[e] = sum_{r of e} dy[r]^T x[r]   across the rows of both; an expert without rows gets zeros
//
// fp32 accumulation, one rounding. No workspace and one launch: how many tiles of rows an expert has is known on the
// device only, so the grid holds the most there can be, and every workgroup finds its tile by a scan over the offsets.
#include "moe_grouped.h"
#include "../../include/hk355.h"

namespace hk {

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
    int lo = 0, rows = R;
    if (offsets) {
        const int lane = lane_id();
        int top = offsets[min(lane, e)];
        if (e >= 64) top = max(top, offsets[min(lane + 64, e)]);
        for (int i = 128; i <= e; i += 64) top = max(top, offsets[min(lane + i, e)]);
        lo = to_sgpr(min(max(offsets[e], 0), R));
        top = min(top, R);
        if (__any(top > lo)) {   // (not for a table of the sort's)
            for (int d = 32; d >= 1; d >>= 1) top = max(top, __shfl_xor(top, d, 64));
            lo = to_sgpr(top);
        }
        rows = to_sgpr(min(max(offsets[e + 1], lo), R)) - lo;
    }
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
    if (!a || !b || !c || (!offsets && E != 1)) return HK_ERR_NULL_POINTER;
    // (rows of at most 4 MB: 32-bit offsets inside a K-step's or a tile's rows)
    if (R <= 0 || R >= (1 << 30) || E <= 0 || E > kGroupedMaxE || N <= 0 || K <= 0 || (N % 8) != 0 || (K % 8) != 0 ||
        N > (1 << 21) || K > (1 << 21))
        return HK_ERR_BAD_SHAPE;
    if (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 15u) return HK_ERR_BAD_ALIGNMENT;
    return HK_OK;
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

template <bool DGRAD>
static int launch_grouped(const void* x, const void* W, const int32_t* offsets, void* y, int R, int E, int N, int K, hipStream_t s) {
    switch (grouped_choice(R, E, DGRAD ? N : K, DGRAD ? K : N, !offsets)) {
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
    if (!expert_offsets) return HK_ERR_NULL_POINTER;
    if (const int st = hk::grouped_check(x_bf16, w_bf16, y_bf16, expert_offsets, R, E, N, K)) return st;
    return hk::launch_grouped<false>(x_bf16, w_bf16, expert_offsets, y_bf16, R, E, N, K, (hipStream_t)stream);
}

extern "C" int hk_moe_grouped_gemm_dgrad(const void* dy_bf16, const void* w_bf16, const int32_t* expert_offsets, void* dx_bf16,
                                         int R, int E, int N, int K, void* stream) {
    if (!expert_offsets) return HK_ERR_NULL_POINTER;
    if (const int st = hk::grouped_check(dy_bf16, w_bf16, dx_bf16, expert_offsets, R, E, N, K)) return st;
    return hk::launch_grouped<true>(dy_bf16, w_bf16, expert_offsets, dx_bf16, R, E, N, K, (hipStream_t)stream);
}

extern "C" int hk_moe_grouped_gemm_wgrad(const void* dy_bf16, const void* x_bf16, const int32_t* expert_offsets, void* dw,
                                         int dw_type, int R, int E, int N, int K, void* stream) {
    if (!expert_offsets) return HK_ERR_NULL_POINTER;
    if (const int st = hk::grouped_check(dy_bf16, x_bf16, dw, expert_offsets, R, E, N, K)) return st;
    if (dw_type != 0 && dw_type != 1) return HK_ERR_UNSUPPORTED;
    return dw_type == 0 ? hk::launch_wgrad<uint16_t>(dy_bf16, x_bf16, expert_offsets, dw, R, E, N, K, (hipStream_t)stream)
                        : hk::launch_wgrad<float>(dy_bf16, x_bf16, expert_offsets, dw, R, E, N, K, (hipStream_t)stream);
}

// The gradients of a product without experts: the same kernels, all rows in one group.
extern "C" int hk_bf16_gemm_dgrad(const void* dy_bf16, const void* w_bf16, void* dx_bf16, int M, int N, int K, void* stream) {
    if (const int st = hk::grouped_check(dy_bf16, w_bf16, dx_bf16, nullptr, M, 1, N, K)) return st;
    return hk::launch_grouped<true>(dy_bf16, w_bf16, nullptr, dx_bf16, M, 1, N, K, (hipStream_t)stream);
}

extern "C" int hk_bf16_gemm_wgrad(const void* dy_bf16, const void* x_bf16, void* dw, int dw_type, int M, int N, int K, void* stream) {
    if (const int st = hk::grouped_check(dy_bf16, x_bf16, dw, nullptr, M, 1, N, K)) return st;
    if (dw_type != 0 && dw_type != 1) return HK_ERR_UNSUPPORTED;
    return dw_type == 0 ? hk::launch_wgrad<uint16_t>(dy_bf16, x_bf16, nullptr, dw, M, 1, N, K, (hipStream_t)stream)
                        : hk::launch_wgrad<float>(dy_bf16, x_bf16, nullptr, dw, M, 1, N, K, (hipStream_t)stream);
}
