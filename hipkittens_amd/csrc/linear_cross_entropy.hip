// Softmax cross entropy of the logits l = x W^T (x [M, K], W [V, K] bf16) from the hidden states, and its gradients, without
// the logits in memory.
//
//   forward   lse[m] = log sum_v exp l[m, v],  loss[m] = lse[m] - l[m, label[m]]
//   backward  dl[m, v] = dloss[m] (exp(l[m, v] - lse[m]) - [v = label[m]]),  dx = dl W,  dW = dl^T x
//
// A row whose label lies outside [0, V) has no loss: loss 0, dl 0 (lse is written all the same).
//
// Forward: one tile product; its epilogue leaves each row's maximum and sum of exponentials over the tile's columns (fp32) and
// the label's logit, a second launch joins them column block by column block, in order. Backward, for pieces of the vocabulary:
// the logits again, with dl rounded to bf16 as the epilogue (an operand of the two products that follow, whose other operand
// is bf16; it adds 2^-9 relative to each term of sums whose result is rounded to bf16), then dx += dl W in fp32 and dW = dl^T x.
#include <algorithm>

#include "gemm_layouts.h"
#include "../../include/hk355.h"

namespace hk {

struct HeadLabels {
    const void* p;
    int is64;
    // the label of row m, -1 where it counts for nothing
    __device__ __forceinline__ int at(int64_t m, int V) const {
        const int64_t l = is64 ? ((const int64_t*)p)[m] : (int64_t)((const int32_t*)p)[m];
        return l >= 0 && l < V ? (int)l : -1;
    }
};

constexpr int kHeadCols = kLayoutTile / 2;   // columns of one partial result: a wave's

__global__ __launch_bounds__(256) void head_logits_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ W,
                                                          HeadLabels labels, int M, int V, int K, int tiles_m, int tiles_n,
                                                          float2* __restrict__ partial, float* __restrict__ label_logit) {
    extern __shared__ __attribute__((aligned(2048))) uint8_t smem[];
    int pm, pn;
    grouped_raster(xcd_chunk_order(blockIdx.x, tiles_m * tiles_n, kCuPerXcd), tiles_m, tiles_n, 8, pm, pn);
    const int w = wave_id(), row0 = pm * kLayoutTile, col0 = pn * kLayoutTile;
    v4f acc[4][4];
    tile_product<false, false>(smem, operand_along(x, 2ull * K, row0, min(M, row0 + kLayoutTile), K),
                               operand_along(W, 2ull * K, col0, min(V, col0 + kLayoutTile), K), K, acc);
    const int r = lane_id() & 15, g = lane_id() >> 4;
    const int row = row0 + (w >> 1) * 64 + r, col = col0 + (w & 1) * 64 + 4 * g;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
        const int at = row + 16 * m;
        float top = -INFINITY;
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + 16 * n + j < V) top = fmaxf(top, acc[m][n][j]);
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        float sum = 0.f;
        const int label = at < M ? labels.at(at, V) : -1;
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (col + 16 * n + j < V) sum += __expf(acc[m][n][j] - top);
                if (col + 16 * n + j == label) label_logit[at] = acc[m][n][j];
            }
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        if (g == 0 && at < M) partial[(size_t)(col / kHeadCols) * M + at] = make_float2(top, sum);
    }
}

// Joins the partial results of a row: 16 rows a workgroup, 16 threads each, thread i every 16th block from i on; then thread by thread.
__global__ __launch_bounds__(256) void head_loss_kernel(const float2* __restrict__ partial, const float* __restrict__ label_logit,
                                                        HeadLabels labels, int M, int V, int blocks, float* __restrict__ loss,
                                                        float* __restrict__ lse) {
    __shared__ float2 part[16][17];
    const int r = threadIdx.x & 15, seg = threadIdx.x >> 4;
    const int64_t m = (int64_t)blockIdx.x * 16 + r;
    auto join = [](float2 a, float2 b) {
        const float top = fmaxf(a.x, b.x);
        // (a block of columns behind V, or of logits of -inf, has a sum of 0 and adds nothing)
        return top == -INFINITY ? make_float2(top, a.y + b.y) : make_float2(top, a.y * __expf(a.x - top) + b.y * __expf(b.x - top));
    };
    float2 all = make_float2(-INFINITY, 0.f);
    if (m < M)
        for (int b = seg; b < blocks; b += 16) all = join(all, partial[(size_t)b * M + m]);
    part[seg][r] = all;
    __syncthreads();
    if (seg == 0 && m < M) {
        for (int s = 1; s < 16; ++s) all = join(all, part[s][r]);
        const float l = all.x + logf(all.y);
        lse[m] = l;
        loss[m] = labels.at(m, V) >= 0 ? l - label_logit[m] : 0.f;
    }
}

// dl of the columns [v0, v0 + cols) of the vocabulary; `width` columns of it are written, those behind V as zeros.
__global__ __launch_bounds__(256) void head_dlogits_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ W,
                                                           HeadLabels labels, const float* __restrict__ lse,
                                                           const float* __restrict__ dloss, int M, int V, int K, int v0, int width,
                                                           int pitch, int tiles_m, int tiles_n, uint16_t* __restrict__ dl) {
    extern __shared__ __attribute__((aligned(2048))) uint8_t smem[];
    int pm, pn;
    grouped_raster(xcd_chunk_order(blockIdx.x, tiles_m * tiles_n, kCuPerXcd), tiles_m, tiles_n, 8, pm, pn);
    const int w = wave_id(), row0 = pm * kLayoutTile, col0 = v0 + pn * kLayoutTile;
    v4f acc[4][4];
    tile_product<false, false>(smem, operand_along(x, 2ull * K, row0, min(M, row0 + kLayoutTile), K),
                               operand_along(W, 2ull * K, col0, min(V, col0 + kLayoutTile), K), K, acc);
    const int r = lane_id() & 15, g = lane_id() >> 4;
    const int row = row0 + (w >> 1) * 64, col = col0 + (w & 1) * 64;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
        const int at = row + 16 * m + r;
        const int label = at < M ? labels.at(at, V) : -1;
        const float scale = label >= 0 ? dloss[at] : 0.f, l = at < M ? lse[at] : 0.f;
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int v = col + 16 * n + 4 * g + j;
                const float p = __expf(acc[m][n][j] - l) - (v == label ? 1.f : 0.f);
                acc[m][n][j] = label >= 0 && v < V ? scale * p : 0.f;
            }
    }
    store_tile(acc, dl + (size_t)row * pitch + (col - v0), pitch, M - row, v0 + width - col);
}

// dx of one piece, dl [M, cols] W [cols rows from v0 on]: `first` writes the fp32 sums, others add to them, `last` rounds.
__global__ __launch_bounds__(256) void head_dx_kernel(const uint16_t* __restrict__ dl, const uint16_t* __restrict__ W, int M, int V,
                                                      int K, int v0, int width, int pitch, int tiles_m, int tiles_n, bool first,
                                                      bool last, float* __restrict__ sums, uint16_t* __restrict__ dx) {
    extern __shared__ __attribute__((aligned(2048))) uint8_t smem[];
    int pm, pn;
    grouped_raster(xcd_chunk_order(blockIdx.x, tiles_m * tiles_n, kCuPerXcd), tiles_m, tiles_n, 8, pm, pn);
    const int w = wave_id(), row0 = pm * kLayoutTile, col0 = pn * kLayoutTile;
    v4f acc[4][4];
    tile_product<false, true>(smem, operand_along(dl, 2ull * pitch, row0, min(M, row0 + kLayoutTile), width),
                              operand_across(W + (size_t)v0 * K, 2ull * K, col0, min(width, V - v0)), width, acc);
    const int r = lane_id() & 15, g = lane_id() >> 4;
    const int row = row0 + (w >> 1) * 64, col = col0 + (w & 1) * 64;
    if (!first) {
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int n = 0; n < 4; ++n)
                if (row + 16 * m + r < M && col + 16 * n + 4 * g < K)
                    acc[m][n] += *(const v4f*)(sums + (size_t)(row + 16 * m + r) * K + col + 16 * n + 4 * g);
    }
    if (last) store_tile(acc, dx + (size_t)row * K + col, K, M - row, K - col);
    else store_tile(acc, sums + (size_t)row * K + col, K, M - row, K - col);
}

// dW of one piece: dl^T x over the M rows.
template <typename T>
__global__ __launch_bounds__(256) void head_dw_kernel(const uint16_t* __restrict__ dl, const uint16_t* __restrict__ x, int M, int cols,
                                                      int K, int pitch, int tiles_m, int tiles_n, T* __restrict__ dw) {
    extern __shared__ __attribute__((aligned(2048))) uint8_t smem[];
    int pm, pn;
    grouped_raster(xcd_chunk_order(blockIdx.x, tiles_m * tiles_n, kCuPerXcd), tiles_m, tiles_n, 8, pm, pn);
    const int w = wave_id(), row0 = pm * kLayoutTile, col0 = pn * kLayoutTile;
    v4f acc[4][4];
    tile_product<true, true>(smem, operand_across(dl, 2ull * pitch, row0, M), operand_across(x, 2ull * K, col0, M), M, acc);
    const int row = row0 + (w >> 1) * 64, col = col0 + (w & 1) * 64;
    store_tile(acc, dw + (size_t)row * K + col, K, cols - row, K - col);
}

static int head_tiles(int n) { return (n + kLayoutTile - 1) / kLayoutTile; }
static size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// forward: label logits, then the partial results; backward: dl of a piece, then the fp32 sums of dx
struct HeadForwardLayout {
    size_t label_logit, partial, bytes;
    HeadForwardLayout(int M, int V) {
        label_logit = 0;
        partial = up256((size_t)M * 4);
        bytes = partial + up256((size_t)M * 2 * head_tiles(V) * sizeof(float2));
    }
};
struct HeadBackwardLayout {
    int piece;   // columns of a piece, a multiple of the tile
    size_t dl, sums, bytes;
    HeadBackwardLayout(int M, int V, int K) {
        // pieces of 256 MB, and rows of at most 4 MB (32-bit offsets inside a K-step's rows)
        const long long most = std::min((256ll << 20) / (2ll * M), 1ll << 21) / kLayoutTile * kLayoutTile;
        const long long all = (long long)head_tiles(V) * kLayoutTile;
        piece = (int)(most < kLayoutTile ? kLayoutTile : most < all ? most : all);
        dl = 0;
        sums = up256((size_t)M * piece * 2);
        bytes = sums + (piece < V ? up256((size_t)M * K * 4) : 0);
    }
};

static int head_check(int M, int V, int K) {
    if (M <= 0 || V <= 0 || K <= 0 || (K % 8) != 0 || M >= (1 << 30) || V >= (1 << 30) || K > (1 << 21)) return HK_ERR_BAD_SHAPE;
    if ((long long)head_tiles(M) * (head_tiles(V) > head_tiles(K) ? head_tiles(V) : head_tiles(K)) >= (1ll << 31) ||
        (long long)head_tiles(V) * head_tiles(K) >= (1ll << 31))
        return HK_ERR_BAD_SHAPE;
    return HK_OK;
}

template <typename... P, typename... A>
static int launch_head(void (*kern)(P...), DeviceOnce& once, long long tiles, hipStream_t s, A... args) {
    if (!set_lds_limit_once((const void*)kern, kLayoutLdsBytes, once)) return HK_ERR_LAUNCH;
    hipLaunchKernelGGL(kern, dim3((unsigned)tiles), dim3(256), kLayoutLdsBytes, s, args...);
    return hipGetLastError() == hipSuccess ? HK_OK : HK_ERR_LAUNCH;
}

}  // namespace hk

extern "C" size_t hk_linear_cross_entropy_workspace_bytes(int M, int V, int K, int backward) {
    using namespace hk;
    if (head_check(M, V, K) != HK_OK) return 0;
    const size_t f = HeadForwardLayout(M, V).bytes, b = backward ? HeadBackwardLayout(M, V, K).bytes : 0;
    return f > b ? f : b;
}

extern "C" int hk_linear_cross_entropy(const void* x_bf16, const void* w_bf16, const void* labels, int label_type, float* loss,
                                       float* lse, int M, int V, int K, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace hk;
    if (!x_bf16 || !w_bf16 || !labels || !loss || !lse) return HK_ERR_NULL_POINTER;
    if (const int st = head_check(M, V, K)) return st;
    if (label_type != 0 && label_type != 1) return HK_ERR_UNSUPPORTED;
    if (((uintptr_t)x_bf16 | (uintptr_t)w_bf16 | (uintptr_t)workspace) & 15u) return HK_ERR_BAD_ALIGNMENT;
    const HeadForwardLayout L(M, V);
    if (!workspace || workspace_bytes < L.bytes) return HK_ERR_WORKSPACE;
    const hipStream_t s = (hipStream_t)stream;
    uint8_t* ws = (uint8_t*)workspace;
    const HeadLabels lab{labels, label_type};
    const int tm = head_tiles(M), tn = head_tiles(V);
    static DeviceOnce once;
    const int st = launch_head(head_logits_kernel, once, (long long)tm * tn, s, (const uint16_t*)x_bf16, (const uint16_t*)w_bf16, lab, M, V,
                               K, tm, tn, (float2*)(ws + L.partial), (float*)(ws + L.label_logit));
    if (st != HK_OK) return st;
    hipLaunchKernelGGL(head_loss_kernel, dim3((M + 15) / 16), dim3(256), 0, s, (const float2*)(ws + L.partial),
                       (const float*)(ws + L.label_logit), lab, M, V, 2 * tn, loss, lse);
    return hipGetLastError() == hipSuccess ? HK_OK : HK_ERR_LAUNCH;
}

extern "C" int hk_linear_cross_entropy_backward(const void* x_bf16, const void* w_bf16, const void* labels, int label_type,
                                                const float* lse, const float* dloss, void* dx_bf16_or_null, void* dw_or_null,
                                                int dw_type, int M, int V, int K, void* workspace, size_t workspace_bytes,
                                                void* stream) {
    using namespace hk;
    if (!x_bf16 || !w_bf16 || !labels || !lse || !dloss || (!dx_bf16_or_null && !dw_or_null)) return HK_ERR_NULL_POINTER;
    if (const int st = head_check(M, V, K)) return st;
    if ((label_type != 0 && label_type != 1) || (dw_type != 0 && dw_type != 1)) return HK_ERR_UNSUPPORTED;
    if (((uintptr_t)x_bf16 | (uintptr_t)w_bf16 | (uintptr_t)dx_bf16_or_null | (uintptr_t)dw_or_null | (uintptr_t)workspace) & 15u)
        return HK_ERR_BAD_ALIGNMENT;
    const HeadBackwardLayout L(M, V, K);
    if (!workspace || workspace_bytes < L.bytes) return HK_ERR_WORKSPACE;
    const hipStream_t s = (hipStream_t)stream;
    uint8_t* ws = (uint8_t*)workspace;
    const HeadLabels lab{labels, label_type};
    uint16_t* dl = (uint16_t*)(ws + L.dl);
    const uint16_t *x = (const uint16_t*)x_bf16, *w = (const uint16_t*)w_bf16;
    const int tm = head_tiles(M), tk = head_tiles(K);
    static DeviceOnce once_dl, once_dx, once_dw, once_dw32;
    for (int v0 = 0; v0 < V; v0 += L.piece) {
        const int cols = V - v0 < L.piece ? V - v0 : L.piece, width = (cols + 7) / 8 * 8, tv = head_tiles(cols);
        int st = launch_head(head_dlogits_kernel, once_dl, (long long)tm * tv, s, x, w, lab, lse, dloss, M, V, K, v0, width, L.piece, tm, tv, dl);
        if (st != HK_OK) return st;
        if (dx_bf16_or_null) {
            st = launch_head(head_dx_kernel, once_dx, (long long)tm * tk, s, (const uint16_t*)dl, w, M, V, K, v0, width, L.piece, tm, tk,
                             v0 == 0, v0 + L.piece >= V, (float*)(ws + L.sums), (uint16_t*)dx_bf16_or_null);
            if (st != HK_OK) return st;
        }
        if (dw_or_null) {
            const size_t at = (size_t)v0 * K;
            st = dw_type == 0 ? launch_head(head_dw_kernel<uint16_t>, once_dw, (long long)tv * tk, s, (const uint16_t*)dl, x, M, cols, K, L.piece,
                                            tv, tk, (uint16_t*)dw_or_null + at)
                              : launch_head(head_dw_kernel<float>, once_dw32, (long long)tv * tk, s, (const uint16_t*)dl, x, M, cols, K, L.piece,
                                            tv, tk, (float*)dw_or_null + at);
            if (st != HK_OK) return st;
        }
    }
    return HK_OK;
}
