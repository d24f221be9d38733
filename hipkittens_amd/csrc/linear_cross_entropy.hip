// Softmax cross entropy of the logits l = x W^T (x [M, K], W [V, K] bf16) from the hidden states, and its gradients, without
// the logits in memory.
//
//   forward   lse[m] = log sum_v exp l[m, v],  loss[m] = lse[m] - l[m, label[m]]
//   backward  dl[m, v] = dloss[m] (exp(l[m, v] - lse[m]) - [v = label[m]]),  dx = dl W,  dW = dl^T x
//
// A row whose label lies outside [0, V) has no loss: loss 0, dl 0 (lse is written all the same), and takes no part in dx and dW
// whatever its x holds.
//
// Forward: one tile product; its epilogue leaves each row's maximum and sum of exponentials over the tile's columns (fp32) and
// the label's logit, a second launch joins them column block by column block, in order. Backward, for pieces of the vocabulary:
// the logits again, with dl rounded to bf16 as the epilogue (an operand of the two products that follow, whose other operand
// is bf16), then dx += dl W in fp32 and dW = dl^T x. The rounding is at most 2^-8 of each term, and a row's largest term is most
// often its label's, scale (p - 1): that one's remainder, r[m], is kept in fp32 and its products r[m] W[label] and r[m] x[m] are
// added in the epilogues of dx and dW. (Error of dx and dW against 64 bits, relative, 1111 rows: 0.0024 without the remainder, 0.0031
// and more for a few rows; 0.0017 with it, which is the rounding of dx and dW themselves. Before that rounding 1.3e-4 to 1.6e-4
// with flat logits, 2e-4 to 1.1e-3 where other classes than the label have large shares: up to 1.2 times the error of rounding a
// bf16 result, which is what holding dl in half the bytes and multiplying it once costs.)
// For dW in fp32 that would be all its error, so there dl is two numbers of bf16, the value and what is left of it (then 2^-16 of each
// term), one below the other as 2 M rows, times two copies of x below one another; the label's remainder behind both is kept likewise.
#include <algorithm>

#include "gemm_layouts_ring.h"
#include "moe_common.h"
#include "../../include/hk355.h"

namespace hk {

constexpr float kLog2e = 1.4426950408889634f;

// Tile rows of a raster group, as the BF16 GEMM takes them: bands where the operands do not fit the memory-side cache (us, without /
// with: forward 8192 x 129280 x 7168 10957 / 10600, 4096 x 201088 x 2880 3555 / 3522, backward of the first 33689 / 32919).
__device__ __forceinline__ int head_group(int band_n, int tiles_n) { return band_n < tiles_n ? 4 : 8; }

struct HeadLabels {
    const void* p;
    int is64;
    // the label of row m, -1 where it counts for nothing
    __device__ __forceinline__ int at(int64_t m, int V) const {
        const int64_t l = is64 ? ((const int64_t*)p)[m] : (int64_t)((const int32_t*)p)[m];
        return l >= 0 && l < V ? (int)l : -1;
    }
};

template <typename Tile>
__global__ __launch_bounds__(256) void head_logits_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ W,
                                                          HeadLabels labels, int M, int V, int K, int tiles_m, int tiles_n, int band_n,
                                                          float2* __restrict__ partial, float* __restrict__ label_logit) {
    extern __shared__ __attribute__((aligned(2048))) uint8_t smem[];
    int pm, pn;
    banded_raster(xcd_chunk_order(blockIdx.x, tiles_m * tiles_n, kCuPerXcd), tiles_m, tiles_n, head_group(band_n, tiles_n), band_n, pm, pn);
    const int w = wave_id(), row0 = pm * Tile::kTile, col0 = pn * Tile::kTile;
    v4f acc[Tile::F][Tile::F];
    Tile::template product<false, false>(smem, operand_along(x, 2ull * K, row0, min(M, row0 + Tile::kTile), K),
                               operand_along(W, 2ull * K, col0, min(V, col0 + Tile::kTile), K), K, acc);
    const int r = lane_id() & 15, g = lane_id() >> 4;
    const int row = row0 + (w >> 1) * Tile::kPatch + r, first = col0 + (w & 1) * Tile::kPatch, left = V - first;
#pragma unroll
    for (int m = 0; m < Tile::F; ++m) {
        const int at = row + 16 * m;
        v4f l[Tile::F];
        Tile::read_row(acc[m], l);
        if (left < Tile::kPatch) {   // columns behind V
#pragma unroll
            for (int n = 0; n < Tile::F; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) l[n][j] = 16 * n + 4 * g + j < left ? l[n][j] : -INFINITY;
        }
        const int label = (at < M ? labels.at(at, V) : -1) - first;   // its column of the patch
        const bool here = label >= 0 && label < Tile::kPatch && ((label >> 2) & 3) == g;   // ... among this lane's
        if (__any(here)) {
            float mine = 0.f;
#pragma unroll
            for (int n = 0; n < Tile::F; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) mine = label == 16 * n + 4 * g + j ? l[n][j] : mine;
            if (here) label_logit[at] = mine;
        }
        float top = -INFINITY;
#pragma unroll
        for (int n = 0; n < Tile::F; ++n) top = fmaxf(fmaxf(top, fmaxf(l[n].x, l[n].y)), fmaxf(l[n].z, l[n].w));
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        // exponents of 2 from here on: the sum is exactly relative to 2^top2, whatever the rounding of top2
        const float top2 = top * kLog2e, off = top == -INFINITY ? 0.f : -top2;
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < Tile::F; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(l[n][j], kLog2e, off));
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        if (g == 0 && at < M) partial[(size_t)(first / Tile::kPatch) * M + at] = make_float2(top2, sum);
        slot_fence();   // (one row block's values in registers at a time)
    }
}

// Joins the partial results (exponents of 2) of a row: 16 rows a workgroup, 64 threads each, thread i the blocks i, 64 + i, .., eight loads
// at a time; then pair by pair. (Forward of 60 x 100000 x 600, 1564 blocks: 66 us with 16 threads a row and a load at a time, now 39.)
constexpr int kJoin = 64;
__global__ __launch_bounds__(16 * kJoin) void head_loss_kernel(const float2* __restrict__ partial, const float* __restrict__ label_logit,
                                                               HeadLabels labels, int M, int V, int blocks, float* __restrict__ loss,
                                                               float* __restrict__ lse) {
    __shared__ float2 part[kJoin][17];
    const int r = threadIdx.x & 15, seg = threadIdx.x >> 4;
    const int64_t m = (int64_t)blockIdx.x * 16 + r;
    auto join = [](float2 a, float2 b) {
        const float top = fmaxf(a.x, b.x);
        // (a block of columns behind V, or of logits of -inf, has a sum of 0 and adds nothing)
        return top == -INFINITY ? make_float2(top, a.y + b.y)
                                : make_float2(top, a.y * __builtin_amdgcn_exp2f(a.x - top) + b.y * __builtin_amdgcn_exp2f(b.x - top));
    };
    float2 all = make_float2(-INFINITY, 0.f);
    if (m < M)
        for (int b0 = seg; b0 < blocks; b0 += 8 * kJoin) {
            float2 p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = b0 + i * kJoin < blocks ? partial[(size_t)(b0 + i * kJoin) * M + m] : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int i = 0; i < 8; ++i) all = join(all, p[i]);
        }
    part[seg][r] = all;
    for (int off = kJoin / 2; off >= 1; off >>= 1) {
        __syncthreads();
        if (seg < off) part[seg][r] = all = join(all, part[seg + off][r]);
    }
    if (seg == 0 && m < M) {
        // lse is rounded once. The loss does not come from it: for a confident row it is far smaller than a step of lse, but the label's distance
        // from the largest logit and the logarithm of the sum are of its own size. (No loss is negative; a rounding of the sum, 1 or more, may be.)
        constexpr double kToNatural = 1.0 / (double)kLog2e;
        const float sum2 = log2f(all.y);
        lse[m] = (float)(((double)all.x + (double)sum2) * kToNatural);
        float l = 0.f;
        if (labels.at(m, V) >= 0) l = (sum2 - __builtin_fmaf(label_logit[m], kLog2e, -all.x)) * (float)kToNatural;
        loss[m] = l < 0.f ? 0.f : l;
    }
}

__device__ __forceinline__ float bf16_value(float v) { return __uint_as_float(pack_bf16(0.f, v) & 0xffff0000u); }
__device__ __forceinline__ v4f bf16_quad(const uint16_t* p) {
    const v2i q = *(const v2i*)p;
    return v4f{__uint_as_float((uint32_t)q.x << 16), __uint_as_float((uint32_t)q.x & 0xffff0000u),
               __uint_as_float((uint32_t)q.y << 16), __uint_as_float((uint32_t)q.y & 0xffff0000u)};
}

// Rows by the block of 16 classes that holds their label: list = the rows of block 0, of block 1, .. in ascending order,
// starts[b] = where block b's begin (blocks + 1 entries). One workgroup per 256 classes: the labels below its first class tell
// where its rows begin. Each wave takes a quarter of the rows, in order, twice: to count (lane b < 16: rows of block b) and to place.
// Eight times 64 labels are read at a time; of 64, those of one block are taken together (16 steps at most, one where all are of one class).
struct HeadRows {
    int32_t *starts, *list;
    uint16_t* x;          // x with zeros for the rows that count for nothing
    uint16_t* x_again;    // the same once more, behind the other, or null
    int groups, copies;   // workgroups of 256 classes, of kHeadCopyRows rows of x; 0: not wanted
};
constexpr int kHeadCopyRows = 8;
// Rows of x for dW, whose products with dl's zeros must be zeros whatever a row without a label (padding) holds.
__device__ __forceinline__ void head_copy_rows(const uint16_t* __restrict__ x, const HeadLabels& labels, int M, int V, int K,
                                               uint16_t* __restrict__ out, uint16_t* __restrict__ again, int group) {
    const int64_t m0 = (int64_t)group * kHeadCopyRows;
    const int chunks = K / 8, n = (int)min((int64_t)kHeadCopyRows, M - m0) * chunks;
    for (int c0 = threadIdx.x; c0 < n; c0 += 8 * 256) {
        v4i row[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = c0 + i * 256;
            row[i] = v4i{0, 0, 0, 0};
            if (c < n && labels.at(m0 + c / chunks, V) >= 0) row[i] = *(const v4i*)(x + m0 * K + (int64_t)c * 8);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c0 + i * 256 < n) {
                *(v4i*)(out + m0 * K + (int64_t)(c0 + i * 256) * 8) = row[i];
                if (again) *(v4i*)(again + m0 * K + (int64_t)(c0 + i * 256) * 8) = row[i];
            }
    }
}
__device__ __forceinline__ void head_label_rows(int* counts, const HeadLabels& labels, int M, int V, const HeadRows& rows, int group) {
    const int lane = lane_id(), w = wave_id(), first = group * 256;
    const int quarter = (M + 3) / 4, from = min(w * quarter, M), to = min(from + quarter, M);
    int below = 0;
    // found(row0, block, which): rows row0 + l for the bits l of `which` are of the block; wave by wave in the order of the rows
    auto scan = [&](auto found) __attribute__((always_inline)) {
        for (int m0 = from; m0 < to; m0 += 8 * 64) {
            int label[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) label[i] = m0 + 64 * i + lane < to ? labels.at(m0 + 64 * i + lane, V) : -1;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                below += __popcll(__ballot(label[i] >= 0 && label[i] < first));
                uint64_t in = __ballot(label[i] >= first && label[i] < first + 256);
                while (in) {
                    const int block = (__builtin_amdgcn_readlane(label[i], __ffsll((unsigned long long)in) - 1) - first) / 16;
                    const uint64_t which = __ballot(label[i] >= first && (label[i] - first) / 16 == block);
                    in &= ~which;
                    found(m0 + 64 * i, block, which);
                }
            }
        }
    };
    int mine = 0;
    scan([&](int, int block, uint64_t which) __attribute__((always_inline)) { mine += lane == block ? __popcll(which) : 0; });
    if (lane < 16) counts[w * 17 + lane] = mine;
    if (lane == 16) counts[w * 17 + 16] = below;
    __syncthreads();
    int at = 0;   // lane b: where this wave's first row of block b goes
    if (lane <= 16) {
        for (int v = 0; v < 4; ++v) {
            at += counts[v * 17 + 16];
            for (int b = 0; b < lane; ++b) at += counts[v * 17 + b];
        }
        if (w == 0 && (lane < 16 || group == rows.groups - 1)) rows.starts[group * 16 + lane] = at;
        if (lane < 16)
            for (int v = 0; v < w; ++v) at += counts[v * 17 + lane];
    }
    scan([&](int row0, int block, uint64_t which) __attribute__((always_inline)) {
        const int pos = __builtin_amdgcn_readlane(at, block);
        if (which >> lane & 1) rows.list[pos + __popcll(which & ((1ull << lane) - 1))] = row0 + lane;
        at += lane == block ? __popcll(which) : 0;
    });
}

// What is left of dl's label terms, in fp32: behind one number of bf16, for dx and dW; and behind two, for dW in fp32.
struct HeadRemainders { float *one, *two; };

// dl of the columns [v0, v0 + cols) of the vocabulary; `width` columns of it are written, those behind V as zeros; what the rounding
// leaves of it goes to dl_rest (null: not wanted). The last
// workgroups copy x and sort the rows by label for the launch behind this one.
template <typename Tile>
__global__ __launch_bounds__(256) void head_dlogits_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ W,
                                                           HeadLabels labels, const float* __restrict__ lse,
                                                           const float* __restrict__ dloss, int M, int V, int K, int v0, int width,
                                                           int pitch, int tiles_m, int tiles_n, int band_n,
                                                           uint16_t* __restrict__ dl, uint16_t* __restrict__ dl_rest,
                                                           HeadRemainders rest, HeadRows rows) {
    extern __shared__ __attribute__((aligned(2048))) uint8_t smem[];
    const int extra = (int)blockIdx.x - tiles_m * tiles_n;
    if (extra >= rows.copies) return head_label_rows((int*)smem, labels, M, V, rows, extra - rows.copies);
    if (extra >= 0) return head_copy_rows(x, labels, M, V, K, rows.x, rows.x_again, extra);
    int pm, pn;
    banded_raster(xcd_chunk_order(blockIdx.x, tiles_m * tiles_n, kCuPerXcd), tiles_m, tiles_n, head_group(band_n, tiles_n), band_n, pm, pn);
    const int w = wave_id(), row0 = pm * Tile::kTile, col0 = v0 + pn * Tile::kTile;
    v4f acc[Tile::F][Tile::F];
    Tile::template product<false, false>(smem, operand_along(x, 2ull * K, row0, min(M, row0 + Tile::kTile), K),
                               operand_along(W, 2ull * K, col0, min(V, col0 + Tile::kTile), K), K, acc);
    const int r = lane_id() & 15, g = lane_id() >> 4;
    const int row = row0 + (w >> 1) * Tile::kPatch, col = col0 + (w & 1) * Tile::kPatch, left = V - col;
#pragma unroll
    for (int m = 0; m < Tile::F; ++m) {
        const int at = row + 16 * m + r;
        const int label = at < M ? labels.at(at, V) : -1;
        const float scale = label >= 0 ? dloss[at] : 0.f, own = label >= 0 ? lse[at] : 0.f, lse2 = own * kLog2e;
        // what the rounding of lse2 leaves (of lse2 = 500 up to 2^-16, more than a confident row's p - 1) goes into the exponentials' factor
        const float part = fabsf(lse2) < INFINITY ? scale * __builtin_amdgcn_exp2f(-__builtin_fmaf(own, kLog2e, -lse2)) : scale;
        v4f d[Tile::F];
        Tile::read_row(acc[m], d);
#pragma unroll
        for (int n = 0; n < Tile::F; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) d[n][j] = part * __builtin_amdgcn_exp2f(__builtin_fmaf(d[n][j], kLog2e, -lse2));
        const bool here = label >= col && label < col + Tile::kPatch && ((label >> 2) & 3) == g;   // among this lane's
        if (__any(here)) {
            float left_over = 0.f;
#pragma unroll
            for (int n = 0; n < Tile::F; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bool hot = label == col + 16 * n + 4 * g + j;
                    d[n][j] -= hot ? scale : 0.f;
                    left_over = hot ? d[n][j] - bf16_value(d[n][j]) : left_over;
                }
            if (here) {
                rest.one[at] = left_over;
                if (dl_rest) rest.two[at] = left_over - bf16_value(left_over);
            }
        }
        if (left < Tile::kPatch || __any(label < 0)) {   // zeros, not products with zero
#pragma unroll
            for (int n = 0; n < Tile::F; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) d[n][j] = label >= 0 && 16 * n + 4 * g + j < left ? d[n][j] : 0.f;
        }
        store_block_row(d, m, dl + (size_t)row * pitch + (col - v0), pitch, M - row, v0 + width - col);
        if (dl_rest) {
#pragma unroll
            for (int n = 0; n < Tile::F; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) d[n][j] -= bf16_value(d[n][j]);
            store_block_row(d, m, dl_rest + (size_t)row * pitch + (col - v0), pitch, M - row, v0 + width - col);
        }
        slot_fence();
    }
}

// Both gradients of one piece in one launch, the items of dx, dl [M, cols] W [cols rows from v0 on], and those of dW, dl^T x, the
// longer ones first (65536 x 32000 x 1024 with dx's always first 18501 us, 15444 so, both with pieces of 4096 classes). The contraction of
// dx runs over the piece, a few hundred K-steps for few tiles: with dW's tiles behind it in the same grid CUs that hold no item of dx
// work on dW from the start, and `splits` cuts it where its items would still outlast the rest.
struct HeadPiece {
    const uint16_t *dl, *W, *x;   // x: with zeros for the rows that count for nothing; dl and x: dw_rows rows of them for dW
    float* sums;      // [splits][M][K]: dx so far, when there are several pieces or splits
    HeadLabels labels;
    const float *dx_rest, *dw_rest;   // r[m], of the rows whose label lies in this piece or an earlier one
    const int32_t *starts, *list;    // rows by their label's block of 16 classes
    uint16_t* dx;
    int M, V, K, v0, cols, pitch;
    int dw_rows;   // M, or 2 M: dl's values and what is left of them, x twice
    int tiles_m, tiles_k, tiles_v, band_dx, band_dw, splits, split_cols;   // splits 0: no dx; tiles_v 0: no dW
    bool first, last, reduce;   // reduce: a launch of its own adds the splits and rounds
    bool dw_first;    // dW's tiles are the longer ones
};

template <typename Tile>
__device__ __forceinline__ void head_dx_item(uint8_t* smem, const HeadPiece& p, int id) {
    const int tiles = p.tiles_m * p.tiles_k, split = id / tiles;
    int pm, pn;
    banded_raster(id - split * tiles, p.tiles_m, p.tiles_k, head_group(p.band_dx, p.tiles_k), p.band_dx, pm, pn);
    const int w = wave_id(), row0 = pm * Tile::kTile, col0 = pn * Tile::kTile;
    const int c0 = split * p.split_cols, n = min(p.split_cols, (p.cols + 7) / 8 * 8 - c0);   // (columns of dl behind `cols`: zeros)
    v4f acc[Tile::F][Tile::F];
    Tile::template product<false, true>(smem, operand_along(p.dl + c0, 2ull * p.pitch, row0, min(p.M, row0 + Tile::kTile), n),
                                        operand_across(p.W + (size_t)(p.v0 + c0) * p.K, 2ull * p.K, col0, min(n, p.V - p.v0 - c0)), n, acc);
    const int r = lane_id() & 15, g = lane_id() >> 4;
    const int row = row0 + (w >> 1) * Tile::kPatch, col = col0 + (w & 1) * Tile::kPatch;
    float* sums = p.sums + (size_t)split * p.M * p.K;
#pragma unroll
    for (int m = 0; m < Tile::F; ++m) {
        const int at = row + 16 * m + r;
        v4f v[Tile::F];
        Tile::read_row(acc[m], v);
#pragma unroll
        for (int c = 0; c < Tile::F; ++c) {
            if (!p.first && at < p.M && col + 16 * c + 4 * g < p.K) v[c] += *(const v4f*)(sums + (size_t)at * p.K + col + 16 * c + 4 * g);
        }
        if (p.last && !p.reduce) {
            const int label = at < p.M ? p.labels.at(at, p.V) : -1;
            if (label >= 0) {
                const float rest = p.dx_rest[at];
#pragma unroll
                for (int c = 0; c < Tile::F; ++c)
                    if (col + 16 * c + 4 * g < p.K) v[c] += rest * bf16_quad(p.W + (size_t)label * p.K + col + 16 * c + 4 * g);
            }
            store_block_row(v, m, p.dx + (size_t)row * p.K + col, p.K, p.M - row, p.K - col);
        } else {
            store_block_row(v, m, sums + (size_t)row * p.K + col, p.K, p.M - row, p.K - col);
        }
        slot_fence();
    }
}

template <typename Tile, typename T>
__global__ __launch_bounds__(256) void head_gradients_kernel(HeadPiece p, T* __restrict__ dw) {
    extern __shared__ __attribute__((aligned(2048))) uint8_t smem[];
    const int dx_items = p.splits * p.tiles_m * p.tiles_k, dw_items = p.tiles_v * p.tiles_k;
    const int dx_id = (int)blockIdx.x - (p.dw_first ? dw_items : 0);
    if (dx_id >= 0 && dx_id < dx_items) {
        head_dx_item<Tile>(smem, p, xcd_chunk_order(dx_id, dx_items, kCuPerXcd));
        return;
    }
    int pm, pn;
    banded_raster(xcd_chunk_order((int)blockIdx.x - (p.dw_first ? 0 : dx_items), dw_items, kCuPerXcd), p.tiles_v, p.tiles_k,
                  head_group(p.band_dw, p.tiles_k), p.band_dw, pm, pn);
    const int lane = lane_id(), r = lane & 15, g = lane >> 4;
    const int w = wave_id(), row0 = pm * Tile::kTile, col0 = pn * Tile::kTile;
    const int row = row0 + (w >> 1) * Tile::kPatch, col = col0 + (w & 1) * Tile::kPatch;
    // The rows with a label among this wave's classes, in the order of their blocks: the first 64 of them, one per lane, with label
    // and remainder, before the product.
    const int block0 = (p.v0 + row) / 16, blocks = min(Tile::F, max(0, (p.cols - row + 15) / 16));
    int begin = blocks ? to_sgpr(p.starts[block0]) : 0, count = blocks ? to_sgpr(p.starts[block0 + blocks]) - begin : 0;
    int my_row = 0, my_label = -1;
    float my_rest = 0.f;
    auto entries = [&](int first) {
        my_label = -1;
        my_rest = 0.f;
        if (first + lane < count) {
            my_row = p.list[begin + first + lane];
            my_label = p.labels.at(my_row, p.V);
            my_rest = p.dw_rest[my_row];
        }
    };
    entries(0);
    asm volatile("" : "+v"(begin), "+v"(count));   // (in vector registers over the product, which needs the scalar ones)
    v4f acc[Tile::F][Tile::F];
    Tile::template product<true, true>(smem, operand_across(p.dl, 2ull * p.pitch, row0, p.dw_rows),
                                       operand_across(p.x, 2ull * p.K, col0, p.dw_rows), p.dw_rows, acc);
    begin = to_sgpr(begin);
    count = to_sgpr(count);
    // Their columns of x, 64 rows at a time, in this wave's part of the LDS that the product is done with, several rows under way at once,
    // and their labels and remainders behind all waves' rows. A block's 16 classes take 32 of these rows at a time by matrix instructions:
    // [classes x rows], the remainder where the row's label is the class, in two numbers of bf16, times [rows x columns]. (Row by row, a row
    // was 0.2 us of one wave: 8192 rows of one label of 1000, K = 1024, backward 2083 us; now 418, with labels spread evenly 219.)
    constexpr int kRowBytes = 2 * Tile::kPatch, kLanes = kRowBytes / 16, kAtOnce = 64 / kLanes;   // lanes of a row, rows of a load
    static_assert(4 * 64 * (kRowBytes + 8) <= Tile::kLds);
    block_barrier();
    uint8_t* mine = smem + w * 64 * kRowBytes;
    uint8_t* info = smem + 4 * 64 * kRowBytes + w * 512;
    const uint32_t rows_at = (uint32_t)(uintptr_t)mine + (8 * g + (r >> 2)) * kRowBytes + (r & 3) * 8;   // a lane's place in the transposing reads
    auto stage = [&](int first) {
        const int n = min(64, count - first), piece = lane % kLanes * 8;
        *(v2i*)(info + lane * 8) = v2i{my_label, __float_as_int(my_rest)};
        for (int e0 = 0; e0 < (n + 31) / 32 * 32; e0 += 4 * kAtOnce) {   // (zeros behind the last one)
            v4i q[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int e = e0 + i * kAtOnce + lane / kLanes, at = __shfl(my_row, e & 63, 64);
                q[i] = v4i{0, 0, 0, 0};
                if (e < n && col + piece < p.K) q[i] = *(const v4i*)(p.x + (size_t)at * p.K + col + piece);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) *(v4i*)(mine + (e0 / kAtOnce + i) * 1024 + lane * 16) = q[i];
        }
    };
    if (count > 0) stage(0);
    int staged = 0;   // the first of the 64
#pragma unroll
    for (int m = 0; m < Tile::F; ++m) {
        v4f v[Tile::F];
        Tile::read_row(acc[m], v);
        const int block = block0 + m;
        while (count > 0) {
            const uint64_t in = __ballot(my_label >= 0 && my_label / 16 == block);
            for (int h = 0; h < 2; ++h) {
                if (!(uint32_t)(in >> 32 * h)) continue;
                v4i value, rest;   // of this lane's class, rows 32 h + 8 g .. +8
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const v4i two = *(const v4i*)(info + (32 * h + 8 * g + 2 * i) * 8);
                    const float a = two.x == 16 * block + r ? __int_as_float(two.y) : 0.f, b = two.z == 16 * block + r ? __int_as_float(two.w) : 0.f;
                    value[i] = (int)pack_bf16(a, b);
                    rest[i] = (int)pack_bf16(a - bf16_value(a), b - bf16_value(b));
                }
#pragma unroll
                for (int c = 0; c < Tile::F; ++c) {
                    const uint32_t at = rows_at + 32 * h * kRowBytes + c * 32;
                    const v2i lo = lds_read_tr(at), hi = lds_read_tr(at + 4 * kRowBytes);
                    const v8bf_t x = __builtin_bit_cast(v8bf_t, v4i{lo.x, lo.y, hi.x, hi.y});
                    v[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, __builtin_bit_cast(v8bf_t, value), v[c], 0, 0, 0);
                    v[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, __builtin_bit_cast(v8bf_t, rest), v[c], 0, 0, 0);
                }
            }
            if (staged + 64 >= count || __builtin_amdgcn_readlane(my_label, 63) / 16 > block) break;
            staged += 64;
            entries(staged);
            stage(staged);
        }
        store_block_row(v, m, dw + (size_t)row * p.K + col, p.K, p.cols - row, p.K - col);
        slot_fence();
    }
}

// dx = the splits' sums, added in order, and the label's remainder (a thread: four columns of a row; K a multiple of 8).
__global__ __launch_bounds__(256) void head_dx_reduce_kernel(const float* __restrict__ sums, int splits, int M, int V, int K, HeadLabels labels,
                                                             const float* __restrict__ resid, const uint16_t* __restrict__ W,
                                                             uint16_t* __restrict__ dx) {
    const size_t n = (size_t)M * K, at = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (at >= n) return;
    const int m = (int)(at / K), label = labels.at(m, V);
    v4f v = *(const v4f*)(sums + at);
#pragma unroll 8
    for (int s = 1; s < splits; ++s) v += *(const v4f*)(sums + (size_t)s * n + at);   // (loads several at a time)
    if (label >= 0) v += resid[m] * bf16_quad(W + (size_t)label * K + (at - (size_t)m * K));
    *(v2i*)(dx + at) = v2i{(int)pack_bf16(v.x, v.y), (int)pack_bf16(v.z, v.w)};
}

static int tiles_of(int n, int tile) { return (n + tile - 1) / tile; }
static size_t up256(size_t n) { return (n + 255) / 256 * 256; }
static LayoutChoice head_choice(int rows, int cols, int k) {   // a product of rows x cols over k
    auto tiles = [&](int tile) { return (double)tiles_of(rows, tile) * tiles_of(cols, tile); };
    return choose_layout({tiles(256), tiles(128), tiles(64)}, tiles_of(k, kLayoutStep), moe_num_compute_units());
}

// forward: label logits, then the partial results. bytes: what any number of rows up to M takes, so that a workspace for the largest batch
// serves the smaller ones, whose tiles may be smaller and their partial results more.
struct HeadForwardPlan {
    LayoutChoice tile;
    int blocks;   // columns of a partial result: a wave's patch
    size_t label_logit, partial, bytes;
    HeadForwardPlan(int M, int V, int K) {
        tile = head_choice(M, V, K);
        blocks = 2 * tiles_of(V, tile == kLayout256 ? 256 : tile == kLayout64Deep ? 64 : 128);
        label_logit = 0;
        partial = up256((size_t)M * 4);
        const size_t rows64 = std::min(M, 64 * (moe_num_compute_units() / tiles_of(V, 64)));   // most that 64x64 tiles are taken for
        bytes = partial + up256(std::max((size_t)M * tiles_of(V, 128), rows64 * tiles_of(V, 64)) * 2 * sizeof(float2));
    }
};
// backward: dl of a piece, then the fp32 sums of dx. parts: the numbers of bf16 that dl is held in, 2 for dW in fp32.
struct HeadBackwardPlan {
    int piece;   // columns of a piece, a multiple of 256
    LayoutChoice logits;
    LayoutChoice grads;
    int splits, split_cols;
    size_t rest, starts, list, x, dl, sums, bytes;   // rest: `parts` remainders of each row
    // Bytes of dl and the second copy of x, which are held together. Neither grows when there are fewer rows.
    static long long held_for_dl(long long M, int V, int K) {
        const long long fill = 256ll * tiles_of(moe_num_compute_units(), tiles_of(K, 256));
        return std::max(512ll << 20, std::min({2 * M * fill, 4ll << 30, 512 * M * tiles_of(V, 512)}));
    }
    // What any number of rows up to M takes, with either type of dW. Fewer rows than `cut` have dx tiles for less than the CUs' places, and up to
    // 1 + 9/8 places / tiles sums of dx (per_split below is at least 8/9 of all K-steps over the places): bounded by the places' tiles.
    static size_t bytes_up_to(int M, int V, int K) {
        const long long all = (long long)tiles_of(V, 256) * 256, cus = moe_num_compute_units();
        auto uncut = [&](long long m) {
            const long long held = held_for_dl(m, V, K), copy = 2 * m * K;
            const long long one = std::min(std::max(held, 512 * m), 2 * m * all);
            const long long two = std::min(std::max({held - copy, held / 4, 1024 * m}), 4 * m * all) + copy;
            return up256((size_t)m * 8) + up256((size_t)m * 4) + up256(((size_t)tiles_of(V, 256) * 16 + 1) * 4) + up256((size_t)copy) +
                   up256((size_t)std::max(one, two)) + up256((size_t)m * K * 4) + 1024;
        };
        const long long cut = std::min((long long)M, std::max(256 * ((cus - 1) / tiles_of(K, 256)), 128 * ((2 * cus - 1) / tiles_of(K, 128))));
        auto tile_bytes = [&](long long t) { return 4 * std::min(t, cut) * std::min<long long>(t, K); };
        const long long sums = std::min(4 * cut * K * tiles_of(tiles_of(V, kLayoutStep), 8), std::max(cus * tile_bytes(256), 2 * cus * tile_bytes(128)) * 9 / 8);
        return std::max(uncut(M), uncut(cut) + up256((size_t)sums));
    }
    HeadBackwardPlan(int M, int V, int K, int parts) {
        // Pieces of 512 MB: a piece's items of dx are the longer and its tiles the more, the fewer pieces there are (backward, us, pieces of
        // 128 / 256 / 512 / 2048 MB: 4096 x 201088 x 2880 11492 / 11737 / 11571 / 11331, 8192 x 129280 x 7168 34150 / 33106 / 32755 /
        // 33109, 16384 x 50257 x 1024 7282 / 5552 / 4747 / 4644). Where that gives dW fewer tiles than CUs (many rows, few columns of x: tiles
        // of M / 64 K-steps, and the rest of the chip idle), as many classes as fill the CUs, up to 4 GB and half of dl (512 MB / 1 / 2 / 4 GB
        // at most: 65536 x 32000 x 1024 15444 / 11947 / 11416 / 11394, 262144 x 32000 x 1024 180717 / 104194 / 65851 / 47530).
        // Rows of at most 4 MB: 32-bit offsets inside a K-step's rows.
        // dl in two parts, and the second copy of x, are held in the same bytes: pieces of half the classes and less.
        const long long copies = 2ll * M * K * (parts - 1);
        long long held = held_for_dl(M, V, K);
        held = std::max(held - copies, held / 4);
        const long long most = std::min(held / (2ll * parts * M), 1ll << 21) / 256 * 256, all = (long long)tiles_of(V, 256) * 256;
        piece = (int)std::max(256ll, std::min(most, all));
        const int cols = std::min(piece, V);
        logits = head_choice(M, cols, K);
        // dx and dW together. dx's contraction is cut to the K-steps that a workgroup's place has (8 at least); the time of a tile's kernel is
        // that of all K-steps over the places, or of the longest item if that is longer (large: one workgroup a CU; small: two).
        // (Gradients, us, without regard to the longest item and without LayoutTile128Deep / so: 973 x 1187 x 792 79 / 48, 395 x 1029 x 3552
        // 59 / 43, 4096 x 4096 x 1024 195 / 143, 1024 x 8192 x 1024 73 / 73.)
        const int cus = moe_num_compute_units(), steps_v = tiles_of(cols, kLayoutStep), steps_m = tiles_of(parts * M, kLayoutStep);
        struct Cut { int splits, split_cols; bool deep; double us; };
        auto cut = [&](int tile) {
            const double dx = (double)tiles_of(M, tile) * tiles_of(K, tile), dw = (double)tiles_of(cols, tile) * tiles_of(K, tile);
            const int places = tile == 256 ? cus : 2 * cus;
            const int per_split = std::max(8, (int)std::min((double)steps_v, (dx * steps_v + dw * steps_m) / places));
            Cut c;
            c.split_cols = tiles_of(steps_v, tiles_of(steps_v, per_split)) * kLayoutStep;
            c.splits = tiles_of(cols, c.split_cols);
            const double fixed = tile == 256 ? kLargeFixed : kSmallFixed, items = dx * c.splits + dw;
            const double along = tile == 256 ? kLargeStep : kSmallStepAlong, across = tile == 256 ? kLargeStep : kSmallStepAcross;
            const double longest = std::max(along * std::min(per_split, steps_v), across * steps_m);
            c.us = std::max((dx * (fixed + along * steps_v) + dw * (fixed + across * steps_m)) / places, fixed + longest);
            if (tile == 128 && items <= cus) c.us = kSmallFixed + kDeepStep * std::max(std::min(per_split, steps_v), steps_m);   // LayoutTile128Deep
            c.deep = tile == 128 && items <= cus;
            return c;
        };
        const Cut large = cut(256), small = cut(128);
        grads = large.us < small.us ? kLayout256 : small.deep ? kLayout128Deep : kLayout128;
        splits = (grads == kLayout256 ? large : small).splits;
        split_cols = (grads == kLayout256 ? large : small).split_cols;
        rest = 0;
        list = up256((size_t)M * 4 * parts);
        starts = list + up256((size_t)M * 4);
        x = starts + up256(((size_t)tiles_of(V, 256) * 16 + 1) * 4);
        dl = x + up256((size_t)M * K * 2 * parts);
        sums = dl + up256((size_t)M * piece * 2 * parts);
        bytes = std::max(bytes_up_to(M, V, K), sums + (piece < V || splits > 1 ? up256((size_t)splits * M * K * 4) : 0));
    }
};

static int head_check(int M, int V, int K) {
    // (a launch has fewer than 2^32 threads: the join takes 64 a row. So fewer than 2^24 workgroups of 256: half of it for the tiles, or for each
    // part of the gradients' launch, a quarter each for the copies of kHeadCopyRows rows and for the sort by label)
    if (M <= 0 || V <= 0 || K <= 0 || (K % 8) != 0 || M >= (1 << 25) || V >= (1 << 30) || K > (1 << 21)) return HK_ERR_BAD_SHAPE;
    const long long tm = tiles_of(M, 128), tv = tiles_of(V, 128), tk = tiles_of(K, 128), most = 1ll << 23;
    if (tm * tv >= most || tm * tk >= most || tv * tk >= most) return HK_ERR_BAD_SHAPE;
    return HK_OK;
}

template <typename Tile, typename... P, typename... A>
static int launch_head(void (*kern)(P...), DeviceOnce& once, long long tiles, hipStream_t s, A... args) {
    if (!set_lds_limit_once((const void*)kern, Tile::kLds, once)) return HK_ERR_LAUNCH;
    hipLaunchKernelGGL(kern, dim3((unsigned)tiles), dim3(256), Tile::kLds, s, args...);
    return hipGetLastError() == hipSuccess ? HK_OK : HK_ERR_LAUNCH;
}

template <typename Tile>
static int launch_logits(const uint16_t* x, const uint16_t* W, HeadLabels labels, int M, int V, int K, float2* partial, float* label_logit,
                         hipStream_t s) {
    static DeviceOnce once;
    const int tm = tiles_of(M, Tile::kTile), tv = tiles_of(V, Tile::kTile);
    return launch_head<Tile>(head_logits_kernel<Tile>, once, (long long)tm * tv, s, x, W, labels, M, V, K, tm, tv,
                             raster_band(2ll * K * ((long long)M + V), tv), partial, label_logit);
}
template <typename Tile>
static int launch_dlogits(const uint16_t* x, const uint16_t* W, HeadLabels labels, const float* lse, const float* dloss, int M, int V, int K,
                          int v0, int cols, int pitch, uint16_t* dl, uint16_t* dl_rest, HeadRemainders rest, HeadRows rows, hipStream_t s) {
    static DeviceOnce once;
    const int tm = tiles_of(M, Tile::kTile), tv = tiles_of(cols, Tile::kTile);
    return launch_head<Tile>(head_dlogits_kernel<Tile>, once, (long long)tm * tv + rows.groups + rows.copies, s, x, W, labels, lse, dloss, M, V, K, v0,
                             (cols + 7) / 8 * 8, pitch, tm, tv, raster_band(2ll * K * ((long long)M + cols), tv), dl, dl_rest, rest, rows);
}
template <typename Tile, typename T>
static int launch_gradients(HeadPiece p, bool dx, T* dw, hipStream_t s) {
    static DeviceOnce once;
    p.tiles_m = tiles_of(p.M, Tile::kTile);
    p.tiles_k = tiles_of(p.K, Tile::kTile);
    p.tiles_v = dw ? tiles_of(p.cols, Tile::kTile) : 0;
    p.band_dx = raster_band(2ll * p.cols * ((long long)p.M + p.K), p.tiles_k);
    p.band_dw = raster_band(2ll * p.dw_rows * ((long long)p.cols + p.K), p.tiles_k);
    p.splits = dx ? tiles_of(p.cols, p.split_cols) : 0;
    p.dw_first = p.dw_rows > p.split_cols;
    const long long items = (long long)p.splits * p.tiles_m * p.tiles_k + (long long)p.tiles_v * p.tiles_k;
    return launch_head<Tile>(head_gradients_kernel<Tile, T>, once, items, s, p, dw ? dw + (size_t)p.v0 * p.K : nullptr);
}

}  // namespace hk

extern "C" size_t hk_linear_cross_entropy_workspace_bytes(int M, int V, int K, int backward) {
    using namespace hk;
    if (head_check(M, V, K) != HK_OK) return 0;
    const size_t f = HeadForwardPlan(M, V, K).bytes;
    return backward ? std::max({f, HeadBackwardPlan(M, V, K, 1).bytes, HeadBackwardPlan(M, V, K, 2).bytes}) : f;
}

extern "C" int hk_linear_cross_entropy(const void* x_bf16, const void* w_bf16, const void* labels, int label_type, float* loss,
                                       float* lse, int M, int V, int K, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace hk;
    if (!x_bf16 || !w_bf16 || !labels || !loss || !lse) return HK_ERR_NULL_POINTER;
    if (const int st = head_check(M, V, K)) return st;
    if (label_type != 0 && label_type != 1) return HK_ERR_UNSUPPORTED;
    if (((uintptr_t)x_bf16 | (uintptr_t)w_bf16 | (uintptr_t)workspace) & 15u) return HK_ERR_BAD_ALIGNMENT;
    const HeadForwardPlan L(M, V, K);
    if (!workspace || workspace_bytes < L.bytes) return HK_ERR_WORKSPACE;
    const hipStream_t s = (hipStream_t)stream;
    float2* partial = (float2*)((uint8_t*)workspace + L.partial);
    float* label_logit = (float*)((uint8_t*)workspace + L.label_logit);
    const HeadLabels lab{labels, label_type};
    const uint16_t *x = (const uint16_t*)x_bf16, *w = (const uint16_t*)w_bf16;
    auto logits = [&]<typename Tile>() { return launch_logits<Tile>(x, w, lab, M, V, K, partial, label_logit, s); };
    const int st = L.tile == kLayout256       ? logits.template operator()<LayoutTile256>()
                   : L.tile == kLayout128     ? logits.template operator()<LayoutTile128>()
                   : L.tile == kLayout128Deep ? logits.template operator()<LayoutTile128Deep>()
                                              : logits.template operator()<LayoutTile64Deep>();
    if (st != HK_OK) return st;
    hipLaunchKernelGGL(head_loss_kernel, dim3((M + 15) / 16), dim3(16 * kJoin), 0, s, (const float2*)partial, (const float*)label_logit, lab, M, V,
                       L.blocks, loss, lse);
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
    const int parts = dw_or_null && dw_type == 1 ? 2 : 1;
    const HeadBackwardPlan L(M, V, K, parts);
    if (!workspace || workspace_bytes < L.bytes) return HK_ERR_WORKSPACE;
    const hipStream_t s = (hipStream_t)stream;
    uint8_t* ws = (uint8_t*)workspace;
    const HeadLabels lab{labels, label_type};
    const uint16_t *x = (const uint16_t*)x_bf16, *w = (const uint16_t*)w_bf16;
    uint16_t* dl = (uint16_t*)(ws + L.dl);
    uint16_t* dl_rest = parts == 2 ? dl + (size_t)M * L.piece : nullptr;
    const bool want_dx = dx_bf16_or_null != nullptr;
    const HeadRemainders rest{(float*)(ws + L.rest), (float*)(ws + L.rest) + (parts == 2 ? M : 0)};
    int32_t *starts = (int32_t*)(ws + L.starts), *list = (int32_t*)(ws + L.list);
    uint16_t* x0 = (uint16_t*)(ws + L.x);
    HeadPiece p{dl, w, x0, (float*)(ws + L.sums), lab, rest.one, rest.two, starts, list, (uint16_t*)dx_bf16_or_null, M, V, K, 0, 0, L.piece, parts * M, 0, 0, 0, 0, 0, 0,
                L.split_cols,
                false, false, L.splits > 1, false};
    for (int v0 = 0; v0 < V; v0 += L.piece) {
        p.v0 = v0;
        p.cols = V - v0 < L.piece ? V - v0 : L.piece;
        p.first = v0 == 0;
        p.last = v0 + p.cols == V;
        const bool first_dw = dw_or_null && v0 == 0;
        const HeadRows rows{starts, list, x0, parts == 2 ? x0 + (size_t)M * K : nullptr, first_dw ? tiles_of(V, 256) : 0,
                            first_dw ? tiles_of(M, kHeadCopyRows) : 0};
        auto dlogits = [&]<typename Tile>() {
            return launch_dlogits<Tile>(x, w, lab, lse, dloss, M, V, K, v0, p.cols, L.piece, dl, dl_rest, rest, rows, s);
        };
        int st = L.logits == kLayout256       ? dlogits.template operator()<LayoutTile256>()
                 : L.logits == kLayout128     ? dlogits.template operator()<LayoutTile128>()
                 : L.logits == kLayout128Deep ? dlogits.template operator()<LayoutTile128Deep>()
                                              : dlogits.template operator()<LayoutTile64Deep>();
        if (st != HK_OK) return st;
        auto gradients = [&]<typename Tile>() {
            return dw_type == 0 ? launch_gradients<Tile>(p, want_dx, (uint16_t*)dw_or_null, s)
                                : launch_gradients<Tile>(p, want_dx, (float*)dw_or_null, s);
        };
        st = L.grads == kLayout256   ? gradients.template operator()<LayoutTile256>()
             : L.grads == kLayout128 ? gradients.template operator()<LayoutTile128>()
                                     : gradients.template operator()<LayoutTile128Deep>();
        if (st != HK_OK) return st;
        if (V - v0 <= L.piece) break;
    }
    if (want_dx && L.splits > 1) {
        const size_t n = (size_t)M * K;
        hipLaunchKernelGGL(head_dx_reduce_kernel, dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, s, (const float*)(ws + L.sums),
                           L.splits, M, V, K, lab, (const float*)rest.one, w, (uint16_t*)dx_bf16_or_null);
        if (hipGetLastError() != hipSuccess) return HK_ERR_LAUNCH;
    }
    return HK_OK;
}
