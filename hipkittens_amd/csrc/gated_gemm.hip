// The gated feed-forward block in bf16: both projections, the activation and the product in one kernel, and the way back through the
// down projection and the activation in another. Rows of a dense block, or grouped by expert (expert_offsets [E+1], on the device).
//
//   forward    g[r, c] = x[r] . Wg[c], u[r, c] = x[r] . Wu[c], h = (u' + b) g' s(a g') with g' = min(g, l), u' = clamp(u, -l, l),
//              s the logistic function: SiLU(g) u is a = 1, l = inf, b = 0, the clamped form b = 1 with its a and l
//   backward   dh = dy W2, dg = [g <= l] dh (u' + b) s (1 + a g' (1 - s)), du = [|u| <= l] dh g' s, and h again, for dW2 = dy^T h
//
// What follows the backward kernel are products: dx = dgu W13, dW13 = dgu^T x. g and u are kept in bf16 (gate_up [R, 2I], in the
// order of W13's rows), each rounded once; h in the forward pass comes from the unrounded values.
//
// fp32 accumulation and activation, one rounding. The products are those of gemm_layouts_ring.h, which bound both kernels; in the forward one
// every 32 rows of the weight tile in LDS are 16 gate rows and the 16 up rows of the same columns (kPairs), so that both values of
// an element are in one lane's accumulators and the activation needs no exchange between lanes.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>

#include "gemm_skinny.h"
#include "moe_grouped.h"
#include "../../include/hk355.h"

namespace hk {

// The activation. SiLU has a form of its own: the backward kernel's epilogue, 256 elements a lane, is bound by their instructions (65536 rows of 32
// experts, N = 7168, I = 2048, in one form for both 1780 us). A NaN stays one: the clamps are IEEE's minimum and maximum.
struct GateArgs { float alpha, limit; };
template <bool CLAMPED>
struct Gate {
    GateArgs a;
    __device__ __forceinline__ static float sig(float z) {
        return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f));
    }
    __device__ __forceinline__ float top(float g) const { return CLAMPED ? __builtin_elementwise_minimum(g, a.limit) : g; }
    __device__ __forceinline__ float lin(float u) const {
        return CLAMPED ? __builtin_elementwise_maximum(__builtin_elementwise_minimum(u, a.limit), -a.limit) + 1.0f : u;
    }
    __device__ __forceinline__ float value(float g, float u) const {
        const float t = top(g);
        return lin(u) * (t * sig(CLAMPED ? a.alpha * t : t));
    }
    // h of (g, u), and from dh the gradients of both
    __device__ __forceinline__ float gradients(float g, float u, float dh, float& dg, float& du) const {
        const float t = top(g), v = lin(u), z = CLAMPED ? a.alpha * t : t, s = sig(z), ts = t * s;
        // s (1 + z (1 - s)); alpha comes last, behind products that are 0 where s is 0 or 1: z may have left fp32 (a gate value
        // that is the type's lowest, as a mask), and infinity times 0 is no number
        dg = dh * v * (CLAMPED ? __builtin_fmaf(a.alpha, ts * (1.0f - s), s) : __builtin_fmaf(ts, 1.0f - s, s));
        du = dh * ts;
        if (CLAMPED) {
            dg = g > a.limit ? 0.f : dg;
            du = __builtin_fabsf(u) > a.limit ? 0.f : du;
        }
        return v * ts;
    }
};

struct GatedForward {
    const uint16_t *x, *w13;
    const int32_t* offsets;   // null: dense
    uint16_t *h, *gate_up;    // gate_up null: not wanted
    int R, E, I, K, tiles_n, interleaved, clamped;
    GateArgs gate;
};

// Stores of a wave's patch into rows of bf16, sixteen rows at a time, through a buffer descriptor that ends behind the last row (its range
// check takes the scalar offset, which holds the row block, with it): a lane has one offset for each piece of 16 bytes, out of range where the row
// ends in front of it, and a store is one instruction. (Through pointers, a test and an address for each, a sixth of the backward kernel's
// epilogue were those.) Written as statements of their own: behind a store of 16 bytes with a scalar offset its data may not be overwritten for
// two wait states, which the compiler does not keep here.
constexpr uint32_t kOutside = 0x80000000u;
template <int PIECES>
struct PatchRows {
    v4i srd;
    uint32_t pitch, at[PIECES];
    // first: the patch's first row; rows: what is left of them; column(i): the first column of the lane's piece i, of `cols` columns of `bytes` bytes
    template <typename C>
    __device__ __forceinline__ PatchRows(uint16_t* first, uint32_t pitch_bytes, int rows, int cols, uint32_t bytes, C&& column) {
        pitch = to_sgpr(pitch_bytes);
        srd = make_srd(first, rows > 0 ? (uint32_t)min(rows, kRingTile) * pitch_bytes : 0u);   // (at most 256 rows of 4 MB)
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int c = column(i);
            at[i] = c < cols ? (lane_id() & 15) * pitch_bytes + (uint32_t)c * bytes : kOutside;
        }
    }
    __device__ __forceinline__ void store(v4i v, int i, int m, uint32_t more = 0) const {
        asm volatile("buffer_store_dwordx4 %0, %1, %2, %3 offen\n\ts_nop 1" ::"v"(v), "v"(at[i]), "s"(srd), "s"(to_sgpr(16 * m * pitch + more)) : "memory");
    }
    __device__ __forceinline__ void store(v2i v, int i, int m, uint32_t more = 0) const {
        asm volatile("buffer_store_dwordx2 %0, %1, %2, %3 offen" ::"v"(v), "v"(at[i]), "s"(srd), "s"(to_sgpr(16 * m * pitch + more)) : "memory");
    }
};
// One matrix of F column blocks, in store_block_row's places.
template <int F>
struct PatchMatrix {
    PatchRows<(F + 1) / 2> rows;
    __device__ __forceinline__ PatchMatrix(uint16_t* first, uint32_t pitch_bytes, int n, int col, int cols)
        : rows(first, pitch_bytes, n, cols, 2, [&](int i) {
              const int q = lane_id() >> 4;
              return col + 32 * i + (2 * i + 1 < F ? 8 * (q >> 1) + 16 * (q & 1) : 4 * q);
          }) {}
    // more: bytes from the matrix's columns to those that are written
    __device__ __forceinline__ void store(const v4f (&v)[F], int m, uint32_t more = 0) const {
#pragma unroll
        for (int i = 0; i < F / 2; ++i) {
            v4i out;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const v4f a = v[2 * i], b = v[2 * i + 1];
                const auto s = __builtin_amdgcn_permlane16_swap(pack_bf16(a[2 * h], a[2 * h + 1]), pack_bf16(b[2 * h], b[2 * h + 1]), false, false);
                out[h] = (int)s[0];
                out[2 + h] = (int)s[1];
            }
            rows.store(out, i, m, more);
        }
        if constexpr (F % 2 == 1) rows.store(v2i{(int)pack_bf16(v[F - 1].x, v[F - 1].y), (int)pack_bf16(v[F - 1].z, v[F - 1].w)}, F / 2, m, more);
    }
};
// Gate and up values, or their gradients: the one's columns behind the other's, or alternating.
template <int F, bool INTERLEAVED>
struct PatchPairs {
    PatchMatrix<F> rows;
    uint32_t half;
    __device__ __forceinline__ PatchPairs(uint16_t* first, int n, int col, int I) : rows(first, 4u * I, n, col, I), half(to_sgpr(2u * I)) {}
    __device__ __forceinline__ void store(const v4f (&g)[F], const v4f (&u)[F], int m) const {
        rows.store(g, m);
        rows.store(u, m, half);
    }
};
template <int F>
struct PatchPairs<F, true> {
    PatchRows<F> rows;
    __device__ __forceinline__ PatchPairs(uint16_t* first, int n, int col, int I)
        : rows(first, 4u * I, n, I, 4, [&](int i) { return col + 16 * i + 4 * (lane_id() >> 4); }) {}
    __device__ __forceinline__ void store(const v4f (&g)[F], const v4f (&u)[F], int m) const {
#pragma unroll
        for (int n = 0; n < F; ++n)
            rows.store(v4i{(int)pack_bf16(g[n].x, u[n].x), (int)pack_bf16(g[n].y, u[n].y), (int)pack_bf16(g[n].z, u[n].z), (int)pack_bf16(g[n].w, u[n].w)}, n, m);
    }
};

// The kept gate and up values of a wave's patch, row block by row block (16 rows) through LDS: the first blocks, as many as what the product leaves of a
// CU's LDS holds, in front of the product (all of a 64x64 tile's, half of those of a 128x128 tile with a CU to itself; 300 rows of 2880 x 2880 17.3
// us, so 16.4), the others through the wave's share of the LDS that the product is done with, as many under way at once as that holds. Rows of
// LDS hold 16-byte chunk c of row r at c ^ swz(r): a read of a column block touches every bank once. (Read straight into registers, a block at a
// time: 65536 rows of 32 experts, N = 7168, I = 2048 1864 us where this takes 1780, with the activation in one form.)
template <typename Tile, bool INTERLEAVED>
struct GateUpLoads {
    static constexpr int F = Tile::FC, kBlocks = Tile::F, kBlockBytes = Tile::kPatchCols * 64, kLoads = kBlockBytes / 1024;
    static constexpr int kRoom = 160 * 1024 / (Tile::kLds > 80 * 1024 ? 1 : 2) - Tile::kLds;
    static constexpr int kAhead = std::min(kRoom / 4 / kBlockBytes, kBlocks), kRest = kBlocks - kAhead;
    static constexpr int kLds = Tile::kLds + 4 * kAhead * kBlockBytes;
    static constexpr int kSlots = std::min(Tile::kLds / 4 / kBlockBytes, kRest);
    static_assert(kRest == 0 || (kSlots >= 1 && (kSlots - 1) * kLoads < 64));
    // 16-byte chunks of a row of LDS: of its gate or of its up values, or of both where they alternate; rows of a load
    static constexpr uint32_t kChunks = INTERLEAVED ? Tile::kPatchCols / 4 : Tile::kPatchCols / 8, kLoadRows = 64 / kChunks;
    v4i srd;
    uint32_t lds, lds_ahead, voff, pitch, half;   // voff: the lane's place in an even load's first row; half: bytes between a row's gate and up values

    __device__ __forceinline__ static uint32_t swz(uint32_t r) { return kChunks >= 16 ? r & 15u : (r / (16u / kChunks)) & (kChunks - 1); }
    // at: the patch's first row; col: its first column of I; rows: what is left of the rows (none: everything reads as zeros)
    __device__ __forceinline__ GateUpLoads(uint8_t* smem, const uint16_t* at, int col, int I, int rows) {
        pitch = to_sgpr(4u * (uint32_t)I);
        half = 2u * (uint32_t)I;
        srd = make_srd(at, rows > 0 ? (uint32_t)rows * pitch : 0u);   // (at most 256 rows of 4 MB)
        lds = to_sgpr((uint32_t)(uintptr_t)smem + wave_id() * (Tile::kLds / 4));
        lds_ahead = to_sgpr((uint32_t)(uintptr_t)smem + Tile::kLds + wave_id() * (kAhead * kBlockBytes));
        voff = lane_id() / kChunks * pitch + (uint32_t)col * (INTERLEAVED ? 4u : 2u);
    }
    __device__ __forceinline__ uint32_t slot(int m) const {
        return m < kAhead ? lds_ahead + m * kBlockBytes : lds + (m - kAhead) % std::max(kSlots, 1) * kBlockBytes;
    }
    __device__ __forceinline__ void issue(int m) const {
        const uint32_t lane = lane_id(), dst = slot(m);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {   // the gate values' loads, then the up values'
            const uint32_t k = INTERLEAVED ? i : i % (kLoads / 2);
            const uint32_t row = k * kLoadRows + lane / kChunks;
            const uint32_t at = voff + (16 * m + k * kLoadRows) * pitch + ((lane % kChunks) ^ swz(row)) * 16u + (!INTERLEAVED && i >= kLoads / 2 ? half : 0u);
            dma16(srd, to_sgpr(dst + i * 1024), at, 0u);
        }
    }
    __device__ __forceinline__ void read(int m, v4f (&g)[F], v4f (&u)[F]) const {
        const uint32_t r = lane_id() & 15, q = lane_id() >> 4, at = slot(m) + r * (kChunks * 16);
#pragma unroll
        for (int n = 0; n < F; ++n) {
            if constexpr (INTERLEAVED) {
                const v4i in = *(lds_v4i_t*)(uintptr_t)(at + ((4 * n + q) ^ swz(r)) * 16);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    g[n][j] = __uint_as_float((uint32_t)in[j] << 16);
                    u[n][j] = __uint_as_float((uint32_t)in[j] & 0xffff0000u);
                }
            } else {
                const uint32_t p = at + ((2 * n + (q >> 1)) ^ swz(r)) * 16 + (q & 1) * 8;
                const v2i a = *(lds_v2i_t*)(uintptr_t)p, b = *(lds_v2i_t*)(uintptr_t)(p + kBlockBytes / 2);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    g[n][2 * j] = __uint_as_float((uint32_t)a[j] << 16);
                    g[n][2 * j + 1] = __uint_as_float((uint32_t)a[j] & 0xffff0000u);
                    u[n][2 * j] = __uint_as_float((uint32_t)b[j] << 16);
                    u[n][2 * j + 1] = __uint_as_float((uint32_t)b[j] & 0xffff0000u);
                }
            }
        }
    }
};

// A tile takes kTileCols / 2 columns of h.
template <typename Tile, bool CLAMPED, bool INTERLEAVED>
__global__ __launch_bounds__(256) void gated_gemm_kernel(GatedForward p) {
    extern __shared__ __attribute__((aligned(2048))) uint8_t smem[];
    const GroupedTile t = grouped_tile(p.offsets, p.E, p.R, Tile::kTile, p.tiles_n, p.K, 2 * p.I, xcd_chunk_order(blockIdx.x, gridDim.x, kCuPerXcd));
    if (t.expert < 0) return;
    const int col0 = t.tile_n * (Tile::kTileCols / 2);
    const uint16_t* w = p.w13 + (size_t)t.expert * 2 * p.I * p.K;
    const size_t pitch = 2ull * p.K;   // bytes
    v4f acc[Tile::F][Tile::FC];
    Tile::template product<kAlong, kPairs>(
        smem, operand_along(p.x, pitch, t.row0, t.row0 + t.rows, p.K),
        operand_pairs(w, w + (INTERLEAVED ? (size_t)p.K : (size_t)p.I * p.K), INTERLEAVED ? 2 * pitch : pitch, col0, p.I, p.K), p.K, acc);
    const Gate<CLAMPED> gate{p.gate};
    constexpr int B = Tile::FC / 2;   // blocks of 16 columns of h
    const int wv = wave_id(), row = (wv >> 1) * Tile::kPatch, col = col0 + (wv & 1) * (Tile::kPatchCols / 2), rows = t.rows - row;
    const size_t first = (size_t)(t.row0 + row);
    const PatchMatrix<B> out(p.h + first * p.I, 2u * p.I, rows, col, p.I);
    const PatchPairs<B, INTERLEAVED> pairs(p.gate_up + first * 2 * p.I, p.gate_up ? rows : 0, col, p.I);
#pragma unroll
    for (int m = 0; m < Tile::F; ++m) {
        v4f v[Tile::FC], g[B], u[B], h[B];
        Tile::read_row(acc[m], v);
#pragma unroll
        for (int n = 0; n < B; ++n) {
            g[n] = v[2 * n];
            u[n] = v[2 * n + 1];
#pragma unroll
            for (int j = 0; j < 4; ++j) h[n][j] = gate.value(g[n][j], u[n][j]);
        }
        out.store(h, m);
        if (p.gate_up) pairs.store(g, u, m);
        slot_fence();
    }
}

// Few rows of a dense block or an expert (decode): one pass over the weights at HBM speed, the skinny kernel with gate and up rows in its two halves.
struct GatedMma {
    static constexpr bool kScaled = false;
    static __device__ __forceinline__ void mma(v4f& acc, const v8i& b, const v8i& a) {
        auto half = [](const v8i& v, int h) { return __builtin_bit_cast(v8bf_t, h ? __builtin_shufflevector(v, v, 4, 5, 6, 7) : __builtin_shufflevector(v, v, 0, 1, 2, 3)); };
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(half(b, 0), half(a, 0), acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(half(b, 1), half(a, 1), acc, 0, 0, 0);
    }
};
struct GatedSkinnyOut {
    static constexpr bool kPairs = true;
    GatedForward p;
    int column_block;
    __device__ __forceinline__ int block() const { return column_block; }
    __device__ __forceinline__ uint32_t pitch() const { return (uint32_t)p.K * (p.interleaved ? 4u : 2u); }
    __device__ __forceinline__ const uint8_t* other() const { return (const uint8_t*)(p.w13 + (p.interleaved ? (size_t)p.K : (size_t)p.I * p.K)); }
    // columns c .. c + 4 of h
    __device__ __forceinline__ void store(int row, int c, const v4f& g, const v4f& u) const {
        float h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = p.clamped ? Gate<true>{p.gate}.value(g[j], u[j]) : Gate<false>{p.gate}.value(g[j], u[j]);
        *(v2i*)(p.h + (size_t)row * p.I + c) = v2i{(int)pack_bf16(h[0], h[1]), (int)pack_bf16(h[2], h[3])};
        if (!p.gate_up) return;
        uint16_t* at = p.gate_up + (size_t)row * 2 * p.I;
        if (p.interleaved) {
            *(v4i*)(at + 2 * c) = v4i{(int)pack_bf16(g.x, u.x), (int)pack_bf16(g.y, u.y), (int)pack_bf16(g.z, u.z), (int)pack_bf16(g.w, u.w)};
        } else {
            *(v2i*)(at + c) = v2i{(int)pack_bf16(g.x, g.y), (int)pack_bf16(g.z, g.w)};
            *(v2i*)(at + p.I + c) = v2i{(int)pack_bf16(u.x, u.y), (int)pack_bf16(u.z, u.w)};
        }
    }
};
template <int R, int NW, int D, int NF, bool NT, bool EXPERTS>
__global__ __launch_bounds__(64 * NW) void gated_skinny_kernel(GatedForward p) {
    extern __shared__ __attribute__((aligned(2048))) uint8_t smem[];
    int column_block = blockIdx.x;
    if constexpr (EXPERTS) {   // up to 16 R of an expert's rows
        const GroupedTile t = grouped_tile(p.offsets, p.E, p.R, 16 * R, p.tiles_n, p.K, 2 * p.I, xcd_chunk_order(blockIdx.x, gridDim.x, kCuPerXcd));
        if (t.expert < 0) return;
        column_block = t.tile_n;
        p.x += (size_t)t.row0 * p.K;
        p.w13 += (size_t)t.expert * 2 * p.I * p.K;
        p.h += (size_t)t.row0 * p.I;
        if (p.gate_up) p.gate_up += (size_t)t.row0 * 2 * p.I;
        p.R = t.rows;
    }
    gemm_skinny_body<GatedMma, R, NW, D, NF, NT>(smem, (const uint8_t*)p.x, (const uint8_t*)p.w13, nullptr, p.R, p.I, 2 * p.K, 1.0f,
                                                 SkinnyScales{nullptr, nullptr, 0, 0, 0}, GatedSkinnyOut{p, column_block});
}

struct GatedBackward {
    const uint16_t *dy, *w2;
    const int32_t* offsets;
    const uint16_t* gate_up;
    uint16_t *dgate_up, *h;   // dgate_up may be gate_up; h null: not wanted
    int R, E, N, I, tiles_n, interleaved, clamped;
    GateArgs gate;
};

template <typename Tile, bool CLAMPED, bool INTERLEAVED>
__global__ __launch_bounds__(256) void gated_dgrad_kernel(GatedBackward p) {
    extern __shared__ __attribute__((aligned(2048))) uint8_t smem[];
    const GroupedTile t = grouped_tile(p.offsets, p.E, p.R, Tile::kTile, p.tiles_n, p.N, p.I, xcd_chunk_order(blockIdx.x, gridDim.x, kCuPerXcd));
    if (t.expert < 0) return;
    const int col0 = t.tile_n * Tile::kTileCols;
    const int w = wave_id(), row = (w >> 1) * Tile::kPatch, col = col0 + (w & 1) * Tile::kPatchCols, rows = t.rows - row;
    const size_t first = (size_t)(t.row0 + row);
    typedef GateUpLoads<Tile, INTERLEAVED> Loads;
    const Loads kept(smem, p.gate_up + first * 2 * p.I, col, p.I, rows);
#pragma unroll
    for (int m = 0; m < Loads::kAhead; ++m) kept.issue(m);
    v4f acc[Tile::F][Tile::FC];
    Tile::template product<kAlong, kAcross>(smem, operand_along(p.dy, 2ull * p.N, t.row0, t.row0 + t.rows, p.N),
                                            operand_across(p.w2 + (size_t)t.expert * p.N * p.I, 2ull * p.I, col0, p.N), p.N, acc);
    const Gate<CLAMPED> gate{p.gate};
    const PatchMatrix<Tile::FC> out(p.h + first * p.I, 2u * p.I, p.h ? rows : 0, col, p.I);
    const PatchPairs<Tile::FC, INTERLEAVED> pairs(p.dgate_up + first * 2 * p.I, rows, col, p.I);
    wait_vmcnt<0>();   // the first blocks have landed, as the product's loads have
    if constexpr (Loads::kRest > 0) {
        block_barrier();   // everyone is done with the product's LDS
#pragma unroll
        for (int m = 0; m < Loads::kSlots; ++m) kept.issue(Loads::kAhead + m);
    }
    auto block = [&]<int m>() __attribute__((always_inline)) {
        v4f dh[Tile::FC], g[Tile::FC], u[Tile::FC], dg[Tile::FC], du[Tile::FC];
        // the block has landed: no more is under way than the loads issued behind its own (stores in between only make this wait longer)
        constexpr int last = m + Loads::kSlots < Tile::F ? m + Loads::kSlots : Tile::F;
        if constexpr (m >= Loads::kAhead) wait_vmcnt<(last - 1 - m) * Loads::kLoads>();
        kept.read(m, g, u);
        if constexpr (m >= Loads::kAhead && m + Loads::kSlots < Tile::F) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // ... and has been read
            kept.issue(m + Loads::kSlots);
        }
        Tile::read_row(acc[m], dh);
#pragma unroll
        for (int n = 0; n < Tile::FC; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float a, b;
                dh[n][j] = gate.gradients(g[n][j], u[n][j], dh[n][j], a, b);
                dg[n][j] = a;
                du[n][j] = b;
            }
        pairs.store(dg, du, m);
        if (p.h) out.store(dh, m);
        slot_fence();
    };
    [&]<int... m>(std::integer_sequence<int, m...>) __attribute__((always_inline)) {
        (block.template operator()<m>(), ...);
    }(std::make_integer_sequence<int, Tile::F>());
}

// Few rows of a dense block or an expert in the backward pass: one pass over W2, whose rows the contraction crosses. A workgroup owns NC columns of
// h and all rows of dy; its W waves take a part of the K-steps each, on their own: 64 rows of NC columns of W2 and as many elements of every
// row of dy into a ring of D stages of LDS that belongs to the wave, W2's read with the transposing loads (gemm_layouts.h). The waves' partial
// sums meet in LDS, in order, and the activation's gradients follow from what was kept, which the threads have loaded at the start.
// R: 16 rows of dy each.
template <int R, int W, int NC, int D>
struct SkinnyAcross {
    static constexpr int kWaves = W, kRow = 2 * NC, kW = 64 * kRow, kStage = kW + R * 2048, kRegion = D * kStage, kLds = kWaves * kRegion;
    static constexpr int kChunks = kRow / 16, kLoadRows = 64 / kChunks, kLoads = kW / 1024, kAll = kLoads + 2 * R, F = NC / 16;
    static_assert(kLds <= 160 * 1024 && (D - 1) * kAll < 64 && R * F * 1024 <= kRegion);
    // 16-byte chunk c of LDS row k lies at c ^ swz(k) (rows of 64 bytes: four share a line of the banks)
    static __device__ __forceinline__ uint32_t swz(uint32_t k) { return NC == 64 ? across_swz128(k) : 2u * ((k >> 3) & 1u); }
};
template <int R, int W, int NC, int D, bool NT, bool EXPERTS>
__global__ __launch_bounds__(64 * W) void gated_dgrad_skinny_kernel(GatedBackward p) {
    typedef SkinnyAcross<R, W, NC, D> S;
    constexpr int kThreads = 64 * W;
    extern __shared__ __attribute__((aligned(2048))) uint8_t smem[];
    const uint32_t lane = lane_id(), w = wave_id(), r = lane & 15, g = lane >> 4;
    int col0 = xcd_chunk_order(blockIdx.x, gridDim.x, kCuPerXcd) * NC;
    if constexpr (EXPERTS) {   // up to 16 R of an expert's rows
        const GroupedTile t = grouped_tile(p.offsets, p.E, p.R, 16 * R, p.tiles_n, p.N, p.I, xcd_chunk_order(blockIdx.x, gridDim.x, kCuPerXcd));
        if (t.expert < 0) return;
        col0 = t.tile_n * NC;
        p.dy += (size_t)t.row0 * p.N;
        p.w2 += (size_t)t.expert * p.N * p.I;
        p.gate_up += (size_t)t.row0 * 2 * p.I;
        p.dgate_up += (size_t)t.row0 * 2 * p.I;
        if (p.h) p.h += (size_t)t.row0 * p.I;
        p.R = t.rows;
    }
    const int nk = (p.N + kLayoutStep - 1) / kLayoutStep;
    const int s0 = nk * (int)w / S::kWaves, n = nk * ((int)w + 1) / S::kWaves - s0;

    // this thread's elements of the result: four columns of a row each, and their kept values
    constexpr int kItems = (R * S::F * 64 + kThreads - 1) / kThreads;
    v2i kept_g[kItems], kept_u[kItems];
    auto place = [&](int i, int& row, int& col) {
        const int t = i * kThreads + threadIdx.x, l = t & 63;
        row = t / (S::F * 64) * 16 + (l & 15);
        col = col0 + (t >> 6) % S::F * 16 + 4 * (l >> 4);
        return t < R * S::F * 64 && row < p.R && col < p.I;
    };
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        int row, col;
        kept_g[i] = kept_u[i] = v2i{0, 0};
        if (!place(i, row, col)) continue;
        const uint16_t* at = p.gate_up + (size_t)row * 2 * p.I;
        if (p.interleaved) {
            const v4i both = *(const v4i*)(at + 2 * col);
            kept_g[i] = v2i{both.x, both.y};
            kept_u[i] = v2i{both.z, both.w};
        } else {
            kept_g[i] = *(const v2i*)(at + col);
            kept_u[i] = *(const v2i*)(at + p.I + col);
        }
    }

    const uint32_t pitch = to_sgpr(2u * (uint32_t)p.I), dy_pitch = to_sgpr(2u * (uint32_t)p.N);
    const uint64_t base = (uint64_t)(p.w2 + col0);
    const int64_t bytes = 2 * ((int64_t)p.N * p.I - col0);
    const v4i srd_dy = make_srd(p.dy, (uint32_t)p.R * dy_pitch);
    uint32_t voff_w[2], voff_dy[2], tail_or[2];   // even / odd loads (the swizzles take the load's parity)
#pragma unroll
    for (int odd = 0; odd < 2; ++odd) {
        const uint32_t k = lane / S::kChunks;
        voff_w[odd] = k * pitch + ((lane % S::kChunks) ^ S::swz(k + S::kLoadRows * odd)) * 16u;
        const uint32_t row = 8u * odd + (lane >> 3), c = swz_chunk(row, lane & 7) * 16u;
        voff_dy[odd] = row * dy_pitch + c;
        tail_or[odd] = (int)c >= 2 * (p.N - (nk - 1) * kLayoutStep) ? kOutside : 0u;
    }
    const uint32_t lds0 = (uint32_t)(uintptr_t)smem, region = to_sgpr(lds0 + w * S::kRegion);
    auto issue = [&](int stage, int at) {
        const int kt = s0 + at;
        const uint32_t dst = region + (uint32_t)stage * S::kStage;
        const int64_t skip = (int64_t)kt * kLayoutStep * pitch, left = bytes - skip;
        const v4i srd = make_srd((const void*)(base + skip), (uint32_t)(left < 0x7fffffff ? (left > 0 ? left : 0) : 0x7fffffff));
#pragma unroll
        for (int i = 0; i < S::kLoads; ++i) {
            const uint32_t so = to_sgpr(i * S::kLoadRows * pitch);
            if constexpr (NT) dma16_nt(srd, to_sgpr(dst + i * 1024), voff_w[i & 1], so);
            else dma16(srd, to_sgpr(dst + i * 1024), voff_w[i & 1], so);
        }
        const bool last = kt == nk - 1;
#pragma unroll
        for (int i = 0; i < 2 * R; ++i)
            dma16(srd_dy, to_sgpr(dst + S::kW + i * 1024), (voff_dy[i & 1] + (uint32_t)(i >> 1) * 16u * dy_pitch) | (last ? tail_or[i & 1] : 0u),
                  to_sgpr((uint32_t)kt * 128u));
    };
    v4f acc[R][S::F];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int f = 0; f < S::F; ++f) acc[i][f] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < D - 1; ++s)
        if (s < n) issue(s, s);
    const uint32_t k0 = 8 * g + (r >> 2);
    const uint32_t rd_w = region + k0 * S::kRow + (((r >> 1) & 1u) ^ S::swz(k0)) * 16u + (r & 1u) * 8u;
    const uint32_t rd_lo = region + S::kW + r * 128u + swz_chunk(r, g) * 16u, rd_hi = region + S::kW + r * 128u + swz_chunk(r, g + 4) * 16u;
    int st = 0;
    for (int kt = 0; kt < n; ++kt) {
        // K-step kt has landed: no more of the K-steps behind it are under way than were issued
        switch (min(n - 1 - kt, D - 2)) {
            case 0: wait_vmcnt<0>(); break;
            case 1: wait_vmcnt<S::kAll>(); break;
            case 2: wait_vmcnt<(D > 3 ? 2 : 1) * S::kAll>(); break;
            case 3: wait_vmcnt<(D > 4 ? 3 : 1) * S::kAll>(); break;
            default: wait_vmcnt<(D > 5 ? 4 : 1) * S::kAll>(); break;
        }
        static_assert(D >= 2 && D <= 6);
        if (kt + D - 1 < n) issue(st == 0 ? D - 1 : st - 1, kt + D - 1);   // (that stage's reads were waited for before its products)
        const uint32_t so = (uint32_t)st * S::kStage;
        v8i wf[S::F];
#pragma unroll
        for (int f = 0; f < S::F; ++f) {
            const uint32_t at = (rd_w ^ (32u * f)) + so;
            const v2i a = lds_read_tr(at), b = lds_read_tr(at + 4 * S::kRow), c = lds_read_tr(at + 32 * S::kRow), d = lds_read_tr(at + 36 * S::kRow);
            wf[f] = v8i{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const v8i af = lds_frag(rd_lo + so, rd_hi + so, i * 2048);
#pragma unroll
            for (int f = 0; f < S::F; ++f) GatedMma::mma(acc[i][f], wf[f], af);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // this stage's reads are done before a later load may overwrite it
        st = st == D - 1 ? 0 : st + 1;
    }
    __syncthreads();   // every wave is done with its stages
    v4f* red = (v4f*)smem;   // [waves][R][F][64]
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int f = 0; f < S::F; ++f) red[((w * R + i) * S::F + f) * 64 + lane] = acc[i][f];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        int row, col;
        if (!place(i, row, col)) continue;
        v4f dh = red[i * kThreads + threadIdx.x];
#pragma unroll
        for (int v = 1; v < S::kWaves; ++v) dh += red[v * R * S::F * 64 + i * kThreads + threadIdx.x];
        float dg[4], du[4], h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // (alternating: words 2 j .. of both halves hold a pair each; stacked: two gate values a word)
            const uint32_t pair = (uint32_t)(j < 2 ? kept_g[i][j] : kept_u[i][j - 2]);
            const uint32_t two_g = (uint32_t)kept_g[i][j / 2], two_u = (uint32_t)kept_u[i][j / 2];
            const float gv = __uint_as_float(p.interleaved ? pair << 16 : j & 1 ? two_g & 0xffff0000u : two_g << 16);
            const float uv = __uint_as_float(p.interleaved ? pair & 0xffff0000u : j & 1 ? two_u & 0xffff0000u : two_u << 16);
            h[j] = p.clamped ? Gate<true>{p.gate}.gradients(gv, uv, dh[j], dg[j], du[j]) : Gate<false>{p.gate}.gradients(gv, uv, dh[j], dg[j], du[j]);
        }
        uint16_t* at = p.dgate_up + (size_t)row * 2 * p.I;
        if (p.interleaved) {
            *(v4i*)(at + 2 * col) = v4i{(int)pack_bf16(dg[0], du[0]), (int)pack_bf16(dg[1], du[1]), (int)pack_bf16(dg[2], du[2]), (int)pack_bf16(dg[3], du[3])};
        } else {
            *(v2i*)(at + col) = v2i{(int)pack_bf16(dg[0], dg[1]), (int)pack_bf16(dg[2], dg[3])};
            *(v2i*)(at + p.I + col) = v2i{(int)pack_bf16(du[0], du[1]), (int)pack_bf16(du[2], du[3])};
        }
        if (p.h) *(v2i*)(p.h + (size_t)row * p.I + col) = v2i{(int)pack_bf16(h[0], h[1]), (int)pack_bf16(h[2], h[3])};
    }
}

// alpha and limit of the clamped form (1); SiLU (0) has none
static int check_gate(int activation, const GateArgs& g) {
    if (activation == 0) return HK_OK;
    return activation == 1 && g.limit > 0.f && __builtin_fabsf(g.alpha) < __builtin_inff() ? HK_OK : HK_ERR_UNSUPPORTED;
}

// wide: the length of the rows that are not I or 2 I
static int gated_check(int R, int E, int I, int wide, const int32_t* offsets) {
    if (R <= 0 || R >= (1 << 30) || E <= 0 || E > kGroupedMaxE || I <= 0 || wide <= 0 || (I % 8) != 0 || (wide % 8) != 0 || I > (1 << 20) ||
        wide > (1 << 21) || (!offsets && E != 1))
        return HK_ERR_BAD_SHAPE;
    return HK_OK;
}

template <typename Tile, typename P>
static int launch_gated_tile(void (*kern)(P), DeviceOnce& once, P p, int out, int lds_bytes, hipStream_t s) {
    p.tiles_n = (out + Tile::kTileCols - 1) / Tile::kTileCols;
    const long long grid = grouped_tiles_m(p.R, p.E, Tile::kTile) * p.tiles_n;
    if (grid >= kMaxWorkgroups) return HK_ERR_BAD_SHAPE;
    if (!set_lds_limit_once((const void*)kern, lds_bytes, once)) return HK_ERR_LAUNCH;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(256), lds_bytes, s, p);
    return hipGetLastError() == hipSuccess ? HK_OK : HK_ERR_LAUNCH;
}
template <typename Tile, bool CLAMPED, bool INTERLEAVED>
static int launch_gated(const GatedForward& p, hipStream_t s) {
    static DeviceOnce once;
    return launch_gated_tile<Tile>(gated_gemm_kernel<Tile, CLAMPED, INTERLEAVED>, once, p, 2 * p.I, Tile::kLds, s);
}
template <typename Tile, bool CLAMPED, bool INTERLEAVED>
static int launch_gated(const GatedBackward& p, hipStream_t s) {
    static DeviceOnce once;
    return launch_gated_tile<Tile>(gated_dgrad_kernel<Tile, CLAMPED, INTERLEAVED>, once, p, p.I, GateUpLoads<Tile, INTERLEAVED>::kLds, s);
}
template <typename Tile, typename P>
static int launch_gated_form(const P& p, hipStream_t s) {
    if (p.clamped) return p.interleaved ? launch_gated<Tile, true, true>(p, s) : launch_gated<Tile, true, false>(p, s);
    return p.interleaved ? launch_gated<Tile, false, true>(p, s) : launch_gated<Tile, false, false>(p, s);
}
// Workgroups of the kernels for few rows: the column blocks, of every 16 R rows of an expert where there are experts.
template <int R, typename P>
static long long skinny_grid(P& p, int cols) {
    p.tiles_n = (p.I + cols - 1) / cols;
    return p.offsets ? grouped_tiles_m(p.R, p.E, 16 * R) * p.tiles_n : p.tiles_n;
}
// Weights past the caches: where they are too large to stay (a dense block's; experts' of any size, whose workgroups read them once), and where the rows
// of memory that the kernels load are whole cache lines; a line that two loads share would come from HBM twice (one row, I = 9408, K = 2360
// 25.4 us with the hint, 23.4 without; 40 experts of 1432 x 3000, 64 rows 159 / 124; but one row, I = 11008, K = 4096 29.6 / 31.9).
static bool skinny_nt(const void* w, long long bytes, long long row_bytes) { return bytes >= kSkinnyNtBytes && (((uintptr_t)w | row_bytes) % 128) == 0; }
template <int R, int NW, int D, int NF, bool EXPERTS = false>
static int launch_gated_skinny_kernel(GatedForward p, hipStream_t s) {
    const bool nt = skinny_nt(p.w13, EXPERTS ? kSkinnyNtBytes : 4ll * p.I * p.K, 2ll * p.K);
    auto kern = nt ? gated_skinny_kernel<R, NW, D, NF, true, EXPERTS> : gated_skinny_kernel<R, NW, D, NF, false, EXPERTS>;
    constexpr int lds_bytes = skinny_lds_bytes(R, NW, D, false, NF);
    static_assert(lds_bytes <= 160 * 1024, "LDS of one CU");
    static DeviceOnce configured[2];
    const long long grid = skinny_grid<R>(p, 8 * NF);
    if (grid >= kMaxWorkgroups) return HK_ERR_BAD_SHAPE;
    if (!set_lds_limit_once((const void*)kern, lds_bytes, configured[nt])) return HK_ERR_LAUNCH;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(64 * NW), lds_bytes, s, p);
    return hipGetLastError() == hipSuccess ? HK_OK : HK_ERR_LAUNCH;
}
// R: 16 rows of x each. Rows of the weights a workgroup: 16 (NF = 1) while 32 would leave half of the CUs without one; 64 (NF = 4) where their rounds
// over the CUs, one workgroup each, take in fewer bytes than those of 32 (NF = 2): x is loaded once a workgroup, and a CU's loads into LDS, not
// HBM, bound more than 16 rows. (us from HBM, 32 / 64 rows of weights a workgroup / 64-tile kernel: 48 rows, I = 14336, K = 4096 55.7 / 42.2 /
// 55.0; 32 rows 47.5 / 39.0 / 55.2; 32 rows, I = 9216, K = 8192 63.7 / 68.2 / 74.1; with 16 rows and 32 a workgroup 37.6 / - / 55.1, one row
// 36.1. 1 row, I = 2048, K = 7168: 11.2 / - / 30.2.) Rows of weights that are not whole cache lines take two accesses a piece, which bounds a CU, so that one
// with a workgroup more than the others is waited for: 16 again while x is a few rows (16 / 32: one row, I = 9408, K = 2360 18.4 / 23.4; 8 rows, I =
// 4176, K = 6512 31.7 / 37.2; 12 rows, I = 13000, K = 4072 55.6 / 53.2).
// Waves and stages of a workgroup for 16, 32 and 64 rows of weights. Where there are more workgroups than CUs, two of them fit a CU (one row of 14336 x
// 4096 with one a CU 38.5 us, so 35.9; 32 rows, with more stages: 9216 x 8192 65.1, so 63.0, 14336 x 4096 40.7, so 38.8). In one round 12 to 30 KB under
// way a wave are enough, and more stages, as many as the LDS holds, only start later (one row of 912 x 3728 6.4, so 5.5; of 2048 x 7168 11.3 / 11.1; 32
// rows of it 16.1 / 16.1). Of 48 and 64 rows, more than one round is always one of 64 rows of weights.
struct SkinnyForm { int waves, stages; };
template <int R> constexpr SkinnyForm kSkinnyForms[2][3] = {};   // [one round, more]
template <> constexpr SkinnyForm kSkinnyForms<1>[2][3] = {{{4, 4}, {4, 4}, {}}, {{4, 4}, {4, 3}, {}}};
template <> constexpr SkinnyForm kSkinnyForms<2>[2][3] = {{{4, 3}, {4, 3}, {3, 3}}, {{}, {3, 3}, {3, 2}}};
template <> constexpr SkinnyForm kSkinnyForms<3>[2][3] = {{{4, 4}, {4, 4}, {3, 3}}, {{}, {}, {2, 2}}};
template <> constexpr SkinnyForm kSkinnyForms<4>[2][3] = {{{4, 3}, {4, 3}, {3, 3}}, {{}, {}, {2, 2}}};
template <int R>
static int launch_gated_skinny_rows(const GatedForward& p, hipStream_t s) {
    const int cus = moe_num_compute_units();
    auto rounds = [&](int cols) { return ((p.I + cols - 1) / cols + cus - 1) / cus; };
    auto launch = [&]<int I>() {
        constexpr SkinnyForm one = kSkinnyForms<R>[0][I], more = kSkinnyForms<R>[1][I];
        if constexpr (more.waves > 0)
            if (rounds(8 << I) > 1) return launch_gated_skinny_kernel<R, more.waves, more.stages, 1 << I>(p, s);
        return launch_gated_skinny_kernel<R, one.waves, one.stages, 1 << I>(p, s);
    };
    if (2ll * ((p.I + 15) / 16) <= cus || (R == 1 && p.R <= 8 && p.K % 64 != 0 && rounds(16) > 1)) return launch.template operator()<0>();
    if constexpr (R > 1)
        if (rounds(32) * (64 + 16 * R) < rounds(16) * (32 + 16 * R)) return launch.template operator()<2>();
    return launch.template operator()<1>();
}
// Not for short rows of many columns, where a wave has few K-steps of its own (16 rows, skinny / 64-tile kernel, us: I = 57344, K = 512 35.4 / 27.9;
// I = 100000, K = 1024 89.4 / 88.9, 64 rows 105 / 95; I = 28672, K = 2048, 64 rows 52.9 / 59.9).
static bool use_gated_skinny(int R, int I, int K) {
    if (R > kSkinnyMaxM) return false;
    return (I + 15) / 16 <= moe_num_compute_units() || K >= (R <= 32 ? 1024 : 2048);
}
static int launch_gated_skinny(const GatedForward& p, hipStream_t s) {
    if (p.R <= 16) return launch_gated_skinny_rows<1>(p, s);
    if (p.R <= 32) return launch_gated_skinny_rows<2>(p, s);
    if (p.R <= 48) return launch_gated_skinny_rows<3>(p, s);
    return launch_gated_skinny_rows<4>(p, s);
}
template <int R, int W, int NC, int D, bool EXPERTS = false>
static int launch_gated_dgrad_skinny_kernel(GatedBackward p, hipStream_t s) {
    const bool nt = skinny_nt(p.w2, EXPERTS ? kSkinnyNtBytes : 2ll * p.I * p.N, 2ll * p.I);
    auto kern = nt ? gated_dgrad_skinny_kernel<R, W, NC, D, true, EXPERTS> : gated_dgrad_skinny_kernel<R, W, NC, D, false, EXPERTS>;
    constexpr int lds_bytes = SkinnyAcross<R, W, NC, D>::kLds;
    static DeviceOnce configured[2];
    const long long grid = skinny_grid<R>(p, NC);
    if (grid >= kMaxWorkgroups) return HK_ERR_BAD_SHAPE;
    if (!set_lds_limit_once((const void*)kern, lds_bytes, configured[nt])) return HK_ERR_LAUNCH;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(64 * W), lds_bytes, s, p);
    return hipGetLastError() == hipSuccess ? HK_OK : HK_ERR_LAUNCH;
}
// 32 columns a workgroup while that gives no CU a second one (rows of W2 in pieces of 64 bytes: what a CU has under way is counted in
// pieces, so that half as many workgroups of 64 columns are no faster); more columns in pieces of 64 up to 32 rows, and the 64-tile kernel beyond.
// (us from HBM, 64-tile kernel / 32 columns / 64: one row, I = 2048, N = 7168 32.5 / 24.8 / 29.4; I = 912, N = 3728 19.6 / 12.7 / 17.0;
// I = 14336, N = 4096 25.9 / 35.4 / 24.4; 64 rows of it 32.6 / 51.5 / 33.4, of I = 8192, N = 2048 17.1 / 15.8 / 17.8.)
static bool use_gated_dgrad_skinny(int R, int I) {
    return R <= 32 || (R <= kSkinnyMaxM && (I + 31) / 32 <= moe_num_compute_units());
}
static int launch_gated_dgrad_skinny(const GatedBackward& p, hipStream_t s) {
    const bool narrow = (p.I + 31) / 32 <= moe_num_compute_units();
    if (p.R <= 16) return narrow ? launch_gated_dgrad_skinny_kernel<1, 4, 32, 6>(p, s) : launch_gated_dgrad_skinny_kernel<1, 4, 64, 4>(p, s);
    if (p.R <= 32) return narrow ? launch_gated_dgrad_skinny_kernel<2, 4, 32, 5>(p, s) : launch_gated_dgrad_skinny_kernel<2, 4, 64, 3>(p, s);
    return launch_gated_dgrad_skinny_kernel<4, 4, 32, 3>(p, s);
}

// Experts with few rows, of which the host knows only how many there are on average where they spread evenly. Two workgroups a CU and more, by their LDS: a
// launch has many rounds of them, and one's start and end are the others' time. Forward: 16 rows of the weights a workgroup while the CUs hold them
// in one round, 32 for few rounds, else 64 of up to 32 rows of x (16 rows of x take 0 to 8 % less where the experts' rows are even, up to 10 % more where
// they are not); more than 8 rows an expert only where the 128-tile kernel has more than one round of its two workgroups a CU. Backward: 32
// columns a workgroup while they are one round, else 64, but for the 128-tile kernel's one round. Beyond one round not for short rows, where a wave has few
// K-steps. (us, tile kernels / these: forward, 128 experts of 2880 x 2880, 300 rows 662 / 578, 1000 732 / 650, 2000 742 / 675, 3200 756 / 764; 200 of
// 1024 x 4096, 500 rows 549 / 451; 40 of 2048 x 7168, 300 rows 425 / 348; 9 of 576 x 2672, one row 16.1 / 7.4, but 40 rows 17.3 / 18.9. Shares of the
// experts as 1 / rank: 128 of 2880 x 2880, 1000 rows 669 / 646, 200 of 1024 x 4096, 1500 rows 561 / 477, but 32 of 2880 x 2880, 600 rows, 141 of
// them one expert's, 190 / 212. Backward, the first four 372 / 299, 394 / 347, 402 / 383, 410 / 442; 275 / 246; 265 / 207; 16.6 / 8.9, 17.0 / 12.8; uneven
// 377 / 341, 272 / 268, 121 / 117; 40 experts of 1432 x 1024, 40 rows, one round of tiles, 22.3 / 29.1. Short rows: 30 of 3000 x 264, 64 rows
// forward 33.5 / 37.5; 60 of 2048 x 768, 200 rows backward 41.5 / 44.9.)
struct ExpertRows {
    double used, mean;
    ExpertRows(int R, int E) : used(-E * std::expm1(R * std::log1p(-1.0 / E))), mean(R / used) {}
    double blocks(int I, int cols) const { return used * ((I + cols - 1) / cols); }
};
constexpr int kExpertRows16 = 8, kExpertRows32 = 20;   // most on average for 16 and for 32 rows a workgroup
constexpr int kExpertMinWide = 1024;
constexpr int kExpertMaxI = 1 << 16;   // (their grids grow with I faster than the tiles')
static bool launch_gated_experts_skinny(const GatedForward& p, hipStream_t s, int& st) {
    const ExpertRows rows(p.R, p.E);
    const int cus = moe_num_compute_units();
    if (rows.mean > kExpertRows32 || p.I > kExpertMaxI || (p.K < kExpertMinWide && rows.blocks(p.I, 16) > cus)) return false;
    if (rows.blocks(p.I, 8) <= cus && rows.mean <= kExpertRows16) {
        st = launch_gated_skinny_kernel<1, 4, 4, 1, true>(p, s);
    } else if (rows.blocks(p.I, 16) <= cus || (rows.mean <= kExpertRows16 && rows.blocks(p.I, 16) < (p.K < 2048 ? 2 : 6) * cus)) {
        st = rows.mean <= kExpertRows16 ? launch_gated_skinny_kernel<1, 4, 3, 2, true>(p, s) : launch_gated_skinny_kernel<2, 4, 3, 2, true>(p, s);
    } else {
        if (rows.mean > kExpertRows16 && rows.blocks(p.I, 64) <= 2 * cus) return false;
        st = launch_gated_skinny_kernel<2, 2, 3, 4, true>(p, s);
    }
    return true;
}
static bool launch_gated_experts_skinny(const GatedBackward& p, hipStream_t s, int& st) {
    const ExpertRows rows(p.R, p.E);
    const int cus = moe_num_compute_units();
    if (rows.mean > kExpertRows32 || p.I > kExpertMaxI) return false;
    if (rows.blocks(p.I, 32) <= cus) {
        st = rows.mean <= kExpertRows16 ? launch_gated_dgrad_skinny_kernel<1, 4, 32, 3, true>(p, s) : launch_gated_dgrad_skinny_kernel<2, 4, 32, 5, true>(p, s);
    } else {
        const double tiles = rows.blocks(p.I, 128);
        if (p.N < kExpertMinWide || (tiles > cus && tiles <= 2 * cus)) return false;
        st = launch_gated_dgrad_skinny_kernel<2, 2, 64, 3, true>(p, s);
    }
    return true;
}

// The tile: 64x64 with many LDS stages where there are no more of them than CUs, else the least of rounds over the CUs times a fixed part and a part per
// K-step, us. A round begun counts whole between one and two, where the last tiles are most of a round by themselves, and less behind that. (us, with
// choose_layout's rounds / these: forward, 1831 rows, I = 2280, K = 3784 126.5 / 81.5; 11 experts of 1776 x 2688, 1567 rows 90.9 / 66.0; backward,
// 1636 rows, I = 9472, N = 840 72.0 / 50.1, but 1547 rows, I = 12376, N = 2600 150.3 / 172.4; on 230 drawn shapes of more than 64 rows 1.3 %
// less on average.) Tiles of 128 rows and 256 columns, 128x128 or 256x256 otherwise / these: 32 experts of 2048 x 7168, 128 rows each 492 / 425; 128 of
// 2880 x 2880, 64 rows 870 / 841; 64 of 1536 x 4096, 150 rows 435 / 386; 8 of 4096 x 4096, 128 rows 203 / 158, but 64 of 768 x 2048, 128 rows
// 131 / 141; and 128 of 2880 x 2880 with 128 rows, where the rule stays with 256x256, 1008 / 990. Not in the backward pass, where the same rule
// would gain at 128 rows an expert (32 of 2048 x 7168 280 / 270, 8 of 4096 x 4096 92 / 82) and lose beyond and beside it (256 rows 355 / 389; 64 of
// 1536 x 4096, 150 rows 240 / 267; 128 of 2880 x 2880, 64 rows 472 / 490).
constexpr double kWideFixed = 6.0, kWideStep = 0.97, kDeepFixed = 4.0, kDeepStepBusy = 0.5;
enum GatedTile { kGatedWide, kGated256, kGated128, kGated128Deep, kGated64Deep };
static GatedTile gated_tile(int R, int E, int in, int out, bool dense, bool forward) {
    const int cus = moe_num_compute_units();
    auto tiles = [&](int rows, int cols) { return grouped_row_tiles(R, E, rows, dense) * ((out + cols - 1) / cols); };
    if (tiles(64, 64) <= cus) return kGated64Deep;
    const double steps = (in + kLayoutStep - 1) / kLayoutStep, small = tiles(128, 128);
    auto rounds = [](double t) { return t <= 1 ? 1.0 : std::max(t + 0.2, std::min(2.0, t + 0.65)); };
    const bool deep = small <= cus;
    GatedTile t = deep ? kGated128Deep : kGated128;
    double best = deep ? kDeepFixed + kDeepStepBusy * steps : rounds(small / (2.0 * cus)) * (kSmallFixed + kSmallStepAlong * steps);
    auto consider = [&](GatedTile other, double us) {
        if (us < best) {
            best = us;
            t = other;
        }
    };
    consider(kGated256, rounds(tiles(256, 256) / cus) * (kLargeFixed + kLargeStep * steps));
    if (forward && !deep) consider(kGatedWide, rounds(tiles(128, 256) / cus) * (kWideFixed + kWideStep * steps));
    return t;
}

// 64x64 tiles, two workgroups a CU, where the CUs hold them so in one round and one a CU would not; rows of whole cache lines (others take two accesses
// a piece, which bounds a CU here). (us, the kernel otherwise chosen / this: 128 rows forward, I = 4104, K = 4096, 258 tiles, 39.9 / 29.1; I = 8192,
// K = 2048, 512 tiles 25.2 / 23.4; I = 14336, K = 4096, 896 tiles 55.7 / 76.3; 190 rows of 2880 x 2880, 270 tiles 25.5 / 26.7; backward, 520 rows of
// 2880 x 2880, 405 tiles 29.4 / 24.3, of 2440 x 6376, 351 tiles, 56.8 / 72.3. 2 experts of 2048 x 7168, 200 rows forward 69.8 / 39.8; 4 of
// 2880 x 2880 31.4 / 34.5.)
static bool use_pair_tile(int R, int E, int in, int out, bool dense) {
    const int cus = moe_num_compute_units();
    const double tiles = grouped_row_tiles(R, E, 64, dense) * ((out + 63) / 64);
    return tiles > cus && tiles <= 2 * cus && in % 64 == 0;
}
template <typename P>
static int launch_gated_choice(const P& p, int in, int out, hipStream_t s) {
    if (use_pair_tile(p.R, p.E, in, out, !p.offsets)) return launch_gated_form<LayoutTile64Pair>(p, s);
    constexpr bool forward = std::is_same_v<P, GatedForward>;
    const GatedTile t = gated_tile(p.R, p.E, in, out, !p.offsets, forward);
    if constexpr (forward)
        if (t == kGatedWide) return launch_gated_form<LayoutTileWide>(p, s);
    switch (t) {
        case kGated256: return launch_gated_form<LayoutTile256>(p, s);
        case kGated128: return launch_gated_form<LayoutTile128>(p, s);
        case kGated128Deep: return launch_gated_form<LayoutTile128Deep>(p, s);
        default: return launch_gated_form<LayoutTile64Deep>(p, s);
    }
}

}  // namespace hk

extern "C" int hk_gated_gemm(const void* x_bf16, const void* w13_bf16, const int32_t* expert_offsets_or_null, void* h_bf16,
                             void* gate_up_bf16_or_null, int R, int E, int I, int K, int interleaved, int activation, float alpha,
                             float limit, void* stream) {
    using namespace hk;
    if (!x_bf16 || !w13_bf16 || !h_bf16) return HK_ERR_NULL_POINTER;
    if (const int st = gated_check(R, E, I, K, expert_offsets_or_null)) return st;
    if (((uintptr_t)x_bf16 | (uintptr_t)w13_bf16 | (uintptr_t)h_bf16 | (uintptr_t)gate_up_bf16_or_null) & 15u) return HK_ERR_BAD_ALIGNMENT;
    GatedForward p{(const uint16_t*)x_bf16, (const uint16_t*)w13_bf16, expert_offsets_or_null, (uint16_t*)h_bf16, (uint16_t*)gate_up_bf16_or_null,
                   R, E, I, K, 0, interleaved != 0, activation == 1, {alpha, limit}};
    if (const int st = check_gate(activation, p.gate)) return st;
    if (!p.offsets && use_gated_skinny(R, I, K)) return launch_gated_skinny(p, (hipStream_t)stream);
    if (int st; p.offsets && launch_gated_experts_skinny(p, (hipStream_t)stream, st)) return st;
    return launch_gated_choice(p, K, 2 * I, (hipStream_t)stream);
}

extern "C" int hk_gated_gemm_dgrad(const void* dy_bf16, const void* w2_bf16, const int32_t* expert_offsets_or_null, const void* gate_up_bf16,
                                   void* dgate_up_bf16, void* h_bf16_or_null, int R, int E, int N, int I, int interleaved, int activation,
                                   float alpha, float limit, void* stream) {
    using namespace hk;
    if (!dy_bf16 || !w2_bf16 || !gate_up_bf16 || !dgate_up_bf16) return HK_ERR_NULL_POINTER;
    if (const int st = gated_check(R, E, I, N, expert_offsets_or_null)) return st;
    if (((uintptr_t)dy_bf16 | (uintptr_t)w2_bf16 | (uintptr_t)gate_up_bf16 | (uintptr_t)dgate_up_bf16 | (uintptr_t)h_bf16_or_null) & 15u)
        return HK_ERR_BAD_ALIGNMENT;
    GatedBackward p{(const uint16_t*)dy_bf16, (const uint16_t*)w2_bf16, expert_offsets_or_null, (const uint16_t*)gate_up_bf16,
                    (uint16_t*)dgate_up_bf16, (uint16_t*)h_bf16_or_null, R, E, N, I, 0, interleaved != 0, activation == 1, {alpha, limit}};
    if (const int st = check_gate(activation, p.gate)) return st;
    if (!p.offsets && use_gated_dgrad_skinny(R, I)) return launch_gated_dgrad_skinny(p, (hipStream_t)stream);
    if (int st; p.offsets && launch_gated_experts_skinny(p, (hipStream_t)stream, st)) return st;
    return launch_gated_choice(p, N, I, (hipStream_t)stream);
}
