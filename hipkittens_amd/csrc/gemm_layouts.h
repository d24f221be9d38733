// bf16 tile products for operands in either memory order, for the products of a training step: C = A B^T with the
// contraction running along an operand's rows in memory (a row of x or of W, as in the GEMMs) or across them (the
// gradients: dx = dy W contracts over W's rows, dW = dy^T x over the rows of both).
//
// LDS holds a K-step of 64 elements of an operand's TILE rows or columns. Contracted along the rows it is the GEMMs'
// tile: TILE rows of 128 bytes, read with ds_read_b128. Contracted across them it is 64 rows of 2 TILE bytes as they
// lie in memory, read with ds_read_b64_tr_b16: in a group of 16 lanes lane i names four columns (4 (i % 4) .. +4) of row
// i / 4 and receives column i of the four rows. Both give lane l of a fragment row (column) l % 16, elements
// 8 (l / 16) .. +8 of each half of the K-step: no operand is transposed in memory.
#pragma once
#include "gemm_tile.h"
#include "hk_host.h"

namespace hk {

typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s_t;
typedef __bf16 v8bf_t __attribute__((ext_vector_type(8)));

constexpr int kLayoutStep = 64;   // elements of the contraction per K-step

// One operand of a tile product. across = false: `rows` rows of `pitch` bytes, contraction along them. across = true: the
// rows run along the contraction and the tile takes the columns from `base` on.
// bytes: from `base` to the end of what may be read (the last row's last element): loads beyond it give zeros.
struct TileOperand {
    const uint8_t* base;
    uint64_t bytes;
    uint32_t pitch;
};

// Swizzle of an across tile: 16-byte chunk c of LDS row k lies at chunk c ^ across_swz(k). A half wave of the transposing
// read touches two neighbouring chunks of the eight rows k0 + {0..3, 8..11}: they fall on sixteen different chunks of a
// 256-byte line, i.e. on every bank once.
__device__ __forceinline__ uint32_t across_swz(uint32_t k) { return 2u * ((k & 3u) | ((k >> 1) & 4u)); }
// The same for rows of 128 bytes, two of which share a line: row bit 0 is the half of it.
__device__ __forceinline__ uint32_t across_swz128(uint32_t k) { return 2u * (((k >> 1) & 1u) | ((k >> 2) & 2u)); }

__device__ __forceinline__ v2i lds_read_tr(uint32_t addr) {
    return __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t*)(uintptr_t)addr));
}

// Tile product of four waves, each a quarter (TILE / 2 square) of TILE x TILE. Two LDS stages: the next K-step is loaded while this
// one is multiplied, two workgroups on a CU. One: each K-step in turn, four workgroups on a CU, for contractions of a few K-steps.
// acc[m][n] holds, for tile row 16 m + lane % 16 of the wave's quarter, its columns 16 n + 4 (lane / 16) .. +4.
constexpr int kLayoutTile = 128;
constexpr int kLayoutStageBytes = 2 * kLayoutTile * 128;

template <bool ACROSS>
struct TileLoader {
    static constexpr int TILE = kLayoutTile;
    v4i srd;
    uint64_t base, left;
    uint32_t voff, pitch, k_bytes, round;
    __device__ __forceinline__ TileLoader(const TileOperand& op, int K) {
        const int lane = lane_id(), w = wave_id();
        base = (uint64_t)op.base;
        left = op.bytes;
        pitch = op.pitch;
        k_bytes = 2u * (uint32_t)K;
        if constexpr (ACROSS) {
            const uint32_t k = 4 * w + (lane >> 4);                   // + 16 per load
            voff = k * pitch + (((lane & 15u) ^ across_swz(k)) * 16u);
            round = 16u * pitch;
        } else {
            const uint32_t R = 8 * w + (lane >> 3);                   // + 32 per load
            voff = R * pitch + swz_chunk(R, lane & 7) * 16u;
            round = 32u * pitch;
        }
    }
    // K-step kt into the LDS tile at dst (this wave's first KiB of it). The descriptor starts at the K-step (64-bit base),
    // so offsets stay below 64 rows (across) or TILE rows (along).
    __device__ __forceinline__ void load(int kt, uint32_t dst) const {
        const uint64_t skip = ACROSS ? (uint64_t)kt * kLayoutStep * pitch : (uint64_t)kt * 128u;
        const uint64_t rest = left > skip ? left - skip : 0;
        const v4i d = make_srd((const void*)(base + skip), (uint32_t)(rest < 0x7fffffffull ? rest : 0x7fffffffull));
        uint32_t vo = voff;
        if constexpr (!ACROSS) {   // chunks behind the end of a row: out of the descriptor's range, zeros
            const int lane = lane_id(), w = wave_id();
            if (swz_chunk(8 * w + (lane >> 3), lane & 7) * 16u + (uint32_t)kt * 128u >= k_bytes) vo |= 0x80000000u;
        }
#pragma unroll
        for (int i = 0; i < TILE * 128 / 4096; ++i) dma16(d, to_sgpr(dst + i * 4096), vo, to_sgpr(i * round));
    }
};

// Fragment `f` (16 rows or columns) of the quarter that starts at row or column `first` of the tile at `tile`.
template <bool ACROSS>
__device__ __forceinline__ Frag4 tile_fragment(uint32_t tile, int first, int f) {
    const uint32_t lane = lane_id(), i = lane & 15, g = lane >> 4;
    Frag4 out;
    if constexpr (ACROSS) {
        const uint32_t k = 8 * g + (i >> 2), row_bytes = 2 * kLayoutTile;
        const uint32_t chunk = (uint32_t)(first / 8 + 2 * f) + ((i >> 1) & 1u);
        const uint32_t at = tile + k * row_bytes + (chunk ^ across_swz(k)) * 16u + (i & 1u) * 8u;
        const v2i a = lds_read_tr(at), b = lds_read_tr(at + 4 * row_bytes);
        const v2i c = lds_read_tr(at + 32 * row_bytes), d = lds_read_tr(at + 36 * row_bytes);
        out.lo = v4i{a.x, a.y, b.x, b.y};
        out.hi = v4i{c.x, c.y, d.x, d.y};
    } else {
        const uint32_t R = first + 16 * f + i;
        out = lds_frag4(tile + R * 128u + swz_chunk(R, g) * 16u, tile + R * 128u + swz_chunk(R, g + 4) * 16u, 0);
    }
    return out;
}

template <bool A_ACROSS, bool B_ACROSS, int STAGES>
__device__ __forceinline__ void tile_product(uint8_t* smem, const TileOperand& A, const TileOperand& B, int K,
                                             v4f (&acc)[4][4]) {
    constexpr uint32_t kOperand = kLayoutTile * 128, kStage = 2 * kOperand;
    const int w = wave_id(), wm = w >> 1, wn = w & 1;
    const TileLoader<A_ACROSS> la(A, K);
    const TileLoader<B_ACROSS> lb(B, K);
    const uint32_t lds0 = (uint32_t)(uintptr_t)smem, mine = to_sgpr(lds0 + (uint32_t)w * 1024u);
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[m][n] = v4f{0.f, 0.f, 0.f, 0.f};
    const int nk = (K + kLayoutStep - 1) / kLayoutStep;
    if (nk > 0) {
        la.load(0, mine);
        lb.load(0, mine + kOperand);
    }
    for (int kt = 0; kt < nk; ++kt) {
        if (STAGES == 1 && kt > 0) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            block_barrier();   // everyone has read the one stage
            la.load(kt, mine);
            lb.load(kt, mine + kOperand);
        }
        wait_vmcnt<0>();   // this wave's part of K-step kt has landed ...
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        block_barrier();   // ... everyone's, and everyone has read the other stage
        if (STAGES == 2 && kt + 1 < nk) {
            const uint32_t next = mine + (uint32_t)((kt + 1) & 1) * kStage;
            la.load(kt + 1, next);
            lb.load(kt + 1, next + kOperand);
        }
        const uint32_t at = lds0 + (STAGES == 2 ? (uint32_t)(kt & 1) * kStage : 0u);
        Frag4 b[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) b[n] = tile_fragment<B_ACROSS>(at + kOperand, wn * 64, n);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const Frag4 a = tile_fragment<A_ACROSS>(at, wm * 64, m);
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf_t, b[n].lo),
                                                                    __builtin_bit_cast(v8bf_t, a.lo), acc[m][n], 0, 0, 0);
                acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf_t, b[n].hi),
                                                                    __builtin_bit_cast(v8bf_t, a.hi), acc[m][n], 0, 0, 0);
            }
        }
    }
}

// Operand of a tile: rows [row0, rows) of a matrix with K columns in rows of `pitch` bytes (contraction along the rows) ...
__device__ __forceinline__ TileOperand operand_along(const void* p, uint64_t pitch, int64_t row0, int64_t rows, int K) {
    TileOperand o;
    o.base = (const uint8_t*)p + (uint64_t)row0 * pitch;
    o.bytes = (uint64_t)(rows - row0 - 1) * pitch + 2ull * K;
    o.pitch = (uint32_t)pitch;
    return o;
}
// ... or columns from col0 on of a matrix of K rows (contraction across the rows). Columns behind the end of a row read the
// next row's: they reach only rows or columns of C that are not stored.
__device__ __forceinline__ TileOperand operand_across(const void* p, uint64_t pitch, int64_t col0, int K) {
    TileOperand o;
    o.base = (const uint8_t*)p + 2ull * (uint64_t)col0;
    const uint64_t all = (uint64_t)K * pitch;
    o.bytes = all > 2ull * (uint64_t)col0 ? all - 2ull * (uint64_t)col0 : 0;
    o.pitch = (uint32_t)pitch;
    return o;
}

}  // namespace hk
