// The 4-wave ring schedule (gemm_ring.h) for bf16 operands in either memory order: 256x256 tiles, one wave per SIMD with a
// 128x128 patch, two LDS slots for A's K-steps and three for B's, every LDS read, global->LDS load and MFMA at a fixed place.
//
// What differs from gemm_ring_body:
//  * an operand that is contracted across its rows lies in LDS as 64 rows of 512 bytes and is read with the transposing
//    loads (gemm_layouts.h): four of 8 bytes a lane for a fragment of 16 columns x 64 instead of two of 16, which is why the
//    two halves of a fragment (K elements 0..31 and 32..63) are units of their own in the slot plan;
//  * its descriptor moves with the K-step (64-bit base, bytes left), so that neither its length nor its end inside a
//    K-step needs anything else: rows behind the end are out of range and arrive as zeros;
//  * B's rows are not permuted: acc[m][n] holds, for row 16 m + lane % 16 of the wave's patch, its columns
//    16 n + 4 (lane / 16) .. +4 (the epilogues need that order; store_patch swaps between lanes for whole 16-byte stores).
#pragma once
#include "gemm_layouts.h"

namespace hk {

constexpr int kRingTile = 256;
constexpr int kRingSlot = kRingTile * 128;             // one K-step of one operand
constexpr int kRingLdsBytes = 5 * kRingSlot;

__device__ __forceinline__ void mfma_bf16_acc(v4f& acc, const v4i& x, const v4i& y) {
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(x), "v"(y));
}

// Loads and reads of one operand of a tile of TILE rows (columns): TILE / 32 loads a wave. Load i: along, rows 32 i + 8 w .. +8; across,
// TILE 256, K rows 8 i + 2 w and the next, TILE 128, 16 i + 4 w .. +4, TILE 64, 32 i + 8 w .. +8.
template <bool ACROSS, int TILE = kRingTile>
struct RingOperand {
    static constexpr uint32_t kRow = 2 * TILE;   // across: bytes of a K row in LDS
    uint64_t base;        // descriptor of the K-step that is loaded next
    int64_t left;
    uint32_t voff[2];     // even / odd loads (across: the swizzle takes bit 3 of the K row)
    uint32_t round, tail_or;
    uint32_t rd[2];       // along: the lane's two chunks of its row; across: rd[0] = the lane's address in fragment 0
    static __device__ __forceinline__ uint32_t swz(uint32_t k) { return TILE == 64 ? across_swz128(k) : across_swz(k); }

    // `patch`: which half of the tile's rows (columns) this wave reads
    __device__ __forceinline__ void init(const TileOperand& op, int K, int patch, uint32_t lds0) {
        const uint32_t lane = lane_id(), w = wave_id(), r = lane & 15, g = lane >> 4;
        base = ((uint64_t)to_sgpr((uint32_t)((uint64_t)op.base >> 32)) << 32) | to_sgpr((uint32_t)(uint64_t)op.base);
        left = (int64_t)(((uint64_t)to_sgpr((uint32_t)(op.bytes >> 32)) << 32) | to_sgpr((uint32_t)op.bytes));
        const uint32_t pitch = to_sgpr(op.pitch);
        tail_or = 0;
        if constexpr (ACROSS) {
#pragma unroll
            for (int odd = 0; odd < 2; ++odd) {
                constexpr uint32_t kChunks = kRow / 16, kLoadRows = 64 / kChunks;   // chunks of a row, rows of a load
                const uint32_t k = kLoadRows * w + lane / kChunks;
                voff[odd] = k * pitch + (((lane % kChunks) ^ swz(k + 4 * kLoadRows * odd)) * 16u);
                round = 4u * kLoadRows * pitch;
            }
            const uint32_t k = 8 * g + (r >> 2);
            rd[0] = lds0 + k * kRow + (((TILE / 16u * patch + ((r >> 1) & 1u)) ^ swz(k)) * 16u) + (r & 1u) * 8u;
            rd[1] = 0;
        } else {
            const uint32_t R = 8 * w + (lane >> 3), c = swz_chunk(R, lane & 7) * 16u;
            voff[0] = voff[1] = R * pitch + c;
            round = 32u * pitch;
            const int nk = (K + kLayoutStep - 1) / kLayoutStep;
            tail_or = (int)c >= 2 * (K - (nk - 1) * kLayoutStep) ? 0x80000000u : 0u;
            rd[0] = lds0 + (TILE / 2u * patch + r) * 128u + swz_chunk(r, g) * 16u;
            rd[1] = lds0 + (TILE / 2u * patch + r) * 128u + swz_chunk(r, g + 4) * 16u;
        }
    }
    // the descriptor's next K-step
    __device__ __forceinline__ void advance(uint32_t step_bytes) {
        base += step_bytes;
        left = left > (int64_t)step_bytes ? left - step_bytes : 0;
    }
    __device__ __forceinline__ v4i srd(bool any) const {
        const uint32_t n = left < 0x7fffffff ? (uint32_t)left : 0x7fffffffu;
        return v4i{(int)(uint32_t)base, (int)((uint32_t)(base >> 32) & 0xffffu), any ? (int)n : 0, 0x00020000};
    }
    // `rows`: round, through opaque() once a K-step: the multiples are formed at each load instead of being held in scalar
    // registers across the whole loop (two products in one kernel spilled 33 of them)
    static __device__ __forceinline__ uint32_t opaque(uint32_t v) {
        asm volatile("" : "+s"(v));
        return v;
    }
    template <int I, int AT = 0>
    __device__ __forceinline__ void load(uint32_t dst, v4i d, uint32_t vor, uint32_t rows) const {
        dma16_at<AT + I * 4096>(d, dst, ACROSS ? voff[I & 1] : voff[0] | vor, I * rows);
    }
    // half H of fragment f, `slot` bytes behind the operand's first slot
    template <int H>
    __device__ __forceinline__ v4i half(int f, uint32_t slot) const {
        if constexpr (ACROSS) {
            const uint32_t at = (rd[0] ^ (32u * f)) + slot;
            const v2i a = lds_read_tr(at + (32 * H) * kRow), b = lds_read_tr(at + (32 * H + 4) * kRow);
            return v4i{a.x, a.y, b.x, b.y};
        } else {
            return *(lds_v4i_t*)(uintptr_t)(rd[H] + slot + f * 2048);
        }
    }
};

// acc of this wave's 128x128 patch (wave w: rows 128 (w / 2), columns 128 (w % 2) of the tile). K > 0.
template <bool A_ACROSS, bool B_ACROSS>
__device__ __forceinline__ void ring_product(uint8_t* smem, const TileOperand& A, const TileOperand& B, int K, v4f (&acc)[8][8]) {
    constexpr int MT = 8, NT = 8, PG = 4, kLoads = 8;
    const uint32_t lds0 = (uint32_t)(uintptr_t)smem, w = wave_id();
    const uint32_t mine_a = to_sgpr(lds0 + w * 1024u), mine_b = to_sgpr(lds0 + 2 * kRingSlot + w * 1024u);
    RingOperand<A_ACROSS> oa;
    RingOperand<B_ACROSS> ob;
    oa.init(A, K, w >> 1, lds0);
    ob.init(B, K, w & 1, lds0 + 2 * kRingSlot);
    const int nk = (K + kLayoutStep - 1) / kLayoutStep;
    const uint32_t step_a = A_ACROSS ? to_sgpr(kLayoutStep * A.pitch) : 128u, step_b = B_ACROSS ? to_sgpr(kLayoutStep * B.pitch) : 128u;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = v4f{0.f, 0.f, 0.f, 0.f};
    struct Frag { v4i lo, hi; };
    Frag bf[2][NT], af[4];

    auto load_all = [&]<bool OP_A>(uint32_t dst, v4i d, uint32_t vor) __attribute__((always_inline)) {
        auto one = [&]<int I>() __attribute__((always_inline)) {
            if constexpr (OP_A) oa.template load<I>(dst, d, vor, oa.round);
            else ob.template load<I>(dst, d, vor, ob.round);
        };
        one.template operator()<0>(); one.template operator()<1>(); one.template operator()<2>(); one.template operator()<3>();
        one.template operator()<4>(); one.template operator()<5>(); one.template operator()<6>(); one.template operator()<7>();
    };
    load_all.template operator()<false>(mine_b, ob.srd(true), nk == 1 ? ob.tail_or : 0u);
    load_all.template operator()<true>(mine_a, oa.srd(true), nk == 1 ? oa.tail_or : 0u);
    wait_vmcnt<0>();
    block_barrier();
    oa.advance(step_a);
    ob.advance(step_b);
    load_all.template operator()<false>(mine_b + kRingSlot, ob.srd(nk > 1), nk == 2 ? ob.tail_or : 0u);
    load_all.template operator()<true>(mine_a + kRingSlot, oa.srd(nk > 1), nk == 2 ? oa.tail_or : 0u);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        bf[0][n].lo = ob.template half<0>(n, 0);
        bf[0][n].hi = ob.template half<1>(n, 0);
    }
#pragma unroll
    for (int m = 0; m < 3; ++m) {
        af[m].lo = oa.template half<0>(m, 0);
        af[m].hi = oa.template half<1>(m, 0);
    }
    // B slots: K-step kt + 1 is read at off1, K-step kt + 2 loaded at off2
    uint32_t off1 = kRingSlot, off2 = 2 * kRingSlot;

    auto step = [&]<int P>(int kt) __attribute__((always_inline)) {
        mfma_enter_agpr(acc);   // (the loop's tail is a branch of its own; no difference in time)
        oa.advance(oa.opaque(step_a));   // (else multiples of it are held for the unrolled K-steps)
        ob.advance(ob.opaque(step_b));
        const bool more = kt + 2 < nk;
        const v4i da = oa.srd(more), db = ob.srd(more);
        const uint32_t vor_a = kt + 2 == nk - 1 ? oa.tail_or : 0u, vor_b = kt + 2 == nk - 1 ? ob.tail_or : 0u;
        const uint32_t rows_a = oa.opaque(oa.round), rows_b = ob.opaque(ob.round);
        auto load_b = [&](int i) __attribute__((always_inline)) {
            switch (i) {
                case 0: ob.template load<0>(mine_b + off2, db, vor_b, rows_b); break;
                case 1: ob.template load<1>(mine_b + off2, db, vor_b, rows_b); break;
                case 2: ob.template load<2>(mine_b + off2, db, vor_b, rows_b); break;
                case 3: ob.template load<3>(mine_b + off2, db, vor_b, rows_b); break;
                case 4: ob.template load<4>(mine_b + off2, db, vor_b, rows_b); break;
                case 5: ob.template load<5>(mine_b + off2, db, vor_b, rows_b); break;
                case 6: ob.template load<6>(mine_b + off2, db, vor_b, rows_b); break;
                default: ob.template load<7>(mine_b + off2, db, vor_b, rows_b); break;
            }
        };
        auto load_a = [&](int i) __attribute__((always_inline)) {
            switch (i) {
                case 0: oa.template load<0, P * kRingSlot>(mine_a, da, vor_a, rows_a); break;
                case 1: oa.template load<1, P * kRingSlot>(mine_a, da, vor_a, rows_a); break;
                case 2: oa.template load<2, P * kRingSlot>(mine_a, da, vor_a, rows_a); break;
                case 3: oa.template load<3, P * kRingSlot>(mine_a, da, vor_a, rows_a); break;
                case 4: oa.template load<4, P * kRingSlot>(mine_a, da, vor_a, rows_a); break;
                case 5: oa.template load<5, P * kRingSlot>(mine_a, da, vor_a, rows_a); break;
                case 6: oa.template load<6, P * kRingSlot>(mine_a, da, vor_a, rows_a); break;
                default: oa.template load<7, P * kRingSlot>(mine_a, da, vor_a, rows_a); break;
            }
        };
        // behind the barrier, slot q (0 .. 47): halves of the next K-step's B fragments, then of its A fragments 0, 1, 2
        // (their registers are free once groups 4, 5 and 6 are done) in the even slots, A's loads at q = 1, 5, ..
        auto post = [&](int q) __attribute__((always_inline)) {
            if ((q & 1) == 0) {
                const int u = q / 2;
                if (u < 2 * NT) {
                    if (u & 1) bf[P ^ 1][u / 2].hi = ob.template half<1>(u / 2, off1);
                    else bf[P ^ 1][u / 2].lo = ob.template half<0>(u / 2, off1);
                } else if (u < 2 * NT + 6) {
                    const int j = (u - 2 * NT) / 2;
                    if (u & 1) af[j].hi = oa.template half<1>(j, (P ^ 1) * kRingSlot);
                    else af[j].lo = oa.template half<0>(j, (P ^ 1) * kRingSlot);
                }
            } else if (q % 4 == 1 && q / 4 < kLoads) {
                load_a(q / 4);
            }
        };
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                mfma_bf16_acc(acc[m][n], bf[P][n].lo, af[m & 3].lo);
                if (m <= PG) {
                    const int s = m * NT + n;
                    if (n == 0) af[(m + 3) & 3].lo = oa.template half<0>(m + 3, P * kRingSlot);
                    if (n == 1) af[(m + 3) & 3].hi = oa.template half<1>(m + 3, P * kRingSlot);
                    if (s % 5 == 2 && s / 5 < kLoads) load_b(s / 5);
                } else {
                    post((m - PG - 1) * 2 * NT + n);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                mfma_bf16_acc(acc[m][n], bf[P][n].hi, af[m & 3].hi);
                if (m > PG) post((m - PG - 1) * 2 * NT + NT + n);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (m == PG) {
                // every read of A slot P has been issued; K-step kt + 1 (all loads but this step's of B) has landed
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                wait_vmcnt<kLoads>();
                block_barrier();
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        off1 = off2;
        off2 = off2 == 2 * kRingSlot ? 0u : off2 + kRingSlot;
    };
    int kt = 0;
    for (; kt + 1 < nk; kt += 2) {
        step.template operator()<0>(kt);
        step.template operator()<1>(kt + 1);
    }
    if (kt < nk) step.template operator()<0>(kt);
    wait_vmcnt<0>();   // nothing may still be writing LDS when the workgroup retires or uses it otherwise
    mfma_drain_agpr(acc);
}

// 128x128 and 64x64 tiles in the same manner, for problems with no more tiles than CUs, where one workgroup has a CU to itself: four or
// eight LDS stages, all but one or two of them ahead, the next fragments read behind the MFMAs of these (a quarter of the tile a wave).
// Weight gradient of 16384 rows, 1024 x 1024, 64 tiles of 256 K-steps: 155 us with two stages of 128x128, 117 with four, 31 bytes a clock
// into each CU, which bounds it (five stages: 116); 256 tiles of 64x64 with a barrier every K-step 70, every second 66. A K-step of
// 64x64 takes 0.23 to 0.25 us, of 128x128 0.45, also where few rows leave most of A's loads without memory behind them: the issue of
// the loads into LDS bounds a CU, not memory.
template <int TILE>
struct DeepStages {
    static constexpr int kStages = TILE == 128 ? 4 : 8, kBytes = 2 * TILE * 128;
    static constexpr int kGroup = TILE == 128 ? 1 : 2;   // K-steps from barrier to barrier
};
template <int TILE, bool A_ACROSS, bool B_ACROSS>
__device__ __forceinline__ void deep_product(uint8_t* smem, const TileOperand& A, const TileOperand& B, int K,
                                             v4f (&acc)[TILE / 32][TILE / 32]) {
    constexpr int S = DeepStages<TILE>::kStages, kStage = DeepStages<TILE>::kBytes, U = DeepStages<TILE>::kGroup, F = TILE / 32, kLoads = TILE / 32;
    const uint32_t lds0 = (uint32_t)(uintptr_t)smem, w = wave_id();
    const uint32_t mine = to_sgpr(lds0 + w * 1024u);
    RingOperand<A_ACROSS, TILE> oa;
    RingOperand<B_ACROSS, TILE> ob;
    oa.init(A, K, w >> 1, lds0);
    ob.init(B, K, w & 1, lds0 + kStage / 2);
    const int nk = (K + kLayoutStep - 1) / kLayoutStep;
    const uint32_t step_a = A_ACROSS ? to_sgpr(kLayoutStep * A.pitch) : 128u, step_b = B_ACROSS ? to_sgpr(kLayoutStep * B.pitch) : 128u;
#pragma unroll
    for (int m = 0; m < F; ++m)
#pragma unroll
        for (int n = 0; n < F; ++n) acc[m][n] = v4f{0.f, 0.f, 0.f, 0.f};
    struct Frag { v4i lo, hi; };
    Frag af[2][U][F], bf[2][U][F];
    v4i da, db;
    uint32_t vor_a = 0, vor_b = 0, rows_a = 0, rows_b = 0;
    auto next_step = [&](int kt) __attribute__((always_inline)) {   // the descriptors' K-step
        da = oa.srd(kt < nk);
        db = ob.srd(kt < nk);
        vor_a = kt == nk - 1 ? oa.tail_or : 0u;
        vor_b = kt == nk - 1 ? ob.tail_or : 0u;
        rows_a = oa.opaque(oa.round);
        rows_b = ob.opaque(ob.round);
        oa.advance(step_a);
        ob.advance(step_b);
    };
    auto load = [&](int i, uint32_t stage) __attribute__((always_inline)) {   // A's loads of a K-step, then B's
        auto one = [&]<int I>() __attribute__((always_inline)) {
            if constexpr (I < kLoads) oa.template load<I>(mine + stage, da, vor_a, rows_a);
            else if constexpr (I < 2 * kLoads) ob.template load<I - kLoads, kStage / 2>(mine + stage, db, vor_b, rows_b);
        };
        switch (i) {
            case 0: one.template operator()<0>(); break;
            case 1: one.template operator()<1>(); break;
            case 2: one.template operator()<2>(); break;
            case 3: one.template operator()<3>(); break;
            case 4: one.template operator()<4>(); break;
            case 5: one.template operator()<5>(); break;
            case 6: one.template operator()<6>(); break;
            default: one.template operator()<7>(); break;
        }
    };
    // half u (0 .. 4 F U - 1) of a group's fragments into register set Q
    auto read = [&]<int Q>(int u, uint32_t group) __attribute__((always_inline)) {
        const int s = u / (4 * F), f = u % (4 * F) / 4, h = u & 1;
        const uint32_t stage = group + s * kStage;
        if ((u & 2) == 0) {
            if (h) bf[Q][s][f].hi = ob.template half<1>(f, stage);
            else bf[Q][s][f].lo = ob.template half<0>(f, stage);
        } else {
            if (h) af[Q][s][f].hi = oa.template half<1>(f, stage);
            else af[Q][s][f].lo = oa.template half<0>(f, stage);
        }
    };
#pragma unroll
    for (int p = 0; p < S; ++p) {
        next_step(p);
#pragma unroll
        for (int i = 0; i < 2 * kLoads; ++i) load(i, p * kStage);
    }
    wait_vmcnt<(S - U) * 2 * kLoads>();
    block_barrier();
#pragma unroll
    for (int u = 0; u < 4 * F * U; ++u) read.template operator()<0>(u, 0u);
    uint32_t at = 0, at1 = U * kStage;   // stages of groups kg and kg + 1
    auto step = [&]<int P>(int kg) __attribute__((always_inline)) {
        // this group's fragments are here, so its stages are free once everyone says so; the next group has landed
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        wait_vmcnt<(S - 2 * U) * 2 * kLoads>();
        block_barrier();
        __builtin_amdgcn_sched_barrier(0);
        mfma_enter_agpr(acc);
#pragma unroll
        for (int s = 0; s < U; ++s) {
            next_step(kg * U + S + s);
#pragma unroll
            for (int m = 0; m < F; ++m)
#pragma unroll
                for (int pass = 0; pass < 2; ++pass)
#pragma unroll
                    for (int n = 0; n < F; ++n) {
                        if (pass == 0) mfma_bf16_acc(acc[m][n], bf[P][s][n].lo, af[P][s][m].lo);
                        else mfma_bf16_acc(acc[m][n], bf[P][s][n].hi, af[P][s][m].hi);
                        const int q = F * (2 * m + pass) + n;
                        if (F == 2) {   // a read behind each, a load behind every second
                            read.template operator()<P ^ 1>(8 * s + q, at1);
                            if (q & 1) load(q / 2, at + s * kStage);
                        } else if (q < 16) {
                            read.template operator()<P ^ 1>(q, at1);
                        } else if (q & 1) {
                            load((q - 16) / 2, at);
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
        }
        at = at1;
        at1 = at1 == (S - U) * kStage ? 0u : at1 + U * kStage;
    };
    const int groups = (nk + U - 1) / U;
    int kg = 0;
    for (; kg + 1 < groups; kg += 2) {
        step.template operator()<0>(kg);
        step.template operator()<1>(kg + 1);
    }
    if (kg < groups) step.template operator()<0>(kg);
    wait_vmcnt<0>();   // nothing may still be writing LDS when the workgroup retires or uses it otherwise
    mfma_drain_agpr(acc);
}

// One 16-row block of a wave's patch (row block m, v[n]: its F column blocks) to C rows of `ldc` elements, C at the patch (rows,
// cols: what is left of C there, cols a multiple of 8). bf16: neighbouring lane groups swap their halves of two column
// blocks, so that a lane stores eight columns in one piece: groups 0 and 2 columns 0..7 and 8..15 of the pair's 32, groups
// 1 and 3 columns 16..23 and 24..31.
template <typename T, int F>
__device__ __forceinline__ void store_block_row(const v4f (&v)[F], int m, T* __restrict__ C, int64_t ldc, int64_t rows, int64_t cols) {
    const int r = lane_id() & 15, g = lane_id() >> 4, row = 16 * m + r;
    T* at = C + row * ldc;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int n = 0; n < F; ++n) {
            const int col = 16 * n + 4 * g;
            if (row < rows && col < cols) *(v4f*)(at + col) = v[n];
        }
    } else {
#pragma unroll
        for (int p = 0; p < F / 2; ++p) {
            v4i out;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const v4f a = v[2 * p], b = v[2 * p + 1];
                const auto s = __builtin_amdgcn_permlane16_swap(pack_bf16(a[2 * h], a[2 * h + 1]), pack_bf16(b[2 * h], b[2 * h + 1]), false, false);
                out[h] = (int)s[0];
                out[2 + h] = (int)s[1];
            }
            const int col = 32 * p + 8 * (g >> 1) + 16 * (g & 1);
            if (row < rows && col < cols) *(v4i*)(at + col) = out;
        }
    }
}
// The whole patch. (A fence behind every row block: without it the compiler holds more of them in registers than there are.)
template <typename T, int F>
__device__ __forceinline__ void store_patch(const v4f (&acc)[F][F], T* __restrict__ C, int64_t ldc, int64_t rows, int64_t cols) {
#pragma unroll
    for (int m = 0; m < F; ++m) {
        store_block_row(acc[m], m, C, ldc, rows, cols);
        slot_fence();
    }
}

// The two tiles as the kernels take them: product() leaves acc[F][F] of 16x16 blocks of the wave's patch, rows
// kPatch (w / 2) and columns kPatch (w % 2) of the tile; read_row() gives an epilogue one row of blocks.
template <int STAGES>
struct LayoutTile128Stages {
    static constexpr int kTile = kLayoutTile, kPatch = kTile / 2, F = 4, kLds = STAGES * kLayoutStageBytes;
    template <bool A_ACROSS, bool B_ACROSS>
    static __device__ __forceinline__ void product(uint8_t* smem, const TileOperand& A, const TileOperand& B, int K, v4f (&acc)[F][F]) {
        tile_product<A_ACROSS, B_ACROSS, STAGES>(smem, A, B, K, acc);
    }
    static __device__ __forceinline__ void read_row(const v4f (&acc)[F], v4f (&v)[F]) {
#pragma unroll
        for (int n = 0; n < F; ++n) v[n] = acc[n];
    }
};
typedef LayoutTile128Stages<2> LayoutTile128;
struct LayoutTile256 {
    static constexpr int kTile = kRingTile, kPatch = kTile / 2, F = 8, kLds = kRingLdsBytes;
    template <bool A_ACROSS, bool B_ACROSS>
    static __device__ __forceinline__ void product(uint8_t* smem, const TileOperand& A, const TileOperand& B, int K, v4f (&acc)[F][F]) {
        ring_product<A_ACROSS, B_ACROSS>(smem, A, B, K, acc);
    }
    // One row of blocks out of the accumulation registers, here and no sooner: an epilogue with branches otherwise has the
    // compiler move all 256 into vector registers at once, and spill.
    static __device__ __forceinline__ void read_row(const v4f (&acc)[F], v4f (&v)[F]) {
#pragma unroll
        for (int n = 0; n < F; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float x;
                asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(x) : "a"(acc[n][j]));
                v[n][j] = x;
            }
    }
};

template <int TILE>
struct LayoutTileDeep {
    static constexpr int kTile = TILE, kPatch = kTile / 2, F = TILE / 32, kLds = DeepStages<TILE>::kStages * DeepStages<TILE>::kBytes;
    template <bool A_ACROSS, bool B_ACROSS>
    static __device__ __forceinline__ void product(uint8_t* smem, const TileOperand& A, const TileOperand& B, int K, v4f (&acc)[F][F]) {
        deep_product<TILE, A_ACROSS, B_ACROSS>(smem, A, B, K, acc);
    }
    static __device__ __forceinline__ void read_row(const v4f (&acc)[F], v4f (&v)[F]) {
#pragma unroll
        for (int n = 0; n < F; ++n) v[n] = acc[n];
    }
};
typedef LayoutTileDeep<128> LayoutTile128Deep;
typedef LayoutTileDeep<64> LayoutTile64Deep;

// Whether 256x256 tiles take less time than 128x128 ones: rounds of workgroups over the CUs (one of the large kernel or two of
// the small one on a CU; a round that is not full is a round, later ones run into each other) times a fixed part and a part per
// K-step, us. The constants are fits to 32 experts of 4096 x 7168: 65536 rows forward 2873 large / 4130 small, gradient of the
// weights with 3, 9 and 33 K-steps 660, 1167, 3013 / 628, 1290, 3738; small_step: the small kernel's K-step, which the gradient of
// the weights (both operands in runs of 256 bytes) takes faster than the others.
constexpr double kLargeFixed = 7.0, kLargeStep = 1.43, kSmallFixed = 2.7, kSmallStepAlong = 1.1, kSmallStepAcross = 0.945;
constexpr double kDeepStep = 0.45;   // LayoutTile128Deep, alone on its CU
inline bool prefer_tile256(double tiles256, double tiles128, double k_steps, int cus, double small_step = kSmallStepAlong) {
    auto rounds = [](double tiles, double at_once) { return tiles <= at_once ? 1.0 : tiles / at_once + 0.2; };
    return rounds(tiles256, cus) * (kLargeFixed + kLargeStep * k_steps) < rounds(tiles128, 2.0 * cus) * (kSmallFixed + small_step * k_steps);
}
// The tile, and for the small ones the number of LDS stages: many where no CU gets a second workgroup anyway, and 64x64 tiles as long as
// there are no more of them than CUs. (us, 128x128 / 64x64: forward of 16 rows of 4 experts of 4096 x 4096, 256 tiles of 64x64, 32.5 / 23.4;
// loss of 60 x 14000 x 1024, 219 tiles, 16.6 / 12.5; more tiles than CUs: loss of 128 x 16000 x 2880, 500 tiles, 29 / 35.)
enum LayoutChoice { kLayout256, kLayout128, kLayout128Deep, kLayout64Deep };
struct LayoutTiles { double t256, t128, t64; };   // how many tiles of each size there are
inline LayoutChoice choose_layout(LayoutTiles tiles, double k_steps, int cus, double small_step = kSmallStepAlong) {
    if (tiles.t64 <= cus) return kLayout64Deep;
    if (prefer_tile256(tiles.t256, tiles.t128, k_steps, cus, small_step)) return kLayout256;
    return tiles.t128 <= cus ? kLayout128Deep : kLayout128;
}

}  // namespace hk
