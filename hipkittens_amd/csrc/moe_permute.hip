// Tokens to the order of their experts and back in bf16, for training: the row copies and the gradients around the
// weighted un-permute (moe_unpermute_kernel). S = T k slots, pos = slot_to_pos[t k + j]; a position outside [0, S) has no
// row: nothing is read or written there.
//
//   permute              xp[pos(t, j)] = x[t]
//   permute, backward    dx[t] = add[t] + sum_j dxp[pos(t, j)]    (moe_unpermute_kernel without weights)
//   unpermute, backward  do[pos(t, j)] = w[t, j] dy[t],  dw[t, j] = <dy[t], o[pos(t, j)]>
//
// All of them move rows and nothing else, so HBM bounds them. They go token by token rather than position by position:
// a token's row is read once for its k copies, and dy for both gradients.
#include "moe_common.h"
#include "../../include/hk355.h"

namespace hk {

__device__ __forceinline__ float bf16_lo(int v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ float bf16_hi(int v) { return __uint_as_float((uint32_t)v & 0xffff0000u); }

// KU: choices whose positions are held in registers (0: any number, read again for every column chunk). The workgroups of
// one token (gridDim.y) share its columns.
template <int KU>
__global__ __launch_bounds__(256) void moe_permute_kernel(const uint16_t* __restrict__ x, const int32_t* __restrict__ slot_to_pos,
                                                          int T, int k, int H, uint16_t* __restrict__ xp) {
    const int t = blockIdx.x;
    const uint32_t n_rows = (uint32_t)T * (uint32_t)k;
    int pos[KU > 0 ? KU : 1];
#pragma unroll
    for (int j = 0; j < KU; ++j) pos[j] = j < k ? slot_to_pos[(size_t)t * k + j] : -1;
    for (int c = blockIdx.y * blockDim.x + threadIdx.x; c < H / 8; c += gridDim.y * blockDim.x) {
        const v4i row = *(const v4i*)(x + (size_t)t * H + c * 8);
        if constexpr (KU > 0) {
#pragma unroll
            for (int j = 0; j < KU; ++j)
                if ((uint32_t)pos[j] < n_rows) *(v4i*)(xp + (size_t)pos[j] * H + c * 8) = row;
        } else {
            for (int j = 0; j < k; ++j) {
                const int p = slot_to_pos[(size_t)t * k + j];
                if ((uint32_t)p < n_rows) *(v4i*)(xp + (size_t)p * H + c * 8) = row;
            }
        }
    }
}

// One workgroup per token and KU of its choices (gridDim.y): the products with dy are summed over the row in fp32, per
// thread, then over the wave and the four waves in a fixed order.
template <int KU>
__global__ __launch_bounds__(256) void moe_unpermute_backward_kernel(const uint16_t* __restrict__ dy, const uint16_t* __restrict__ o,
                                                                     const float* __restrict__ w,
                                                                     const int32_t* __restrict__ slot_to_pos, int T, int k, int H,
                                                                     uint16_t* __restrict__ d_o, float* __restrict__ dw) {
    __shared__ float part[4][KU];
    const int t = blockIdx.x, j0 = blockIdx.y * KU;
    const uint32_t n_rows = (uint32_t)T * (uint32_t)k;
    int pos[KU];
    float wt[KU], dot[KU];
#pragma unroll
    for (int j = 0; j < KU; ++j) {
        const bool in = j0 + j < k;
        pos[j] = in ? slot_to_pos[(size_t)t * k + j0 + j] : -1;
        wt[j] = in ? w[(size_t)t * k + j0 + j] : 0.f;
        dot[j] = 0.f;
    }
    for (int c = threadIdx.x; c < H / 8; c += 256) {
        const v4i g = *(const v4i*)(dy + (size_t)t * H + c * 8);
        v4i row[KU];
#pragma unroll
        for (int j = 0; j < KU; ++j)
            if ((uint32_t)pos[j] < n_rows) row[j] = __builtin_nontemporal_load((const v4i*)(o + (size_t)pos[j] * H + c * 8));
#pragma unroll
        for (int j = 0; j < KU; ++j)
            if ((uint32_t)pos[j] < n_rows) {
                v4i out;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    out[i] = (int)pack_bf16(wt[j] * bf16_lo(g[i]), wt[j] * bf16_hi(g[i]));
                    dot[j] += bf16_lo(g[i]) * bf16_lo(row[j][i]);
                    dot[j] += bf16_hi(g[i]) * bf16_hi(row[j][i]);
                }
                *(v4i*)(d_o + (size_t)pos[j] * H + c * 8) = out;
            }
    }
#pragma unroll
    for (int j = 0; j < KU; ++j) {
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) dot[j] += __shfl_xor(dot[j], off, 64);
        if (lane_id() == 0) part[threadIdx.x >> 6][j] = dot[j];
    }
    __syncthreads();
    const int j = threadIdx.x;
    if (j < KU && j0 + j < k) dw[(size_t)t * k + j0 + j] = part[0][j] + part[1][j] + part[2][j] + part[3][j];
}

static int permute_check(int T, int k, int H, uintptr_t pointers) {
    // (a workgroup of 256 threads per token, and a launch has fewer than 2^32)
    if (T <= 0 || T >= (1 << 24) || k <= 0 || H <= 0 || (H % 8) != 0 || (long long)T * k > (1ll << 30)) return HK_ERR_BAD_SHAPE;
    return (pointers & 15u) ? HK_ERR_BAD_ALIGNMENT : HK_OK;
}

}  // namespace hk

extern "C" int hk_moe_permute(const void* x_bf16, const int32_t* slot_to_pos, int T, int k, int H, void* xp_bf16, void* stream) {
    using namespace hk;
    if (!x_bf16 || !slot_to_pos || !xp_bf16) return HK_ERR_NULL_POINTER;
    if (const int st = permute_check(T, k, H, (uintptr_t)x_bf16 | (uintptr_t)xp_bf16)) return st;
    auto kern = k <= 4 ? moe_permute_kernel<4> : k <= 8 ? moe_permute_kernel<8> : moe_permute_kernel<0>;
    // fewer tokens than CUs: one-wave workgroups of a column chunk per lane, as in the un-permute
    const bool split = T < moe_num_compute_units();
    hipLaunchKernelGGL(kern, dim3(T, split ? min((H / 8 + 63) / 64, 65535) : 1), dim3(split ? 64 : 256), 0, (hipStream_t)stream,
                       (const uint16_t*)x_bf16, slot_to_pos, T, k, H, (uint16_t*)xp_bf16);
    return hipGetLastError() == hipSuccess ? HK_OK : HK_ERR_LAUNCH;
}

extern "C" int hk_moe_permute_backward(const void* dxp_bf16, const int32_t* slot_to_pos, int T, int k, int H,
                                       const void* add_bf16_or_null, void* dx_bf16, void* stream) {
    using namespace hk;
    if (!dxp_bf16 || !slot_to_pos || !dx_bf16) return HK_ERR_NULL_POINTER;
    if (const int st = permute_check(T, k, H, (uintptr_t)dxp_bf16 | (uintptr_t)dx_bf16 | (uintptr_t)add_bf16_or_null)) return st;
    return moe_launch_unpermute(dxp_bf16, nullptr, slot_to_pos, T, k, H, add_bf16_or_null, dx_bf16, (hipStream_t)stream);
}

extern "C" int hk_moe_unpermute_backward(const void* dy_bf16, const void* o_bf16, const float* w, const int32_t* slot_to_pos, int T,
                                         int k, int H, void* do_bf16, float* dw, void* stream) {
    using namespace hk;
    if (!dy_bf16 || !o_bf16 || !w || !slot_to_pos || !do_bf16 || !dw) return HK_ERR_NULL_POINTER;
    if (const int st = permute_check(T, k, H, (uintptr_t)dy_bf16 | (uintptr_t)o_bf16 | (uintptr_t)do_bf16)) return st;
    if (k > 65535) return HK_ERR_BAD_SHAPE;   // gridDim.y
    auto kern = k <= 4 ? moe_unpermute_backward_kernel<4> : moe_unpermute_backward_kernel<8>;
    const int ku = k <= 4 ? 4 : 8;
    hipLaunchKernelGGL(kern, dim3(T, (k + ku - 1) / ku), dim3(256), 0, (hipStream_t)stream, (const uint16_t*)dy_bf16,
                       (const uint16_t*)o_bf16, w, slot_to_pos, T, k, H, (uint16_t*)do_bf16, dw);
    return hipGetLastError() == hipSuccess ? HK_OK : HK_ERR_LAUNCH;
}
