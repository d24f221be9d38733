// The global norm of a list of gradients, and clipping by it:
//
//   norm = sqrt(sum_i sum_j g_ij^2),   out_ij = g_ij min(1, max_norm / (norm + 1e-6))
//
// HBM bounds both: the gradients are read once for the norm and once to be scaled. A list is any number of bf16 and fp32 tensors of any length
// and alignment, described by a table on the device that a program makes once: one launch goes over all of them. Work is cut into chunks of
// kClipChunk elements, which a workgroup looks up in the table. Squares are added in 64 bits (a square of fp32 does not leave their range,
// and the sum of 2^30 of them keeps fp32's digits), in an order that depends on the list alone.
#include <algorithm>

#include "hk_device.h"
#include "hk_host.h"
#include "../../include/hk355.h"

namespace hk {

constexpr int kClipChunk = 16384;
constexpr int kClipGroups = 2048;   // workgroups of a launch, eight on each of 256 CUs; partial sums of the norm

struct GradEntry {
    uint64_t src, dst;   // dst may be src
    int64_t count;
    int64_t chunk0;      // the list's chunks in front of this tensor's
    int32_t src_fp32, dst_fp32;
};
static_assert(sizeof(GradEntry) == 40);

// The workgroup's chunks: f(entry, from, to), or with REVERSE from the last one to the first. Neighbouring workgroups have neighbouring
// chunks, so that the launch goes through memory front to back (each workgroup a run of its own instead: norm of 2.4 GB 458 us, so 385).
template <bool REVERSE, typename F>
__device__ __forceinline__ void for_chunks(const GradEntry* __restrict__ list, int n, int64_t chunks, F&& f) {
    int at = REVERSE ? n : 0;   // of the chunk before: where the search ends, or begins
    for (int64_t i = blockIdx.x; i < chunks; i += gridDim.x) {
        const int64_t c = REVERSE ? chunks - 1 - i : i;
        // the last tensor whose chunks begin at c or in front of it (tensors without elements have none)
        int lo = REVERSE ? 0 : at, hi = REVERSE ? at : n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (list[mid].chunk0 <= c) lo = mid;
            else hi = mid;
        }
        at = REVERSE ? lo + 1 : lo;
        const GradEntry e = list[lo];
        const int64_t from = (c - e.chunk0) * kClipChunk;
        f(e, from, min(e.count, from + kClipChunk));
    }
}

// Lists of more chunks than the memory-side cache (256 MB) holds in bf16 go past it, but for tensors that the clip converts or meets at two alignments:
// with the non-temporal hint the norm of 2.4 GB takes 342 us instead of 385, the clip 879 instead of 913; smaller ones are still there for the clip
// when the norm has read them. The rule counts chunks, so that fp32, of which 256 MB are half as many, goes past the cache from 512 MB on. (Norm and clip
// in place, us without the hint / with it: lists that the caches held before, bf16 200 MB 99 / 108, 300 MB 153 / 160, 400 MB 210 / 207, fp32 300 MB 155 / 167,
// 500 MB 284 / 272; behind a write of 300 MB, which the figure holds, bf16 200 MB 177 / 155, 300 MB 237 / 206, fp32 300 MB 238 / 211, 500 MB 364 / 320.)
// The clip goes from the last chunk to the first, whose read the caches remember best (both together 1222 us, so 1179).
constexpr int64_t kClipStreamChunks = (256ll << 20) / (2 * kClipChunk);
template <bool NT>
__device__ __forceinline__ v4i load_piece(const v4i* p) {
    if constexpr (NT) return __builtin_nontemporal_load(p);
    else return *p;
}
template <bool NT>
__device__ __forceinline__ void store_piece(v4i* p, v4i v) {
    if constexpr (NT) __builtin_nontemporal_store(v, p);
    else *p = v;
}

// Elements [from, to) of a tensor at `p`: one(i) for those in front of the first and behind the last 16-byte piece, piece(i) for the pieces,
// which begin at element i.
template <int SIZE, typename One, typename Piece>
__device__ __forceinline__ void for_elements(uint64_t p, int64_t from, int64_t to, One&& one, Piece&& piece) {
    constexpr int V = 16 / SIZE;
    const int64_t skip = (int64_t)((16 - ((p + from * SIZE) & 15)) & 15) / SIZE, first = min(from + skip, to);
    const int64_t pieces = (to - first) / V, rest = first + pieces * V;
    if (from + (int64_t)threadIdx.x < first) one(from + threadIdx.x);
    piece(first, pieces);
    if (rest + (int64_t)threadIdx.x < to) one(rest + threadIdx.x);
}

__device__ __forceinline__ float bf16_at(uint64_t p, int64_t i) { return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16); }

template <bool NT>
__global__ __launch_bounds__(256) void grad_square_sum_kernel(const GradEntry* __restrict__ list, int n, int64_t chunks, double* __restrict__ partial) {
    constexpr int kAhead = 4;
    double sum[2] = {0.0, 0.0};
    auto add = [&](float x, int which) { sum[which] = __builtin_fma((double)x, (double)x, sum[which]); };
    for_chunks<false>(list, n, chunks, [&](const GradEntry& e, int64_t from, int64_t to) {
        auto pieces = [&](int64_t first, int64_t count, int size) {
            const v4i* at = (const v4i*)(e.src + first * size);
            for (int64_t i = threadIdx.x; i < count; i += kAhead * 256) {
                v4i q[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) q[k] = i + k * 256 < count ? load_piece<NT>(at + i + k * 256) : v4i{0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < kAhead; ++k)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (size == 4) {
                            add(__int_as_float(q[k][j]), j & 1);
                        } else {
                            add(__uint_as_float((uint32_t)q[k][j] << 16), 0);
                            add(__uint_as_float((uint32_t)q[k][j] & 0xffff0000u), 1);
                        }
                    }
            }
        };
        if (e.src_fp32)
            for_elements<4>(e.src, from, to, [&](int64_t i) { add(((const float*)e.src)[i], 0); }, [&](int64_t a, int64_t b) { pieces(a, b, 4); });
        else
            for_elements<2>(e.src, from, to, [&](int64_t i) { add(bf16_at(e.src, i), 0); }, [&](int64_t a, int64_t b) { pieces(a, b, 2); });
    });
    __shared__ double part[4];
    double all = sum[0] + sum[1];
    for (int d = 32; d >= 1; d >>= 1) all += __shfl_xor(all, d, 64);
    if (lane_id() == 0) part[wave_id()] = all;
    __syncthreads();
    if (threadIdx.x == 0) partial[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

__global__ __launch_bounds__(1024) void grad_norm_kernel(const double* __restrict__ partial, int n, float* __restrict__ norm) {
    __shared__ double part[16];
    double all = 0.0;
    for (int i = threadIdx.x; i < n; i += 1024) all += partial[i];
    for (int d = 32; d >= 1; d >>= 1) all += __shfl_xor(all, d, 64);
    if (lane_id() == 0) part[wave_id()] = all;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) all += part[w];
        norm[0] = (float)__builtin_sqrt(all);
    }
}

template <bool NT>
__global__ __launch_bounds__(256) void grad_clip_kernel(const GradEntry* __restrict__ list, int n, int64_t chunks, const float* __restrict__ norm,
                                                        float max_norm) {
    const float ratio = max_norm / (norm[0] + 1e-6f), factor = ratio >= 1.0f ? 1.0f : ratio;   // (a NaN stays one)
    for_chunks<true>(list, n, chunks, [&](const GradEntry& e, int64_t from, int64_t to) {
        if (factor == 1.0f && e.src == e.dst) return;   // in place, nothing to scale
        auto get = [&](int64_t i) { return e.src_fp32 ? ((const float*)e.src)[i] : bf16_at(e.src, i); };
        auto put = [&](int64_t i, float v) {
            if (e.dst_fp32) ((float*)e.dst)[i] = v;
            else ((uint16_t*)e.dst)[i] = (uint16_t)(pack_bf16(v, 0.f) & 0xffffu);
        };
        auto one = [&](int64_t i) { put(i, get(i) * factor); };
        // 16-byte pieces where both sides reach such an address with the same element; of different types, where both begin at one
        const uint64_t src = e.src + from * (e.src_fp32 ? 4 : 2), dst = e.dst + from * (e.dst_fp32 ? 4 : 2);
        if (e.src_fp32 != e.dst_fp32 && ((src | dst) & 15) == 0) {
            auto convert = [&](auto* at, auto* out) {
                const int64_t count = (to - from) / 8;
                for (int64_t i = threadIdx.x; i < count; i += 2 * 256) {
                    Row8 a = load8(at + 8 * i), b{};
                    const bool two = i + 256 < count;
                    if (two) b = load8(at + 8 * (i + 256));
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        a.v[j] *= factor;
                        b.v[j] *= factor;
                    }
                    store8(out + 8 * i, a);
                    if (two) store8(out + 8 * (i + 256), b);
                }
            };
            if (e.src_fp32) convert((const float*)src, (uint16_t*)dst);
            else convert((const uint16_t*)src, (float*)dst);
            const int64_t rest = from + (to - from) / 8 * 8;
            if (rest + (int64_t)threadIdx.x < to) one(rest + threadIdx.x);
            return;
        }
        if (e.src_fp32 != e.dst_fp32 || ((src ^ dst) & 15) != 0) {
            for (int64_t i = from + threadIdx.x; i < to; i += 256) one(i);
            return;
        }
        constexpr int kAhead = 4;
        auto pieces = [&](int64_t first, int64_t count, int size) {
            const v4i* at = (const v4i*)(e.src + first * size);
            v4i* out = (v4i*)(e.dst + first * size);
            for (int64_t i = threadIdx.x; i < count; i += kAhead * 256) {
                v4i q[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) q[k] = i + k * 256 < count ? load_piece<NT>(at + i + k * 256) : v4i{0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (size == 4) q[k][j] = __float_as_int(__int_as_float(q[k][j]) * factor);
                        else q[k][j] = (int)pack_bf16(__uint_as_float((uint32_t)q[k][j] << 16) * factor,
                                                      __uint_as_float((uint32_t)q[k][j] & 0xffff0000u) * factor);
                    }
                    if (i + k * 256 < count) store_piece<NT>(out + i + k * 256, q[k]);
                }
            }
        };
        if (e.src_fp32) for_elements<4>(e.src, from, to, one, [&](int64_t a, int64_t b) { pieces(a, b, 4); });
        else for_elements<2>(e.src, from, to, one, [&](int64_t a, int64_t b) { pieces(a, b, 2); });
    });
}

static int clip_groups(int64_t chunks) { return (int)std::min<int64_t>(chunks, kClipGroups); }

}  // namespace hk

extern "C" size_t hk_grad_list_bytes(int n) { return n > 0 && n <= (1 << 20) ? (size_t)n * sizeof(hk::GradEntry) : 0; }

extern "C" int hk_grad_list_fill(const void* const* grads, void* const* outs_or_null, const int64_t* counts, const int32_t* types,
                                 const int32_t* out_types_or_null, int n, void* list, size_t list_bytes, int64_t* chunks) {
    using namespace hk;
    if (!grads || !counts || !types || !list || !chunks || (outs_or_null && !out_types_or_null)) return HK_ERR_NULL_POINTER;
    if (hk_grad_list_bytes(n) == 0) return HK_ERR_BAD_SHAPE;
    if (list_bytes < hk_grad_list_bytes(n)) return HK_ERR_WORKSPACE;
    GradEntry* entries = (GradEntry*)list;
    int64_t at = 0;
    for (int i = 0; i < n; ++i) {
        const int64_t count = counts[i];
        const int type = types[i], out_type = outs_or_null ? out_types_or_null[i] : type;
        if ((type != 0 && type != 1) || (out_type != 0 && out_type != 1)) return HK_ERR_UNSUPPORTED;
        if (count < 0 || count >= (1ll << 40)) return HK_ERR_BAD_SHAPE;
        const void* out = outs_or_null ? outs_or_null[i] : grads[i];
        if (count > 0 && (!grads[i] || !out)) return HK_ERR_NULL_POINTER;
        if (count > 0 && out == grads[i] && type != out_type) return HK_ERR_UNSUPPORTED;
        if (((uintptr_t)grads[i] % (type ? 4 : 2)) || ((uintptr_t)out % (out_type ? 4 : 2))) return HK_ERR_BAD_ALIGNMENT;
        entries[i] = GradEntry{(uint64_t)(uintptr_t)grads[i], (uint64_t)(uintptr_t)out, count, at, type, out_type};
        at += (count + kClipChunk - 1) / kClipChunk;
    }
    *chunks = at;
    return HK_OK;
}

extern "C" size_t hk_grad_norm_workspace_bytes(void) { return hk::kClipGroups * sizeof(double); }

extern "C" int hk_grad_norm(const void* list, int n, int64_t chunks, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace hk;
    if (!list || !norm) return HK_ERR_NULL_POINTER;
    if (hk_grad_list_bytes(n) == 0 || chunks < 0 || chunks >= (1ll << 40)) return HK_ERR_BAD_SHAPE;
    if (((uintptr_t)list & 7u) || ((uintptr_t)workspace & 15u) || ((uintptr_t)norm & 3u)) return HK_ERR_BAD_ALIGNMENT;
    if (!workspace || workspace_bytes < hk_grad_norm_workspace_bytes()) return HK_ERR_WORKSPACE;
    const hipStream_t s = (hipStream_t)stream;
    const int groups = clip_groups(chunks);
    if (groups > 0)
        hipLaunchKernelGGL(chunks > kClipStreamChunks ? grad_square_sum_kernel<true> : grad_square_sum_kernel<false>, dim3(groups), dim3(256), 0, s,
                           (const GradEntry*)list, n, chunks, (double*)workspace);
    hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(1024), 0, s, (const double*)workspace, groups, norm);
    return hipGetLastError() == hipSuccess ? HK_OK : HK_ERR_LAUNCH;
}

extern "C" int hk_grad_clip(const void* list, int n, int64_t chunks, const float* norm, float max_norm, void* stream) {
    using namespace hk;
    if (!list || !norm) return HK_ERR_NULL_POINTER;
    if (hk_grad_list_bytes(n) == 0 || chunks < 0 || chunks >= (1ll << 40)) return HK_ERR_BAD_SHAPE;
    if (((uintptr_t)list & 7u) || ((uintptr_t)norm & 3u)) return HK_ERR_BAD_ALIGNMENT;
    if (!(max_norm >= 0.f)) return HK_ERR_UNSUPPORTED;
    const int groups = clip_groups(chunks);
    if (groups == 0) return HK_OK;
    hipLaunchKernelGGL(chunks > kClipStreamChunks ? grad_clip_kernel<true> : grad_clip_kernel<false>, dim3(groups), dim3(256), 0,
                       (hipStream_t)stream, (const GradEntry*)list, n, chunks, norm, max_norm);
    return hipGetLastError() == hipSuccess ? HK_OK : HK_ERR_LAUNCH;
}
