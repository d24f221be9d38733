// The embedding in front of a model's blocks: rows of a table [V, H] by token, times a scale, and the table's gradient.
//
//   forward    out[t] = scale table[id[t]]; zeros for an id outside [0, V)
//   backward   dtable[v] = add[v] + scale sum_{t: id[t] = v} dout[t]
//
// Both move rows, and HBM bounds them. The gradient needs every row's tokens together and in an order of their own: the tokens are sorted by id
// (stable, digit by digit from the lowest), and blocks of the sorted list are summed in order, so that results are the same on every call and
// no value goes through an atomic. Rows without tokens get zeros (or a copy of `add`): the first rows, whether they have tokens or not, in
// the launches that sort, whose few workgroups would leave the chip idle (those with tokens are then written a second time); the
// others beside the sums, where a search of the sorted list finds no token. A row whose tokens are spread over several blocks
// leaves fp32 partial sums, which the last launch joins in order.
#include <algorithm>

#include "hk_device.h"
#include "hk_host.h"
#include "../../include/hk355.h"

namespace hk {

struct Ids {
    const void* p;
    int is64;
    // the id of token t, -1 outside [0, V)
    __device__ __forceinline__ int at(int64_t t, int V) const {
        const int64_t l = is64 ? ((const int64_t*)p)[t] : (int64_t)((const int32_t*)p)[t];
        return l >= 0 && l < V ? (int)l : -1;
    }
};

// A wave takes LOADS times 64 pieces of eight columns of one token (gridDim.y: the parts of a row), all of its loads in flight together.
// STREAM: the stores go past the caches.
template <typename T, int LOADS, bool STREAM>
__global__ __launch_bounds__(256) void embedding_kernel(Ids ids, const T* __restrict__ table, uint16_t* __restrict__ out, int tokens, int V,
                                                        int H, float scale) {
    const int64_t t = (int64_t)blockIdx.x * 4 + wave_id();
    if (t >= tokens) return;
    const int id = to_sgpr(ids.at(t, V)), pieces = H / 8;
    const int first = blockIdx.y * (64 * LOADS) + lane_id();
    Row8 r[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        r[i] = Row8{};
        if (id >= 0 && first + 64 * i < pieces) r[i] = load8(table + (int64_t)id * H + (int64_t)(first + 64 * i) * 8);
    }
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        if (first + 64 * i >= pieces) break;
#pragma unroll
        for (int j = 0; j < 8; ++j) r[i].v[j] = id >= 0 ? r[i].v[j] * scale : 0.f;
        uint16_t* at = out + t * H + (int64_t)(first + 64 * i) * 8;
        if constexpr (STREAM) __builtin_nontemporal_store(pack8(r[i]), (v4i*)at);
        else *(v4i*)at = pack8(r[i]);
    }
}

// ------------------------------------------------------------------------------------------------ sort
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64, kSortIter = 4;
constexpr int kSortChunk = kSortThreads * kSortIter;   // tokens of a workgroup
constexpr int kSortAlone = 2 * kSortChunk;             // most that one workgroup sorts by itself
constexpr int kMaxDigitBits = 9, kMaxDigits = 1 << kMaxDigitBits;

// Bytes that a launch that sorts writes besides, about what takes as long as it does: zeros (which the memory-side cache takes for a table that
// fits it), or copies of `add`, more of them beside the longest lists that one workgroup sorts. (us: 1111 tokens of 50257 rows of 1024 in bf16, 24 MB of
// zeros 31.8, 48 28.0, 128 26.3, written over and over 72 28.9, 128 26.0; 700 tokens of 20000 rows in fp32 with `add`, copies of 24 MB 42.1,
// 64 48.8; 20000 tokens of 50000 rows 121, 137; 8000 of 30000 rows in bf16, 48 MB 46.5, 64 42.9.)
constexpr size_t kSortZeros = (size_t)128 << 20, kSortCopies = (size_t)24 << 20, kSortCopiesLong = (size_t)64 << 20;
// What the sorting launches write besides: `out`'s 16-byte pieces [from, to), from `add` or zeros.
struct Fill {
    v4i* out;
    const v4i* add;   // null: zeros
    size_t from, to;
    int groups;
    int stream;   // more than the memory-side cache holds: past it
};
template <bool STREAM>
__device__ __forceinline__ void fill_pieces(const Fill& f, int group) {
    auto get = [&](size_t i) {
        if (!f.add) return v4i{0, 0, 0, 0};
        if constexpr (STREAM) return __builtin_nontemporal_load(f.add + i);
        else return f.add[i];
    };
    auto put = [&](size_t i, v4i v) {
        if constexpr (STREAM) __builtin_nontemporal_store(v, f.out + i);
        else f.out[i] = v;
    };
    const size_t step = (size_t)f.groups * kSortThreads;
    size_t i = f.from + (size_t)group * kSortThreads + threadIdx.x;
    for (; i + 3 * step < f.to; i += 4 * step) {
        v4i v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = get(i + j * step);
#pragma unroll
        for (int j = 0; j < 4; ++j) put(i + j * step, v[j]);
    }
    for (; i < f.to; i += step) put(i, get(i));
}
__device__ __forceinline__ void fill(const Fill& f, int group) {
    if (f.stream) fill_pieces<true>(f, group);
    else fill_pieces<false>(f, group);
}

struct Digit {
    int shift, bits;
    __device__ __forceinline__ int of(int key) const { return (key >> shift) & ((1 << bits) - 1); }
    __host__ __device__ __forceinline__ int count() const { return 1 << bits; }
};

// The lanes whose `value` (of `bits` bits) is this lane's, among those of `live`.
__device__ __forceinline__ uint64_t same_value(int value, int bits, uint64_t live) {
    uint64_t same = live;
    for (int b = 0; b < bits; ++b) {
        const bool one = value >> b & 1;
        const uint64_t ones = __ballot(one);
        same &= one ? ones : ~ones;
    }
    return same;
}

struct SortLds {
    int count[kSortWaves][kMaxDigits];   // of a wave's items; then where its first item of a digit goes
    int base[kMaxDigits];
    int wave_sum[kMaxDigits / 64];
};
// Exclusive prefix of the counts of `digits` digits (thread d holds digit d's) to lds.base, their sum returned. One call per pass.
__device__ __forceinline__ int scan_digits(SortLds& lds, int mine, int digits) {
    const int tid = threadIdx.x, lane = lane_id();
    int upto = tid < digits ? mine : 0;
    const int own = upto;
    for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(upto, d, 64);
        if (lane >= d) upto += u;
    }
    if (tid < kMaxDigits && lane == 63) lds.wave_sum[tid / 64] = upto;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kMaxDigits / 64; ++w) {
        before += w < tid / 64 ? lds.wave_sum[w] : 0;
        all += lds.wave_sum[w];
    }
    if (tid < digits) lds.base[tid] = before + upto - own;
    return all;
}

// A workgroup's items (key -1: none) in the order of wave, iteration and lane: rank[i] = how many of the wave's items before this one have its
// digit; lds.count then holds the waves' counts. lds.count must be zero and everyone past that.
template <int ITER>
__device__ __forceinline__ void rank_items(SortLds& lds, const int (&key)[ITER], Digit digit, int (&rank)[ITER]) {
    int* count = lds.count[wave_id()];
    const uint64_t below = (1ull << lane_id()) - 1;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const bool live = key[i] >= 0;
        const int d = live ? digit.of(key[i]) : 0;
        const uint64_t same = same_value(d, digit.bits, __ballot(live));
        const int before = __popcll(same & below);
        rank[i] = live ? count[d] + before : 0;
        slot_fence();   // (every lane has read before one of them writes, and the next iteration reads behind that)
        if (live && before == 0) count[d] += __popcll(same);
        slot_fence();
    }
}
// lds.count of wave w and digit d: where the wave's first item of the digit goes. Behind a barrier on count and base; ends with one.
__device__ __forceinline__ void place_waves(SortLds& lds, int digits, int base) {
    if ((int)threadIdx.x < digits) {
        int at = base;
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) {
            const int n = lds.count[w][threadIdx.x];
            lds.count[w][threadIdx.x] = at;
            at += n;
        }
    }
    __syncthreads();
}
__device__ __forceinline__ void clear_counts(SortLds& lds, Digit digit) {
    for (int i = threadIdx.x; i < kSortWaves << digit.bits; i += kSortThreads) lds.count[i >> digit.bits][i & (digit.count() - 1)] = 0;
    __syncthreads();
}

// Tokens of one workgroup, ITER a thread: all passes at once, the items in LDS in between. (7 tokens of 1036 rows with one a thread 4.7 us, with four
// 7.3; 8192 tokens of 50257 rows: in one workgroup 35 us for the
// whole gradient of 1024 columns, in two by launches 42.)
template <int ITER>
__global__ __launch_bounds__(kSortThreads) void embedding_sort_one_kernel(Ids ids, int T, int V, int passes, int bits, int2* __restrict__ sorted,
                                                                          int* __restrict__ length, Fill f) {
    if (blockIdx.x > 0) return fill(f, blockIdx.x - 1);
    __shared__ SortLds lds;
    __shared__ int2 items[ITER * kSortThreads];
    int key[ITER], token[ITER], rank[ITER];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        token[i] = (wave_id() * ITER + i) * 64 + lane_id();
        key[i] = token[i] < T ? ids.at(token[i], V) : -1;
    }
    for (int pass = 0; pass < passes; ++pass) {
        const Digit digit{pass * bits, bits};
        clear_counts(lds, digit);
        rank_items(lds, key, digit, rank);
        __syncthreads();
        int total = 0;
        if ((int)threadIdx.x < digit.count())
            for (int w = 0; w < kSortWaves; ++w) total += lds.count[w][threadIdx.x];
        const int all = scan_digits(lds, total, digit.count());
        place_waves(lds, digit.count(), (int)threadIdx.x < digit.count() ? lds.base[threadIdx.x] : 0);
        int2* out = pass + 1 < passes ? items : sorted;
#pragma unroll
        for (int i = 0; i < ITER; ++i)
            if (key[i] >= 0) out[lds.count[wave_id()][digit.of(key[i])] + rank[i]] = make_int2(key[i], token[i]);
        if (threadIdx.x == 0) *length = all;
        if (pass + 1 == passes) break;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int at = (wave_id() * ITER + i) * 64 + lane_id();
            const int2 item = at < all ? items[at] : make_int2(-1, 0);
            key[i] = item.x;
            token[i] = item.y;
        }
    }
}

// How often every digit of the first pass occurs in each chunk; the counts of the passes behind it start at zero.
__global__ __launch_bounds__(kSortThreads) void embedding_count_kernel(Ids ids, int T, int V, int chunks, Digit digit, int* __restrict__ counts,
                                                                       int passes, Fill f) {
    if ((int)blockIdx.x >= chunks) return fill(f, blockIdx.x - chunks);
    __shared__ int count[kMaxDigits];
    const int digits = digit.count();
    if ((int)threadIdx.x < digits) count[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSortIter; ++i) {
        const int64_t t = (int64_t)blockIdx.x * kSortChunk + i * kSortThreads + threadIdx.x;
        const int key = t < T ? ids.at(t, V) : -1;
        if (key >= 0) atomicAdd(&count[digit.of(key)], 1);
    }
    __syncthreads();
    for (int p = 0; p < passes; ++p)
        if ((int)threadIdx.x < digits) counts[((size_t)p * chunks + blockIdx.x) * digits + threadIdx.x] = p == 0 ? count[threadIdx.x] : 0;
}

// Counts of the next pass that a workgroup gathers in LDS; more (many chunks) go to memory wave by wave. (65536 tokens of 1000 rows, 16 chunks:
// 22.6 us wave by wave, every wave's frequent ids at the same counts.)
constexpr int kNextCounts = 8192;
// One pass: the items of a chunk to their places. The first reads the ids, and drops what is no row; the others `in`. The counts of the
// next pass's chunks are made on the way (sums of integers: their order does not matter).
__global__ __launch_bounds__(kSortThreads) void embedding_scatter_kernel(Ids ids, const int2* __restrict__ in, int T, int V, int chunks, Digit digit,
                                                                         const int* __restrict__ counts, int* __restrict__ next_counts,
                                                                         int2* __restrict__ out, int* __restrict__ length, Fill f) {
    if ((int)blockIdx.x >= chunks) return fill(f, blockIdx.x - chunks);
    __shared__ SortLds lds;
    __shared__ int next_here[kNextCounts];
    const int digits = digit.count(), c = blockIdx.x;
    const bool gather = next_counts && chunks * digits <= kNextCounts;
    if (gather)
        for (int i = threadIdx.x; i < chunks * digits; i += kSortThreads) next_here[i] = 0;   // (barriers behind it: scan_digits')
    int total = 0, before = 0;
    if ((int)threadIdx.x < digits) {
#pragma unroll 8
        for (int i = 0; i < chunks; ++i) {
            const int n = counts[(size_t)i * digits + threadIdx.x];
            total += n;
            before += i < c ? n : 0;
        }
    }
    const int all = scan_digits(lds, total, digits);
    if (c == 0 && threadIdx.x == 0) *length = all;
    int key[kSortIter], token[kSortIter], rank[kSortIter];
#pragma unroll
    for (int i = 0; i < kSortIter; ++i) {
        const int64_t at = (int64_t)c * kSortChunk + (wave_id() * kSortIter + i) * 64 + lane_id();
        if (in) {
            const int2 item = at < all ? in[at] : make_int2(-1, 0);
            key[i] = item.x;
            token[i] = item.y;
        } else {
            key[i] = at < T ? ids.at(at, V) : -1;
            token[i] = (int)at;
        }
    }
    clear_counts(lds, digit);
    rank_items(lds, key, digit, rank);
    __syncthreads();
    place_waves(lds, digits, (int)threadIdx.x < digits ? lds.base[threadIdx.x] + before : 0);
    const Digit next{digit.shift + digit.bits, digit.bits};
    const int chunk_bits = 32 - __clz(chunks - 1);
#pragma unroll
    for (int i = 0; i < kSortIter; ++i) {
        const bool live = key[i] >= 0;
        const int pos = live ? lds.count[wave_id()][digit.of(key[i])] + rank[i] : 0;
        if (live) out[pos] = make_int2(key[i], token[i]);
        const int at = live ? (pos / kSortChunk) * digits + next.of(key[i]) : 0;
        if (gather) {
            if (live) atomicAdd(&next_here[at], 1);
        } else if (next_counts) {   // one addition per chunk and digit of the wave's
            const uint64_t same = same_value(at, digit.bits + chunk_bits, __ballot(live));
            if (live && (same & ((1ull << lane_id()) - 1)) == 0) atomicAdd(next_counts + at, __popcll(same));
        }
    }
    if (gather) {
        __syncthreads();
        for (int i = threadIdx.x; i < chunks * digits; i += kSortThreads)
            if (next_here[i]) atomicAdd(next_counts + i, next_here[i]);
    }
}

// ------------------------------------------------------------------------------------------------ sums
struct EmbedSums {
    const int2* sorted;   // (row, token), ascending
    const int* length;
    const uint16_t* dout;
    float* partial;       // [blocks][2][H]: of a row whose tokens began in an earlier block, of one whose tokens go on in the next
    int H, block;         // block: tokens of a block, 64 at most
    float scale;
};
template <typename T>
__device__ __forceinline__ void write_row(const EmbedSums& p, T* dtable, int row, int col, bool add, const Row8& a, Row8 r) {
#pragma unroll
    for (int j = 0; j < 8; ++j) r.v[j] = add ? __builtin_fmaf(p.scale, r.v[j], a.v[j]) : p.scale * r.v[j];
    store8(dtable + (size_t)row * p.H + col, r);
}

// Rows [from, to) without tokens: zeros, or a copy of `add`; a workgroup takes `rows` of them (4 to kRestRows), a thread finds out whether its row has
// tokens, a wave writes a row.
struct EmbedRest {
    int from, to, rows;   // rows of a workgroup
    int stream;           // more than the memory-side cache holds: past it
};
constexpr int kRestRows = 256;
template <bool STREAM, typename T>
__device__ __forceinline__ void rest_rows(const EmbedSums& p, const EmbedRest& rest, int group, int length, const T* add, T* dtable) {
    __shared__ uint8_t has[kRestRows];
    const int row0 = rest.from + group * rest.rows, n = min(rest.rows, rest.to - row0);
    if ((int)threadIdx.x < n) {
        const int row = row0 + threadIdx.x;
        int lo = 0, hi = length;   // the first item of the row or behind it
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (p.sorted[mid].x < row) lo = mid + 1;
            else hi = mid;
        }
        has[threadIdx.x] = lo < length && p.sorted[lo].x == row;
    }
    __syncthreads();
    const int pieces = p.H * (int)sizeof(T) / 16;
    for (int r = wave_id(); r < n; r += 4) {
        if (has[r]) continue;
        const v4i* in = (const v4i*)(add + (size_t)(row0 + r) * p.H);
        v4i* out = (v4i*)(dtable + (size_t)(row0 + r) * p.H);
        for (int i = lane_id(); i < pieces; i += 4 * 64) {
            v4i v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[k] = v4i{0, 0, 0, 0};
                if (add && i + 64 * k < pieces) v[k] = STREAM ? __builtin_nontemporal_load(in + i + 64 * k) : in[i + 64 * k];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + 64 * k < pieces) {
                    if (STREAM) __builtin_nontemporal_store(v[k], out + i + 64 * k);
                    else out[i + 64 * k] = v[k];
                }
        }
    }
}

// A wave: the tokens of one block, in order, 512 columns of them, eight rows in flight, and with them what is added to the rows that
// end among them. The workgroups behind those of the sums write the rows without tokens.
template <typename T, bool ADD>
__global__ __launch_bounds__(256) void embedding_sum_kernel(EmbedSums p, EmbedRest rest, int groups, int slabs, const T* add, T* dtable) {
    constexpr int kAhead = 8;
    const int length = *p.length, lane = lane_id(), group = blockIdx.x;
    if (group >= groups * slabs) {
        if (rest.stream) rest_rows<true>(p, rest, group - groups * slabs, length, ADD ? add : (const T*)nullptr, dtable);
        else rest_rows<false>(p, rest, group - groups * slabs, length, ADD ? add : (const T*)nullptr, dtable);
        return;
    }
    const int at = group / slabs, slab = group - at * slabs;   // (a row's slabs side by side: it is read in one go)
    const int64_t b = (int64_t)at * 4 + wave_id(), first = b * p.block;
    if (first >= length) return;
    const int n = (int)min((int64_t)p.block, length - first);
    const int2 item = lane < n ? p.sorted[first + lane] : make_int2(-1, 0);
    const int before = to_sgpr(first > 0 ? p.sorted[first - 1].x : -1), behind = to_sgpr(first + n < length ? p.sorted[first + n].x : -1);
    const int col = slab * 512 + lane * 8;
    const bool mine = col < p.H;
    // bit i: token i is its row's last
    const int below = __shfl_down(item.x, 1, 64);   // (with every lane taking part)
    const uint64_t ends = __ballot(lane < n && (lane < n - 1 ? below : behind) != item.x);
    Row8 sum{};
    bool head = __builtin_amdgcn_readlane(item.x, 0) == before;   // the run that is summed began in an earlier block
    for (int i0 = 0; i0 < n; i0 += kAhead) {
        v4i r[kAhead];   // (as they are in memory)
        Row8 a[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            r[i] = v4i{0, 0, 0, 0};
            a[i] = Row8{};
            if (i0 + i < n && mine) r[i] = *(const v4i*)(p.dout + (size_t)__builtin_amdgcn_readlane(item.y, min(i0 + i, 63)) * p.H + col);
            if (ADD && i0 + i < n && mine && (ends >> (i0 + i) & 1))
                a[i] = load8(add + (size_t)__builtin_amdgcn_readlane(item.x, min(i0 + i, 63)) * p.H + col);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (i0 + i >= n) break;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sum.v[2 * j] += __uint_as_float((uint32_t)r[i][j] << 16);
                sum.v[2 * j + 1] += __uint_as_float((uint32_t)r[i][j] & 0xffff0000u);
            }
            const bool last = i0 + i == n - 1, end = ends >> (i0 + i) & 1;
            if (!end && !last) continue;
            if (head || !end) {
                if (mine) store8(p.partial + ((size_t)b * 2 + (head ? 0 : 1)) * p.H + col, sum);
            } else if (mine) {
                write_row(p, dtable, __builtin_amdgcn_readlane(item.x, i0 + i), col, ADD, a[i], sum);
            }
            head = false;
            sum = Row8{};
        }
    }
}

// Rows whose tokens are spread over several blocks: the wave of the block in which they begin adds the partial sums in order; of more blocks than it
// looks ahead the workgroup's waves a run each, and then theirs in order. (A workgroup for each block, which searched for the row's end one
// place at a time: 21880 tokens of 1795 rows, H = 2184, 22.4 us, so 8.8.)
constexpr int kJoinBlocks = 16;   // blocks behind its own that a wave looks at
template <typename T>
__global__ __launch_bounds__(256) void embedding_join_kernel(EmbedSums p, const T* add, T* dtable) {
    __shared__ float part[4][64][9];
    __shared__ int more[4];   // blocks of the waves' rows that are left to the workgroup
    const int length = *p.length, lane = lane_id(), w = wave_id();
    const int64_t b = (int64_t)blockIdx.x * 4 + w, end = (b + 1) * p.block;   // the next block's first token
    // lane l: the row of block b + 1 + l's first token; the last two: of the last tokens of block b and the one in front of it
    const int64_t place = lane < kJoinBlocks ? end + (int64_t)lane * p.block : lane == 62 ? end - 1 : lane == 63 ? b * p.block - 1 : -1;
    const int key = place >= 0 && place < length ? p.sorted[place].x : -1;
    const int row = __builtin_amdgcn_readlane(key, 0);
    const bool begins = row >= 0 && __builtin_amdgcn_readlane(key, 62) == row && __builtin_amdgcn_readlane(key, 63) != row;
    const int behind = __ffsll((unsigned long long)~__ballot(lane < kJoinBlocks && key == row)) - 1;   // blocks that begin with the row, if few
    const int col = blockIdx.y * 512 + lane * 8;
    const bool mine = col < p.H;
    // partial sums of blocks first + [from, to), eight at a time
    auto gather = [&](int64_t first, int from, int to, Row8& sum) __attribute__((always_inline)) {
        for (int i = from; i < to; i += 8) {
            Row8 r[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                r[k] = Row8{};
                if (i + k < to) r[k] = load8(p.partial + ((size_t)(first + i + k) * 2 + (i + k == 0 ? 1 : 0)) * p.H + col);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int j = 0; j < 8; ++j) sum.v[j] += r[k].v[j];
        }
    };
    int left = 0;
    if (begins && behind < kJoinBlocks) {
        if (mine) {
            const Row8 a = add ? load8(add + (size_t)row * p.H + col) : Row8{};
            Row8 sum{};
            gather(b, 0, behind + 1, sum);
            write_row(p, dtable, row, col, add != nullptr, a, sum);
        }
    } else if (begins) {
        const int64_t blocks = ((int64_t)length + p.block - 1) / p.block;
        int64_t lo = b + kJoinBlocks, hi = blocks;   // block lo begins with the row; block hi does not, or is none
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) / 2;
            if (p.sorted[mid * p.block].x == row) lo = mid;
            else hi = mid;
        }
        left = (int)(hi - b);
    }
    if (lane == 0) more[w] = left;
    __syncthreads();
    for (int v = 0; v < 4; ++v) {
        const int64_t count = more[v], first = (int64_t)blockIdx.x * 4 + v;   // of blocks first, first + 1, ..
        if (count == 0) continue;
        Row8 sum{};
        if (mine) gather(first, (int)(count * w / 4), (int)(count * (w + 1) / 4), sum);
#pragma unroll
        for (int j = 0; j < 8; ++j) part[w][lane][j] = sum.v[j];
        __syncthreads();
        if (w == 0 && mine) {
            const int here = p.sorted[(first + 1) * p.block].x;
#pragma unroll
            for (int u = 1; u < 4; ++u)
#pragma unroll
                for (int j = 0; j < 8; ++j) sum.v[j] += part[u][lane][j];
            write_row(p, dtable, here, col, add != nullptr, add ? load8(add + (size_t)here * p.H + col) : Row8{}, sum);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------------ host
static int embed_check(int T, int V, int H) {
    // (2^38 elements of rows or of the table: workgroups of every launch below 2^24)
    if (T <= 0 || V <= 0 || H <= 0 || (H % 8) != 0 || T >= (1 << 24) || V >= (1 << 30) || H > (1 << 21) || (long long)T * H >= (1ll << 38) ||
        (long long)V * H >= (1ll << 38))
        return HK_ERR_BAD_SHAPE;
    return HK_OK;
}
static size_t embed_up(size_t n) { return (n + 255) / 256 * 256; }

// Tokens of a block of the sums: fewer where there are few, so that the chip has waves enough.
static int embed_block(long long T, int H) {
    const long long waves = T * ((H + 511) / 512);
    return waves >= 64 * 4096 ? 64 : waves >= 32 * 4096 ? 32 : waves >= 16 * 4096 ? 16 : 8;
}
struct EmbedPlan {
    int passes, bits, chunks, block;
    size_t counts, a, b, partial, bytes;   // offsets; the list's length stands in front
    EmbedPlan(int T, int V, int H) {
        int all = 1;
        while (all < 30 && (1ll << all) < V) ++all;
        passes = (all + kMaxDigitBits - 1) / kMaxDigitBits;
        bits = (all + passes - 1) / passes;
        chunks = (T + kSortChunk - 1) / kSortChunk;
        block = embed_block(T, H);
        counts = 256;
        a = counts + embed_up((size_t)passes * chunks * sizeof(int) << bits);
        b = a + embed_up((size_t)T * sizeof(int2));
        partial = b + embed_up((size_t)T * sizeof(int2));
        // two partial sums a block; fewer tokens may have more blocks: at most those of the largest number that blocks of 8, 16 or 32 are taken for
        size_t blocks = (T + block - 1) / block;
        const long long slabs = (H + 511) / 512;
        for (int small = 8; small < block; small *= 2) blocks = std::max(blocks, (size_t)((2 * 4096 * small + slabs - 1) / slabs / small + 1));
        bytes = partial + embed_up(blocks * 2 * H * sizeof(float));
    }
};

// Loads of a wave: a row in as few waves as hold it with eight each, evenly (2880 columns: one of six; 7168: two of seven); in waves of two
// where that gives the chip fewer waves than it holds.
template <typename T>
static int launch_embedding(Ids ids, const void* table, void* out, int tokens, int V, int H, float scale, hipStream_t s) {
    const int parts64 = (H / 8 + 63) / 64;
    int waves = (parts64 + 7) / 8, loads = (parts64 + waves - 1) / waves;
    if ((long long)tokens * waves < 4096) loads = std::min(loads, 2);
    waves = (parts64 + loads - 1) / loads;
    // an output of 96 MB or more would push everything else out of the memory-side cache before it is read (us: 32768 tokens of 2880 columns 60 so, with
    // the hint 53; 65536 of 1024 43 / 27)
    const bool stream = 2ll * tokens * H >= (96ll << 20);
    auto launch = [&]<int LOADS>() {
        hipLaunchKernelGGL((stream ? embedding_kernel<T, LOADS, true> : embedding_kernel<T, LOADS, false>),
                           dim3((unsigned)((tokens + 3) / 4), (unsigned)waves), dim3(256), 0, s, ids, (const T*)table, (uint16_t*)out, tokens, V, H,
                           scale);
        return hipGetLastError() == hipSuccess ? HK_OK : HK_ERR_LAUNCH;
    };
    switch (loads) {
        case 1: return launch.template operator()<1>();
        case 2: return launch.template operator()<2>();
        case 3: return launch.template operator()<3>();
        case 4: return launch.template operator()<4>();
        case 5: return launch.template operator()<5>();
        case 6: return launch.template operator()<6>();
        case 7: return launch.template operator()<7>();
        default: return launch.template operator()<8>();
    }
}

template <typename T>
static int launch_embedding_backward(Ids ids, const void* dout, const void* add, void* dtable, int tokens, int V, int H, float scale, uint8_t* ws,
                                     hipStream_t s) {
    const EmbedPlan L(tokens, V, H);
    int* length = (int*)ws;
    int* counts = (int*)(ws + L.counts);
    int2 *a = (int2*)(ws + L.a), *b = (int2*)(ws + L.b);
    // The launches that sort write the first rows, as many as take them about their time, whether these have tokens or not; the launch that sums
    // writes the others, where there are no tokens.
    const int launches = tokens <= kSortAlone ? 1 : 1 + L.passes;
    const size_t row_bytes = (size_t)H * sizeof(T), all_bytes = V * row_bytes;
    const size_t beside = !add ? kSortZeros : tokens > kSortChunk && launches == 1 ? kSortCopiesLong : kSortCopies;   // a launch
    const int blind = add == dtable ? 0 : (int)std::min<size_t>(V, launches * beside / row_bytes);
    const size_t pieces = blind * row_bytes / 16;
    // rows of a workgroup: 128 KB, and less where that would be few workgroups (8000 tokens of 30000 rows of 1024 with `add` 52.2 us, so 46.5)
    const int to = add == dtable ? blind : V;
    const size_t rest_rows = std::max<size_t>(4, std::min<size_t>((128u << 10) / row_bytes, (size_t)(to - blind) / 512));
    const EmbedRest rest{blind, to, (int)std::min<size_t>(kRestRows, rest_rows), all_bytes > (256u << 20)};
    auto part = [&](int launch) {
        Fill f{(v4i*)dtable, (const v4i*)add, pieces * launch / launches, pieces * (launch + 1) / launches, 0, rest.stream};
        f.groups = (int)std::min<size_t>(512, (f.to - f.from + 4 * kSortThreads - 1) / (4 * kSortThreads));
        return f;
    };
    const int2* sorted = a;
    if (tokens <= kSortAlone) {
        const Fill f = part(0);
        auto kern = tokens <= kSortThreads ? embedding_sort_one_kernel<1>
                    : tokens <= kSortChunk ? embedding_sort_one_kernel<kSortIter> : embedding_sort_one_kernel<2 * kSortIter>;
        hipLaunchKernelGGL(kern, dim3(1 + f.groups), dim3(kSortThreads), 0, s, ids, tokens, V, L.passes, L.bits, a, length, f);
    } else {
        const Fill f = part(0);
        hipLaunchKernelGGL(embedding_count_kernel, dim3(L.chunks + f.groups), dim3(kSortThreads), 0, s, ids, tokens, V, L.chunks, Digit{0, L.bits},
                           counts, L.passes, f);
        const int2* in = nullptr;
        for (int p = 0; p < L.passes; ++p) {
            const Fill g = part(1 + p);
            int2* out = p % 2 == 0 ? a : b;
            const size_t row = (size_t)L.chunks << L.bits;
            hipLaunchKernelGGL(embedding_scatter_kernel, dim3(L.chunks + g.groups), dim3(kSortThreads), 0, s, ids, in, tokens, V, L.chunks,
                               Digit{p * L.bits, L.bits}, (const int*)(counts + p * row), p + 1 < L.passes ? counts + (p + 1) * row : nullptr, out,
                               length, g);
            sorted = in = out;
        }
    }
    if (hipGetLastError() != hipSuccess) return HK_ERR_LAUNCH;
    const EmbedSums p{sorted, length, (const uint16_t*)dout, (float*)(ws + L.partial), H, L.block, scale};
    const unsigned blocks = (unsigned)((tokens + L.block - 1) / L.block), slabs = (unsigned)((H + 511) / 512);
    const unsigned groups = (blocks + 3) / 4;
    const unsigned grid = groups * slabs + (unsigned)((rest.to - rest.from + rest.rows - 1) / rest.rows);
    if (add) hipLaunchKernelGGL((embedding_sum_kernel<T, true>), dim3(grid), dim3(256), 0, s, p, rest, (int)groups, (int)slabs, (const T*)add, (T*)dtable);
    else hipLaunchKernelGGL((embedding_sum_kernel<T, false>), dim3(grid), dim3(256), 0, s, p, rest, (int)groups, (int)slabs, (const T*)nullptr, (T*)dtable);
    if (blocks > 1) hipLaunchKernelGGL(embedding_join_kernel<T>, dim3((blocks + 2) / 4, slabs), dim3(256), 0, s, p, (const T*)add, (T*)dtable);
    return hipGetLastError() == hipSuccess ? HK_OK : HK_ERR_LAUNCH;
}

}  // namespace hk

extern "C" int hk_embedding(const void* ids, int id_type, const void* table, int table_type, void* out_bf16, int T, int V, int H, float scale,
                            void* stream) {
    using namespace hk;
    if (!ids || !table || !out_bf16) return HK_ERR_NULL_POINTER;
    if (const int st = embed_check(T, V, H)) return st;
    if ((id_type != 0 && id_type != 1) || (table_type != 0 && table_type != 1)) return HK_ERR_UNSUPPORTED;
    if ((((uintptr_t)table | (uintptr_t)out_bf16) & 15u) || ((uintptr_t)ids & (id_type ? 7u : 3u))) return HK_ERR_BAD_ALIGNMENT;
    const Ids at{ids, id_type};
    return table_type == 0 ? launch_embedding<uint16_t>(at, table, out_bf16, T, V, H, scale, (hipStream_t)stream)
                           : launch_embedding<float>(at, table, out_bf16, T, V, H, scale, (hipStream_t)stream);
}

extern "C" size_t hk_embedding_backward_workspace_bytes(int T, int V, int H) {
    return hk::embed_check(T, V, H) == HK_OK ? hk::EmbedPlan(T, V, H).bytes : 0;
}

extern "C" int hk_embedding_backward(const void* ids, int id_type, const void* dout_bf16, const void* add_or_null, void* dtable, int table_type,
                                     int T, int V, int H, float scale, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace hk;
    if (!ids || !dout_bf16 || !dtable) return HK_ERR_NULL_POINTER;
    if (const int st = embed_check(T, V, H)) return st;
    if ((id_type != 0 && id_type != 1) || (table_type != 0 && table_type != 1)) return HK_ERR_UNSUPPORTED;
    if ((((uintptr_t)dout_bf16 | (uintptr_t)add_or_null | (uintptr_t)dtable | (uintptr_t)workspace) & 15u) || ((uintptr_t)ids & (id_type ? 7u : 3u)))
        return HK_ERR_BAD_ALIGNMENT;
    if (!workspace || workspace_bytes < EmbedPlan(T, V, H).bytes) return HK_ERR_WORKSPACE;
    const Ids at{ids, id_type};
    return table_type == 0 ? launch_embedding_backward<uint16_t>(at, dout_bf16, add_or_null, dtable, T, V, H, scale, (uint8_t*)workspace, (hipStream_t)stream)
                           : launch_embedding_backward<float>(at, dout_bf16, add_or_null, dtable, T, V, H, scale, (uint8_t*)workspace, (hipStream_t)stream);
}
