// Token rows sorted by expert into the grouped GEMM's contiguous layout, and back with the routing weights applied; both with gradients.
//
// Forward there: a stable counting sort of the n = tokens * k (token, choice) pairs.  Expert e's rows start on a multiple of the
// alignment behind the padded rows of the experts before it, its pairs in their order; the buffer has the rows that the host
// can bound without knowing the routing (sorted_rows), rows without a pair are zero, and nothing comes back to the host.
//   pass A   every warp counts its run of pairs per expert: __match_any_sync finds the lanes of one expert, one of them counts them
//   scan     over a block's warps per expert, over blocks, over experts (padded sizes)
//   pass B   every warp walks its run again and hands out rows from its counters
// No atomics: the order does not depend on timing.
// Up to kOneKernelPairs pairs every block of a single kernel works the whole plan out for itself (a few thousand cycles, less than a
// launch) and then takes its share of the buffer's rows; above, a kernel counts chunks of pairs, one hands out rows and one moves the
// rows, each launched while its predecessor drains.  All of it is bound by the bytes of the buffer that is written.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "host_common.hpp"
#include "launchers.hpp"
#include "ptx.cuh"

namespace nvfp4 {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr uint32_t kAll = 0xffffffffu;
constexpr int kMaxExperts = 1024;                    // two per thread in the scans; 64 KB of counters
// One kernel / three, rows of 8 KB, groups padded to 32: 1024 pairs 15.0 us either way, 1600 17.7 / 16.2, 2048 20.0 / 16.8, 4096 29.9 / 24.3.
constexpr int64_t kOneKernelPairs = 1024;

// Shared memory of a block that plans, in words: per-warp counters, then per expert first row, rows, first sorted pair.
__host__ __device__ constexpr size_t plan_words(int experts) { return static_cast<size_t>(experts) * (kWarps + 3) + 1 + 2 * kWarps; }

struct Plan {
    uint32_t* table;       // [kWarps][experts] pairs of an expert in a warp's run, then: in lower warps' runs
    uint32_t* start;       // [experts + 1] first row of the expert's group; last: end of all groups
    uint32_t* count;       // [experts] rows with a pair
    uint32_t* first;       // [experts] pairs of lower experts
    uint32_t* scratch;     // [2 * kWarps]
    __device__ Plan(uint32_t* smem, int experts)
        : table(smem), start(table + kWarps * experts), count(start + experts + 1), first(count + experts), scratch(first + experts)
    {
    }
};

// The lanes' experts for pairs p0 + lane, -1 for pairs behind `hi` and ids out of range.
__device__ __forceinline__ int expert_of(const int64_t* __restrict__ ids, int64_t p, int64_t hi, int experts)
{
    if (p >= hi) return -1;
    const int64_t e = ids[p];
    return e >= 0 && e < experts ? static_cast<int>(e) : -1;
}

// A warp's run of the pairs [lo, hi) that the block handles, in whole groups of 32.
__device__ __forceinline__ void my_run(int64_t lo, int64_t hi, int64_t& from, int64_t& to)
{
    const int64_t groups = (hi - lo + 31) / 32, each = (groups + kWarps - 1) / kWarps, warp = threadIdx.x >> 5;
    from = min(lo + warp * each * 32, hi);
    to = min(from + each * 32, hi);
}

__device__ __forceinline__ void clear_table(const Plan& s, int experts)
{
    for (int i = threadIdx.x; i < kWarps * experts; i += kThreads) s.table[i] = 0;
    __syncthreads();
}

// Pass A over [lo, hi); afterwards table holds, per warp, what lower warps have of an expert, and total(e) is called with the block's sum.
template <typename Total>
__device__ __forceinline__ void count_pairs(const int64_t* __restrict__ ids, int64_t lo, int64_t hi, int experts, const Plan& s, Total&& total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t from, to;
    my_run(lo, hi, from, to);
    for (int64_t p0 = from; p0 < to; p0 += 32) {
        const int e = expert_of(ids, p0 + lane, to, experts);
        const unsigned same = __match_any_sync(kAll, e);
        if (e >= 0 && lane == __ffs(same) - 1) s.table[warp * experts + e] += __popc(same);
        __syncwarp();
    }
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += kThreads) {
        uint32_t sum = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const uint32_t c = s.table[w * experts + e];
            s.table[w * experts + e] = sum;
            sum += c;
        }
        total(e, sum);
    }
    __syncthreads();
}

// Pass B: row(e, rank) for every pair of [lo, hi) in its order, rank among the block's pairs of expert e; row(-1, 0) for a pair without.
template <typename Row>
__device__ __forceinline__ void hand_out(const int64_t* __restrict__ ids, int64_t lo, int64_t hi, int experts, const Plan& s, Row&& row)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t from, to;
    my_run(lo, hi, from, to);
    for (int64_t p0 = from; p0 < to; p0 += 32) {
        const int64_t p = p0 + lane;
        const int e = expert_of(ids, p, to, experts);
        const unsigned same = __match_any_sync(kAll, e);
        const int leader = __ffs(same) - 1;
        uint32_t base = 0;
        if (e >= 0 && lane == leader) {
            base = s.table[warp * experts + e];
            s.table[warp * experts + e] = base + __popc(same);
        }
        base = __shfl_sync(kAll, base, leader);
        if (p < to) row(p, e, base + __popc(same & ((1u << lane) - 1u)));
        __syncwarp();
    }
}

// start and first from count, by all threads of the block.
__device__ __forceinline__ void scan_experts(int experts, uint32_t alignment, const Plan& s)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e0 = 2 * threadIdx.x;
    uint32_t c[2], a[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        c[i] = e0 + i < experts ? s.count[e0 + i] : 0u;
        a[i] = (c[i] + alignment - 1) / alignment * alignment;
    }
    uint32_t rows = a[0] + a[1], pairs = c[0] + c[1];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t r = __shfl_up_sync(kAll, rows, d), q = __shfl_up_sync(kAll, pairs, d);
        if (lane >= d) { rows += r; pairs += q; }
    }
    if (lane == 31) { s.scratch[warp] = rows; s.scratch[kWarps + warp] = pairs; }
    __syncthreads();
    uint32_t rows_before = rows - a[0] - a[1], pairs_before = pairs - c[0] - c[1];
    for (int w = 0; w < warp; ++w) { rows_before += s.scratch[w]; pairs_before += s.scratch[kWarps + w]; }
    if (e0 < experts) { s.start[e0] = rows_before; s.first[e0] = pairs_before; }
    if (e0 + 1 < experts) { s.start[e0 + 1] = rows_before + a[0]; s.first[e0 + 1] = pairs_before + c[0]; }
    if (e0 < experts && e0 + 2 >= experts) s.start[experts] = rows_before + a[0] + a[1];
    __syncthreads();
}

// Expert whose group holds a row; `experts` behind the last group.  Empty groups share their start with the next one.
__device__ __forceinline__ int group_of(const uint32_t* start, int experts, uint32_t row)
{
    int lo = 0, hi = experts + 1;                    // start[lo] <= row < start[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (start[mid] <= row) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Rows move as words W of 16, 4 or 2 bytes: the widest that both buffers' starts, strides and the row's length are multiples of.
// A warp's piece of a row: so many words a lane.
template <typename W>
constexpr int kPieceWords = sizeof(W) == 16 ? 4 : sizeof(W) == 4 ? 8 : 16;

template <typename W>
__global__ void __launch_bounds__(kThreads)
sort_one_kernel(const W* __restrict__ x, int64_t ldx, const int64_t* __restrict__ ids, int64_t n, int k, int experts, uint32_t alignment, uint32_t m,
                uint32_t row_words, W* __restrict__ rows, int64_t* __restrict__ place, int32_t* __restrict__ source, int32_t* __restrict__ m_indices)
{
    extern __shared__ uint32_t smem[];
    const Plan s(smem, experts);
    const uint32_t lane = threadIdx.x & 31, pieces = (row_words + 32 * kPieceWords<W> - 1) / (32 * kPieceWords<W>);
    const uint64_t units = static_cast<uint64_t>(m) * pieces, step = static_cast<uint64_t>(gridDim.x) * kWarps;
    const uint64_t mine = static_cast<uint64_t>(threadIdx.x >> 5) * gridDim.x + blockIdx.x;      // consecutive units to different blocks
    uint16_t* order = reinterpret_cast<uint16_t*>(smem + plan_words(experts));      // pairs in the order of the experts
    ptx::grid_dependency_wait();
    clear_table(s, experts);
    count_pairs(ids, 0, n, experts, s, [&](int e, uint32_t sum) { s.count[e] = sum; });
    scan_experts(experts, alignment, s);
    hand_out(ids, 0, n, experts, s, [&](int64_t p, int e, uint32_t rank) {
        if (e >= 0) order[s.first[e] + rank] = static_cast<uint16_t>(p);
        if (blockIdx.x == 0) place[p] = e >= 0 ? static_cast<int64_t>(s.start[e]) + rank : -1;
    });
    __syncthreads();
    for (uint64_t unit = mine; unit < units; unit += step) {
        const uint32_t r = static_cast<uint32_t>(unit / pieces), piece = static_cast<uint32_t>(unit % pieces);
        const int e = group_of(s.start, experts, r);
        const bool live = e < experts && r - s.start[e] < s.count[e];
        const uint32_t pair = live ? order[s.first[e] + (r - s.start[e])] : 0u;
        if (piece == 0 && lane == 0) {
            source[r] = live ? static_cast<int32_t>(pair) : -1;
            m_indices[r] = e < experts ? e : -1;
        }
        const W* from = x + static_cast<int64_t>(pair / k) * ldx;
        W* to = rows + static_cast<int64_t>(r) * row_words;
        W v[kPieceWords<W>];
        const uint32_t c0 = piece * 32 * kPieceWords<W> + lane;
#pragma unroll
        for (int i = 0; i < kPieceWords<W>; ++i) {
            v[i] = W{};
            if (live && c0 + i * 32 < row_words) v[i] = from[c0 + i * 32];
        }
#pragma unroll
        for (int i = 0; i < kPieceWords<W>; ++i)
            if (c0 + i * 32 < row_words) to[c0 + i * 32] = v[i];
    }
}

__global__ void __launch_bounds__(kThreads)
sort_count_kernel(const int64_t* __restrict__ ids, int64_t n, int64_t chunk, int experts, uint32_t* __restrict__ counts)
{
    extern __shared__ uint32_t smem[];
    const Plan s(smem, experts);
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    clear_table(s, experts);
    const int64_t lo = blockIdx.x * chunk, hi = min(lo + chunk, n);
    count_pairs(ids, lo, hi, experts, s, [&](int e, uint32_t sum) { counts[static_cast<int64_t>(blockIdx.x) * experts + e] = sum; });
}

// groups: [experts + 1] first rows, [experts] rows with a pair; written by block 0.
__global__ void __launch_bounds__(kThreads)
sort_place_kernel(const int64_t* __restrict__ ids, int64_t n, int64_t chunk, int experts, uint32_t alignment, const uint32_t* __restrict__ counts,
                  uint32_t* __restrict__ groups, int64_t* __restrict__ place, int32_t* __restrict__ source)
{
    extern __shared__ uint32_t smem[];
    const Plan s(smem, experts);
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    // column sums of the chunks' counts, all of them and those before this block's; the warps' table is free until pass A and
    // takes the partial sums: slice i of the threads adds every slices-th chunk
    const int width = experts < kThreads ? (experts + 31) / 32 * 32 : kThreads, slices = kThreads / width;      // slices <= kWarps
    const int slice = threadIdx.x / width, column = threadIdx.x % width;
    uint32_t all[2] = {0, 0}, before[2] = {0, 0};
    for (int i = 0; i < 2; ++i) {
        const int e = column + i * width;
        if (e >= experts || slice >= slices) continue;
        // eight loads under way (one at a time, 128 chunks of 65536 pairs took 20 us)
        for (unsigned c0 = slice; c0 < gridDim.x; c0 += 8 * slices) {
            uint32_t v[8];
#pragma unroll
            for (unsigned u = 0; u < 8; ++u) {
                const unsigned c = c0 + u * slices;
                v[u] = c < gridDim.x ? counts[static_cast<int64_t>(c) * experts + e] : 0u;
            }
#pragma unroll
            for (unsigned u = 0; u < 8; ++u) {
                all[i] += v[u];
                if (c0 + u * slices < blockIdx.x) before[i] += v[u];
            }
        }
    }
    auto add_up = [&](const uint32_t (&part)[2], auto&& store) {
        for (int i = 0; i < 2; ++i)
            if (column + i * width < experts && slice < slices) s.table[slice * experts + column + i * width] = part[i];
        __syncthreads();
        for (int e = threadIdx.x; e < experts; e += kThreads) {
            uint32_t sum = 0;
            for (int j = 0; j < slices; ++j) sum += s.table[j * experts + e];
            store(e, sum);
        }
        __syncthreads();
    };
    add_up(all, [&](int e, uint32_t sum) { s.count[e] = sum; });
    scan_experts(experts, alignment, s);
    if (blockIdx.x == 0) {
        for (int e = threadIdx.x; e <= experts; e += kThreads) groups[e] = s.start[e];
        for (int e = threadIdx.x; e < experts; e += kThreads) groups[experts + 1 + e] = s.count[e];
    }
    add_up(before, [&](int e, uint32_t sum) { s.first[e] = s.start[e] + sum; });      // from here on: first row of this chunk's pairs
    clear_table(s, experts);
    const int64_t lo = blockIdx.x * chunk, hi = min(lo + chunk, n);
    count_pairs(ids, lo, hi, experts, s, [](int, uint32_t) {});
    hand_out(ids, lo, hi, experts, s, [&](int64_t p, int e, uint32_t rank) {
        const int64_t r = e >= 0 ? static_cast<int64_t>(s.first[e]) + rank : -1;
        place[p] = r;
        if (r >= 0) source[r] = static_cast<int32_t>(p);
    });
}

// Every token's row is read once and written k times (unit: a piece of a token); behind the tokens come the rows eight at a time: the
// ones without a pair are zeroed, and all get their expert.
constexpr uint32_t kRowsPerUnit = 8;
template <typename W>
__global__ void __launch_bounds__(kThreads)
sort_move_kernel(const W* __restrict__ x, int64_t ldx, uint32_t tokens, int k, int experts, uint32_t m, uint32_t row_words,
                 const uint32_t* __restrict__ groups, const int64_t* __restrict__ place, W* __restrict__ rows, int32_t* __restrict__ source,
                 int32_t* __restrict__ m_indices)
{
    const uint32_t lane = threadIdx.x & 31, pieces = (row_words + 32 * kPieceWords<W> - 1) / (32 * kPieceWords<W>);
    const uint64_t token_units = static_cast<uint64_t>(tokens) * pieces, units = token_units + (m + kRowsPerUnit - 1) / kRowsPerUnit;
    ptx::grid_dependency_wait();
    for (uint64_t unit = static_cast<uint64_t>(threadIdx.x >> 5) * gridDim.x + blockIdx.x; unit < units; unit += static_cast<uint64_t>(gridDim.x) * kWarps) {
        if (unit < token_units) {
            const uint32_t t = static_cast<uint32_t>(unit / pieces), c0 = static_cast<uint32_t>(unit % pieces) * 32 * kPieceWords<W> + lane;
            const W* from = x + static_cast<int64_t>(t) * ldx;
            W v[kPieceWords<W>];
#pragma unroll
            for (int i = 0; i < kPieceWords<W>; ++i)
                if (c0 + i * 32 < row_words) v[i] = from[c0 + i * 32];
            for (int j0 = 0; j0 < k; j0 += 32) {
                const int64_t mine = j0 + static_cast<int>(lane) < k ? place[static_cast<int64_t>(t) * k + j0 + lane] : -1;
                const int here = min(32, k - j0);
                for (int j = 0; j < here; ++j) {
                    const int64_t r = __shfl_sync(kAll, mine, j);
                    if (r < 0) continue;
                    W* to = rows + r * row_words;
#pragma unroll
                    for (int i = 0; i < kPieceWords<W>; ++i)
                        if (c0 + i * 32 < row_words) to[c0 + i * 32] = v[i];
                }
            }
            continue;
        }
        const uint32_t r0 = static_cast<uint32_t>(unit - token_units) * kRowsPerUnit;
        bool pad = false;
        if (lane < kRowsPerUnit && r0 + lane < m) {
            const uint32_t r = r0 + lane;
            const int e = group_of(groups, experts, r);
            pad = e >= experts || r - groups[e] >= groups[experts + 1 + e];
            m_indices[r] = e < experts ? e : -1;
            if (pad) source[r] = -1;
        }
        for (unsigned todo = __ballot_sync(kAll, pad); todo != 0; todo &= todo - 1) {
            W* to = rows + static_cast<int64_t>(r0 + __ffs(todo) - 1) * row_words;
            for (uint32_t c = lane; c < row_words; c += 32) to[c] = W{};
        }
    }
}

// ---- back: y[t] = sum_j w[t, j] * rows[place[t, j]] ------------------------------------------------------------------------------------

// What a lane moves at a time: 16 or 4 bytes of elements of T, or one of them, as bits.  (Arrays of the 16-bit types' classes end up in local
// memory.)  Loads are plain here as elsewhere in this file: __ldg, an asm statement, may be moved ahead of the test that guards it.
template <typename T, int kBytes>
struct Pack {
    using Bits = std::conditional_t<kBytes == 16, uint4, std::conditional_t<kBytes == 4, uint32_t, uint16_t>>;
    static constexpr int kN = kBytes / static_cast<int>(sizeof(T)), kSize = kBytes;
    static __device__ __forceinline__ float2 two(uint32_t w)
    {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
        else return __half22float2(*reinterpret_cast<const __half2*>(&w));
    }
    static __device__ __forceinline__ uint32_t one_word(float a, float b)
    {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
            return *reinterpret_cast<const uint32_t*>(&h);
        } else {
            const __half2 h = __floats2half2_rn(a, b);
            return *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    static __device__ __forceinline__ void unpack(const Bits& bits, float (&f)[kN])
    {
        if constexpr (kBytes == 2) {
            f[0] = two(bits).x;
        } else {
            uint32_t w[kBytes / 4];
            if constexpr (kBytes == 16) { w[0] = bits.x; w[1] = bits.y; w[2] = bits.z; w[3] = bits.w; }
            else w[0] = bits;
#pragma unroll
            for (int i = 0; i < kBytes / 4; ++i) {
                if constexpr (sizeof(T) == 4) {
                    f[i] = __uint_as_float(w[i]);
                } else {
                    const float2 v = two(w[i]);
                    f[2 * i] = v.x;
                    f[2 * i + 1] = v.y;
                }
            }
        }
    }
    static __device__ __forceinline__ Bits pack(const float (&f)[kN])
    {
        if constexpr (kBytes == 2) {
            return static_cast<uint16_t>(one_word(f[0], 0.0f));
        } else {
            uint32_t w[kBytes / 4];
#pragma unroll
            for (int i = 0; i < kBytes / 4; ++i) {
                if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(f[i]);
                else w[i] = one_word(f[2 * i], f[2 * i + 1]);
            }
            if constexpr (kBytes == 16) return make_uint4(w[0], w[1], w[2], w[3]);
            else return w[0];
        }
    }
};

// A warp takes a piece of a token, kPer packs a lane; the rows of up to four choices are under way together.  FP32, ascending j.
// The gradient of the sort is the same sum without weights.
template <typename P>
constexpr int kPer = P::kSize == 16 ? 2 : P::kSize == 4 ? 4 : 8;              // packs of a lane: of narrow ones more
constexpr int kFlight = 4;
template <typename P>
__global__ void __launch_bounds__(256, 3)
unsort_kernel(const typename P::Bits* __restrict__ rows, int64_t ld, const int64_t* __restrict__ place, const float* __restrict__ w, uint32_t tokens,
              int k, int64_t m, uint32_t row_packs, typename P::Bits* __restrict__ y)
{
    constexpr int kN = P::kN;
    const uint32_t lane = threadIdx.x & 31, pieces = (row_packs + 32 * kPer<P> - 1) / (32 * kPer<P>);
    const uint64_t units = static_cast<uint64_t>(tokens) * pieces;
    ptx::grid_dependency_wait();
    for (uint64_t unit = static_cast<uint64_t>(threadIdx.x >> 5) * gridDim.x + blockIdx.x; unit < units; unit += static_cast<uint64_t>(gridDim.x) * 8) {
        const uint32_t t = static_cast<uint32_t>(unit / pieces), c0 = static_cast<uint32_t>(unit % pieces) * 32 * kPer<P> + lane;
        float acc[kPer<P>][kN];
#pragma unroll
        for (int i = 0; i < kPer<P>; ++i)
#pragma unroll
            for (int q = 0; q < kN; ++q) acc[i][q] = 0.0f;
        for (int j0 = 0; j0 < k; j0 += 32) {
            int64_t mine = -1;
            float weight = 1.0f;
            if (j0 + static_cast<int>(lane) < k) {
                mine = place[static_cast<int64_t>(t) * k + j0 + lane];
                if (mine >= m) mine = -1;
                if (w != nullptr) weight = w[static_cast<int64_t>(t) * k + j0 + lane];
            }
            const int here = min(32, k - j0);
            for (int j1 = 0; j1 < here; j1 += kFlight) {
                typename P::Bits v[kFlight][kPer<P>];
                bool live[kFlight];
                float wj[kFlight];
#pragma unroll
                for (int u = 0; u < kFlight; ++u) {
                    const int64_t r = __shfl_sync(kAll, mine, (j1 + u) & 31);
                    wj[u] = __shfl_sync(kAll, weight, (j1 + u) & 31);
                    live[u] = j1 + u < here && r >= 0;
                    if (live[u]) {
#pragma unroll
                        for (int i = 0; i < kPer<P>; ++i)
                            if (c0 + i * 32 < row_packs) v[u][i] = rows[r * ld + c0 + i * 32];
                    }
                }
#pragma unroll
                for (int u = 0; u < kFlight; ++u) {
                    if (!live[u]) continue;
#pragma unroll
                    for (int i = 0; i < kPer<P>; ++i) {
                        float f[kN];
                        P::unpack(v[u][i], f);
#pragma unroll
                        for (int q = 0; q < kN; ++q) acc[i][q] = fmaf(wj[u], f[q], acc[i][q]);
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kPer<P>; ++i) {
            if (c0 + i * 32 >= row_packs) continue;
            y[static_cast<int64_t>(t) * row_packs + c0 + i * 32] = P::pack(acc[i]);
        }
    }
}

// The same sum for many tokens with rows of whole 16-byte words: the rows come by bulk copies into a ring in shared memory, whole pieces
// of up to 8 KB a request, and a block has its entire shared memory under way, where the loads of the kernel above come in pieces of 1 KB
// and no faster than registers for them are to be had (8192 tokens x 8 rows of 8 KB: 171 us, 3.5 TB/s).
// A unit is a piece of one token's rows, or `group` whole tokens whose rows are short; a slot of the ring takes a unit's pairs (at most
// 32), `stride` bytes each.  Warp 0 looks up a pair per lane, one unit ahead, leaves the weights and the mask of pairs with a row beside
// the slot and requests the rows; the other warps add them up in FP32 in ascending j, the order of the kernel above: the same bits.
// Every wait is bounded; a block whose wait ran out leaves NaN in what it did not finish, and leaves when its copies in flight have landed,
// within the same bound.
constexpr int kRingWorkers = 16, kRingThreads = 32 * (1 + kRingWorkers), kRingPairs = 32, kRingMaxDepth = 12;
struct RingSlot {
    float w[kRingPairs];
    uint32_t live;                                   // bit p: pair p has a row, whose bytes were requested
};
// units to an SM from which on the ring is taken
constexpr uint32_t kRingLeast = 2;
struct RingShape {
    uint32_t tokens, k, group, units, pieces, row_bytes, stride, depth;
    long long budget = ptx::kWaitBudgetCycles;       // of every wait, in cycles
    bool withhold = false;                           // test of the expired wait: no row is requested
};
template <typename P>
__global__ void __launch_bounds__(kRingThreads, 1)
unsort_ring_kernel(const uint8_t* __restrict__ rows, int64_t ld_bytes, const int64_t* __restrict__ place, const float* __restrict__ w, int64_t m,
                   const RingShape shape, uint4* __restrict__ y)
{
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem = (ptx::smem_u32(smem_raw) + 127u) & ~127u;
    uint8_t* gen = smem_raw + (smem - ptx::smem_u32(smem_raw));
    const uint32_t pairs = shape.group * shape.k, slot_bytes = pairs * shape.stride;
    uint64_t* full = reinterpret_cast<uint64_t*>(gen + static_cast<size_t>(shape.depth) * slot_bytes);
    uint64_t* freed = full + kRingMaxDepth;
    RingSlot* info = reinterpret_cast<RingSlot*>(freed + kRingMaxDepth);
    volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(info + kRingMaxDepth);
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < shape.depth; ++i) { ptx::mbar_init(full + i, 1); ptx::mbar_init(freed + i, kRingWorkers); }
        *abort_flag = 0;
        ptx::fence_mbar_init();
    }
    __syncthreads();
    ptx::grid_dependency_wait();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t slot = 0, phase = 0;
    auto next = [&] { if (++slot == shape.depth) { slot = 0; phase ^= 1; } };
    if (warp == 0) {
        int64_t row = -1;
        float weight = 0.0f;
        auto look_up = [&](uint32_t unit) {
            row = -1;
            if (unit >= shape.units || lane >= pairs) return;
            const uint32_t t0 = unit / shape.pieces * shape.group;
            if (lane >= min(shape.group, shape.tokens - t0) * shape.k) return;
            const int64_t at = static_cast<int64_t>(t0) * shape.k + lane;
            row = place[at];
            if (row >= m) row = -1;
            weight = w != nullptr ? w[at] : 1.0f;
        };
        look_up(blockIdx.x);
        uint32_t loaded = 0;
        bool ok = true;
        for (uint32_t unit = blockIdx.x; unit < shape.units && !shape.withhold; unit += gridDim.x, ++loaded) {
            if (!ptx::all_lanes(ptx::mbar_wait_budget(freed + slot, phase ^ 1, abort_flag, shape.budget))) { *abort_flag = 1; ok = false; break; }
            const uint32_t from = unit % shape.pieces * shape.stride, bytes = min(shape.stride, shape.row_bytes - from);
            const unsigned live = __ballot_sync(kAll, row >= 0);
            if (lane < pairs) info[slot].w[lane] = weight;
            if (lane == 0) info[slot].live = live;
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive_expect_tx(full + slot, __popc(live) * bytes);
            __syncwarp();
            if (row >= 0) ptx::bulk_load(gen + static_cast<size_t>(slot) * slot_bytes + lane * shape.stride, rows + row * ld_bytes + from, bytes, full + slot);
            look_up(unit + gridDim.x);
            next();
        }
        if (!ok || !ptx::all_lanes(*abort_flag == 0)) {
            const long long until = clock64() + shape.budget;
            for (uint32_t n = loaded > shape.depth ? loaded - shape.depth : 0; n < loaded; ++n)
                ptx::mbar_settle(full + n % shape.depth, n / shape.depth & 1u, until);
        }
        return;
    }
    bool ok = true;
    for (uint32_t unit = blockIdx.x; unit < shape.units; unit += gridDim.x) {
        if (ok && !ptx::all_lanes(ptx::mbar_wait_budget(full + slot, phase, abort_flag, shape.budget))) { *abort_flag = 1; ok = false; }
        const uint32_t base = smem + slot * slot_bytes, live = ok ? info[slot].live : 0u;
        const uint32_t t0 = unit / shape.pieces * shape.group, here = min(shape.group, shape.tokens - t0);
        const uint32_t from = unit % shape.pieces * shape.stride, words = min(shape.stride, shape.row_bytes - from) / 16;
        for (uint32_t c = threadIdx.x - 32; c < here * words; c += 32 * kRingWorkers) {
            const uint32_t g = c / words, word = c % words, first = g * shape.k;
            float acc[P::kN];
#pragma unroll
            for (int q = 0; q < P::kN; ++q) acc[q] = ok ? 0.0f : __uint_as_float(0x7fc00000u);
            for (uint32_t j0 = 0; j0 < shape.k; j0 += 8) {
                uint4 v[8];
                const uint32_t mask = (live >> (first + j0)) & ((2u << min(7u, shape.k - 1 - j0)) - 1);
#pragma unroll
                for (uint32_t u = 0; u < 8; ++u)
                    if (mask >> u & 1u) v[u] = ptx::lds128(base + (first + j0 + u) * shape.stride + word * 16);
#pragma unroll
                for (uint32_t u = 0; u < 8; ++u) {
                    if (!(mask >> u & 1u)) continue;
                    const float wj = info[slot].w[first + j0 + u];
                    float f[P::kN];
                    P::unpack(v[u], f);
#pragma unroll
                    for (int q = 0; q < P::kN; ++q) acc[q] = fmaf(wj, f[q], acc[q]);
                }
            }
            y[(static_cast<int64_t>(t0 + g) * shape.row_bytes + from) / 16 + word] = P::pack(acc);
        }
        // the slot's loads are over: what they brought went into the words that were stored
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(freed + slot);
        next();
    }
}
constexpr size_t kRingExtra = 128 + kRingMaxDepth * (2 * sizeof(uint64_t) + sizeof(RingSlot)) + 16, kRingSmem = 232448 - 1024;
// The ring for these rows; depth 0: there is none.
RingShape ring_shape(int64_t tokens, int k, int64_t row_bytes)
{
    RingShape r{static_cast<uint32_t>(tokens), static_cast<uint32_t>(k), 1, 0, 1, static_cast<uint32_t>(row_bytes), static_cast<uint32_t>(row_bytes), 0};
    if (k > kRingPairs || row_bytes % 16 != 0) return r;
    for (r.stride = 8192; r.stride > 1024 && 3 * static_cast<int64_t>(r.stride) * k > static_cast<int64_t>(kRingSmem - kRingExtra); r.stride /= 2) {}
    if (row_bytes <= r.stride) {
        r.stride = static_cast<uint32_t>(row_bytes);
        while ((r.group + 1) * r.k <= kRingPairs && (r.group + 1) * row_bytes <= 8192) ++r.group;
    }
    r.pieces = static_cast<uint32_t>((row_bytes + r.stride - 1) / r.stride);
    const int64_t units = (tokens + r.group - 1) / r.group * r.pieces, depth = static_cast<int64_t>(kRingSmem - kRingExtra) / (static_cast<int64_t>(r.group) * k * r.stride);
    if (units > INT32_MAX) return r;
    r.units = static_cast<uint32_t>(units);
    r.depth = static_cast<uint32_t>(depth > kRingMaxDepth ? kRingMaxDepth : depth);
    return r;
}

// Gradients of that sum: drows[r] = sum of w[t, j] * dy[t] over the pairs that name row r, dw[t, j] = <dy[t], rows[place[t, j]]>.
// The sum takes any order that names rows, not the sort's alone: a part of its tokens, pairs dropped afterwards, one row for several
// pairs.  So a kernel in front makes a list of every row's pairs, in any order: head[r] is one of them, next[p] the one behind p, kNobody
// ends it (8192 x 8 pairs: with the clearing of the heads 4 us of the 214).
// A warp takes a pair: its dot product stays inside the warp, in a fixed order, and four packs a lane of the row and of dy are under way
// at a time in few registers.  The pairs of a token are neighbouring warps', which read dy from L1 behind the first.  (A block to a token,
// eight rows at a time to a thread, took 138 registers and ran at an eighth of the warps: 455 us for 8192 x 8 rows of 8 KB.)  A row that
// this pair alone names is written on the way.
// Behind the pairs: warps for pieces of rows, four rows at a time (forward and backward of 8192 x 8 rows in a graph: 305 us; one row 338, eight
// 306).  Those that nobody names are zeroed; those of several pairs get the sum in ascending pairs, FP32, rounded once: up to 32 pairs from
// the list, more of them looked up among all pairs (every row named eight times: 0.28 ms in place of 0.21; a hundred times: 19 ms).
// drows or dw may be NULL; rows is read for dw alone, head and next for drows.
constexpr int kBackThreads = 256, kBackWarps = kBackThreads / 32;
constexpr uint32_t kNobody = 0xffffffffu, kBackRows = 4;
template <typename P>
constexpr int kBackPer = P::kSize == 16 ? 4 : 8;                              // packs of a lane under way, or of a piece of a row
__global__ void __launch_bounds__(kBackThreads)
list_names_kernel(const int64_t* __restrict__ place, uint32_t pairs, uint32_t m, uint32_t* __restrict__ head, uint32_t* __restrict__ next)
{
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    for (uint64_t p = static_cast<uint64_t>(blockIdx.x) * kBackThreads + threadIdx.x; p < pairs; p += static_cast<uint64_t>(gridDim.x) * kBackThreads) {
        const int64_t r = place[p];
        if (r >= 0 && r < m) next[p] = atomicExch(head + r, static_cast<uint32_t>(p));
    }
}
// The gradient of row r, named by several pairs, in pack c of the lane (all lanes run this together, whether they have a pack or not).
template <typename P>
__device__ __forceinline__ typename P::Bits sum_of_names(const typename P::Bits* __restrict__ dy, int64_t ldy, const int64_t* __restrict__ place,
                                                         const uint32_t* __restrict__ next, uint32_t first, const float* __restrict__ w, uint32_t pairs,
                                                         uint32_t k, int64_t r, uint32_t c, bool there)
{
    constexpr int kN = P::kN;
    const uint32_t lane = threadIdx.x & 31;
    float acc[kN];
#pragma unroll
    for (int q = 0; q < kN; ++q) acc[q] = 0.0f;
    auto add = [&](uint32_t p) {
        if (!there) return;
        const float weight = w != nullptr ? w[p] : 1.0f;
        float f[kN];
        P::unpack(dy[static_cast<int64_t>(p / k) * ldy + c], f);
#pragma unroll
        for (int q = 0; q < kN; ++q) acc[q] = fmaf(weight, f[q], acc[q]);
    };
    uint32_t mine = kNobody, count = 0, at = first;                           // lane i holds the i-th of the list
    for (; at != kNobody && count < 32; ++count) {
        if (lane == count) mine = at;
        at = next[at];
    }
    if (at == kNobody) {
        uint32_t rank = 0;
        for (uint32_t i = 0; i < count; ++i) rank += __shfl_sync(kAll, mine, i) < mine;
        for (uint32_t i = 0; i < count; ++i) add(__shfl_sync(kAll, mine, __ffs(__ballot_sync(kAll, lane < count && rank == i)) - 1));
    } else {
        for (uint32_t p0 = 0; p0 < pairs; p0 += 32)
            for (unsigned here = __ballot_sync(kAll, p0 + lane < pairs && place[p0 + lane] == r); here != 0; here &= here - 1) add(p0 + __ffs(here) - 1);
    }
    return P::pack(acc);
}
template <typename P>
__global__ void __launch_bounds__(kBackThreads, 4)
unsort_backward_kernel(const typename P::Bits* __restrict__ dy, int64_t ldy, const typename P::Bits* __restrict__ rows, int64_t ld,
                       const int64_t* __restrict__ place, const uint32_t* __restrict__ head, const uint32_t* __restrict__ next, const float* __restrict__ w,
                       uint32_t pairs, uint32_t k, uint32_t m, uint32_t row_packs, typename P::Bits* __restrict__ drows, float* __restrict__ dw)
{
    using Bits = typename P::Bits;
    constexpr int kN = P::kN, kPer = kBackPer<P>;
    const uint32_t lane = threadIdx.x & 31, pieces = (row_packs + 32 * kPer - 1) / (32 * kPer);
    const uint64_t units = static_cast<uint64_t>(pairs) + (drows != nullptr ? static_cast<uint64_t>((m + kBackRows - 1) / kBackRows) * pieces : 0);
    ptx::grid_dependency_wait();
    for (uint64_t unit = static_cast<uint64_t>(blockIdx.x) * kBackWarps + (threadIdx.x >> 5); unit < units; unit += static_cast<uint64_t>(gridDim.x) * kBackWarps) {
        if (unit >= pairs) {
            const uint64_t u = unit - pairs;
            const uint32_t r0 = static_cast<uint32_t>(u / pieces) * kBackRows, c0 = static_cast<uint32_t>(u % pieces) * 32 * kPer + lane;
            uint32_t first = kNobody;
            bool mine = false;                                                // the lane's row has no pair or several
            if (lane < kBackRows && r0 + lane < m) {
                first = head[r0 + lane];
                mine = first == kNobody || next[first] != kNobody;
            }
            for (unsigned todo = __ballot_sync(kAll, mine); todo != 0; todo &= todo - 1) {
                const int i = __ffs(todo) - 1;
                const uint32_t r = r0 + i, of_row = __shfl_sync(kAll, first, i);
                Bits* to = drows + static_cast<int64_t>(r) * row_packs;
                if (of_row == kNobody) {
#pragma unroll
                    for (int j = 0; j < kPer; ++j)
                        if (c0 + j * 32 < row_packs) to[c0 + j * 32] = Bits{};
                    continue;
                }
#pragma unroll 1
                for (uint32_t c = c0; c - lane < row_packs && c < c0 + 32 * kPer; c += 32) {
                    const Bits sum = sum_of_names<P>(dy, ldy, place, next, of_row, w, pairs, k, r, c, c < row_packs);
                    if (c < row_packs) to[c] = sum;
                }
            }
            continue;
        }
        const uint32_t p = static_cast<uint32_t>(unit);
        const int64_t r = place[p];
        if (r < 0 || r >= m) {
            if (dw != nullptr && lane == 0) dw[p] = 0.0f;
            continue;
        }
        const bool write = drows != nullptr && head[r] == p && next[p] == kNobody;
        if (dw == nullptr && !write) continue;
        const float weight = w != nullptr ? w[p] : 1.0f;
        const Bits* from = dy + static_cast<int64_t>(p / k) * ldy;
        const Bits* row = rows + r * ld;
        Bits* to = drows + r * row_packs;
        float dot = 0.0f;
        for (uint32_t c0 = lane; c0 < row_packs; c0 += 32 * kPer) {
            Bits g[kPer], v[kPer];
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (c0 + i * 32 < row_packs) g[i] = from[c0 + i * 32];
            if (dw != nullptr) {
#pragma unroll
                for (int i = 0; i < kPer; ++i)
                    if (c0 + i * 32 < row_packs) v[i] = row[c0 + i * 32];
            }
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                if (c0 + i * 32 >= row_packs) continue;
                float gf[kN], f[kN];
                P::unpack(g[i], gf);
                if (dw != nullptr) {
                    P::unpack(v[i], f);
#pragma unroll
                    for (int q = 0; q < kN; ++q) dot = fmaf(gf[q], f[q], dot);
                }
                if (write) {
#pragma unroll
                    for (int q = 0; q < kN; ++q) f[q] = weight * gf[q];
                    to[c0 + i * 32] = P::pack(f);
                }
            }
        }
        if (dw == nullptr) continue;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(kAll, dot, d);
        if (lane == 0) dw[p] = dot;
    }
}

// Calls f(Pack<type, bytes>*) for a type code and the widest pack that everything in `bits` (addresses, strides and lengths in bytes) is a
// multiple of.
template <typename F>
int with_pack(int dtype, uintptr_t bits, F&& f)
{
    auto packs = [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        if ((bits & 15u) == 0) return f(static_cast<Pack<T, 16>*>(nullptr));
        if constexpr (sizeof(T) == 2)
            if ((bits & 3u) != 0) return f(static_cast<Pack<T, 2>*>(nullptr));
        return f(static_cast<Pack<T, 4>*>(nullptr));
    };
    switch (dtype) {
        case NVFP4_DTYPE_BF16: return packs(static_cast<__nv_bfloat16*>(nullptr));
        case NVFP4_DTYPE_F16: return packs(static_cast<__half*>(nullptr));
        default: return packs(static_cast<float*>(nullptr));
    }
}

size_t elem_bytes(int dtype) { return dtype == NVFP4_DTYPE_F32 ? 4 : 2; }

// Blocks of `warps` warps for so many units, at most `per_sm` to an SM.
unsigned blocks_for(uint64_t units, int warps, int num_sms, int per_sm)
{
    const uint64_t most = static_cast<uint64_t>(num_sms) * per_sm, want = (units + warps - 1) / warps;
    // few units: one warp's worth to a block rather than one block's worth to an SM
    const uint64_t spread = units < static_cast<uint64_t>(num_sms) ? units : (want < static_cast<uint64_t>(num_sms) ? num_sms : want);
    return static_cast<unsigned>(spread < most ? spread : most);
}

template <typename W>
int sort_with(const void* x, int64_t ldx_bytes, int64_t tokens, int k, int64_t row_bytes, const int64_t* ids, int experts, int alignment, int64_t m,
              void* rows, int64_t* place, int32_t* source, int32_t* m_indices, int num_sms, cudaStream_t stream)
{
    const int64_t n = tokens * k, ldx = ldx_bytes / static_cast<int64_t>(sizeof(W));
    const uint32_t row_words = static_cast<uint32_t>(row_bytes / static_cast<int64_t>(sizeof(W)));
    const uint64_t pieces = (row_words + 32 * kPieceWords<W> - 1) / (32 * kPieceWords<W>);
    const size_t plan_bytes = plan_words(experts) * sizeof(uint32_t);
    int dev = 0;
    NVFP4_CUDA_CHECK(cudaGetDevice(&dev));
    constexpr size_t kMostSmem = plan_words(kMaxExperts) * sizeof(uint32_t) + kOneKernelPairs * sizeof(uint16_t);
    static bool attr_set[host::kMaxDevices] = {};
    if (!attr_set[dev]) {
        NVFP4_CUDA_CHECK(cudaFuncSetAttribute(sort_one_kernel<W>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMostSmem)));
        NVFP4_CUDA_CHECK(cudaFuncSetAttribute(sort_count_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMostSmem)));
        NVFP4_CUDA_CHECK(cudaFuncSetAttribute(sort_place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMostSmem)));
        attr_set[dev] = true;
    }
    if (n <= kOneKernelPairs)
        return host::launch_kernel(sort_one_kernel<W>, dim3(blocks_for(static_cast<uint64_t>(m) * pieces, kWarps, num_sms, 2)), dim3(kThreads),
                                   plan_bytes + static_cast<size_t>(n) * sizeof(uint16_t), stream, true, static_cast<const W*>(x), ldx, ids, n, k,
                                   experts, static_cast<uint32_t>(alignment), static_cast<uint32_t>(m), row_words, static_cast<W*>(rows), place, source,
                                   m_indices);
    int64_t chunk = (n + num_sms - 1) / num_sms;
    chunk = (chunk + kThreads - 1) / kThreads * kThreads;
    const unsigned blocks = static_cast<unsigned>((n + chunk - 1) / chunk);
    cudaMemPool_t pool;
    if (int rc = host::workspace_pool(dev, &pool)) return rc;
    uint32_t* counts = nullptr;
    const size_t count_words = static_cast<size_t>(blocks) * experts;
    NVFP4_CUDA_CHECK(cudaMallocFromPoolAsync(reinterpret_cast<void**>(&counts), (count_words + 2 * experts + 1) * sizeof(uint32_t), pool, stream));
    uint32_t* groups = counts + count_words;
    int rc = host::launch_kernel(sort_count_kernel, dim3(blocks), dim3(kThreads), plan_bytes, stream, true, ids, n, chunk, experts, counts);
    if (rc == NVFP4_OK)
        rc = host::launch_kernel(sort_place_kernel, dim3(blocks), dim3(kThreads), plan_bytes, stream, true, ids, n, chunk, experts,
                                 static_cast<uint32_t>(alignment), counts, groups, place, source);
    if (rc == NVFP4_OK)
        rc = host::launch_kernel(sort_move_kernel<W>,
                                 dim3(blocks_for(static_cast<uint64_t>(tokens) * pieces + (m + kRowsPerUnit - 1) / kRowsPerUnit, kWarps, num_sms, 4)),
                                 dim3(kThreads), 0, stream, true, static_cast<const W*>(x), ldx, static_cast<uint32_t>(tokens), k, experts,
                                 static_cast<uint32_t>(m), row_words, groups, place, static_cast<W*>(rows), source, m_indices);
    cudaFreeAsync(counts, stream);
    return rc;
}

}  // namespace

int launch_sort_tokens(const void* x, int64_t ldx_bytes, int64_t tokens, int k, int64_t row_bytes, const int64_t* ids, int experts, int alignment,
                       int64_t m, void* rows, int64_t* place, int32_t* source, int32_t* m_indices, int num_sms, cudaStream_t stream)
{
    const uintptr_t bits = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(rows) | static_cast<uintptr_t>(ldx_bytes | row_bytes);
    auto with = (bits & 15u) == 0 ? sort_with<uint4> : (bits & 3u) == 0 ? sort_with<uint32_t> : sort_with<uint16_t>;
    return with(x, ldx_bytes, tokens, k, row_bytes, ids, experts, alignment, m, rows, place, source, m_indices, num_sms, stream);
}

int launch_unsort_tokens(const void* rows, int64_t ld, int dtype, int64_t m, const int64_t* place, const float* w, int64_t tokens, int k, int hidden,
                         void* y, int num_sms, cudaStream_t stream, int64_t budget)
{
    const size_t size = elem_bytes(dtype);
    const uintptr_t bits = reinterpret_cast<uintptr_t>(rows) | reinterpret_cast<uintptr_t>(y) | static_cast<uintptr_t>(ld * size) | hidden * size;
    return with_pack(dtype, bits, [&](auto* type) {
        using P = std::remove_pointer_t<decltype(type)>;
        using Bits = typename P::Bits;
        constexpr int kN = P::kN;
        if constexpr (P::kSize == 16) {
            RingShape shape = ring_shape(tokens, k, static_cast<int64_t>(hidden * size));
            if (budget > 0) { shape.budget = budget; shape.withhold = true; }
            if (shape.depth >= 2 && shape.units >= kRingLeast * static_cast<uint32_t>(num_sms)) {
                static bool attr_set[host::kMaxDevices] = {};
                int dev = 0;
                NVFP4_CUDA_CHECK(cudaGetDevice(&dev));
                if (!attr_set[dev]) {
                    NVFP4_CUDA_CHECK(cudaFuncSetAttribute(unsort_ring_kernel<P>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kRingSmem)));
                    attr_set[dev] = true;
                }
                return host::launch_kernel(unsort_ring_kernel<P>, dim3(static_cast<unsigned>(num_sms)), dim3(kRingThreads),
                                           static_cast<size_t>(shape.depth) * shape.group * shape.k * shape.stride + kRingExtra, stream, true,
                                           static_cast<const uint8_t*>(rows), static_cast<int64_t>(ld * size), place, w, m, shape, static_cast<uint4*>(y));
            }
        }
        const uint32_t packs = static_cast<uint32_t>(hidden / kN);
        const uint64_t units = static_cast<uint64_t>(tokens) * ((packs + 32 * kPer<P> - 1) / (32 * kPer<P>));
        return host::launch_kernel(unsort_kernel<P>, dim3(blocks_for(units, 8, num_sms, 8)), dim3(256), 0, stream, true,
                                   static_cast<const Bits*>(rows), ld / kN, place, w, static_cast<uint32_t>(tokens), k, m, packs,
                                   static_cast<Bits*>(y));
    });
}

int launch_unsort_tokens_backward(const void* dy, int64_t ldy, const void* rows, int64_t ld, int dtype, int64_t m, const int64_t* place,
                                  const float* w, int64_t tokens, int k, int hidden, void* drows, float* dw, int num_sms, cudaStream_t stream)
{
    const size_t size = elem_bytes(dtype);
    const uintptr_t bits = reinterpret_cast<uintptr_t>(dy) | reinterpret_cast<uintptr_t>(rows) | reinterpret_cast<uintptr_t>(drows) |
                           static_cast<uintptr_t>(ldy * size) | static_cast<uintptr_t>(ld * size) | hidden * size;
    const uint64_t pairs = static_cast<uint64_t>(tokens) * k, units = pairs + (drows != nullptr ? m : 0);       // (sizes the grid; the kernel has units of its own)
    uint32_t *head = nullptr, *next = nullptr;
    if (drows != nullptr && m > 0) {
        int dev = 0;
        NVFP4_CUDA_CHECK(cudaGetDevice(&dev));
        cudaMemPool_t pool;
        if (int rc = host::workspace_pool(dev, &pool)) return rc;
        NVFP4_CUDA_CHECK(cudaMallocFromPoolAsync(reinterpret_cast<void**>(&head), (static_cast<size_t>(m) + pairs) * sizeof(uint32_t), pool, stream));
        next = head + m;
        int rc = NVFP4_OK;
        if (cudaError_t err = cudaMemsetAsync(head, 0xff, static_cast<size_t>(m) * sizeof(uint32_t), stream); err != cudaSuccess)
            rc = host::fail(NVFP4_E_CUDA, "clearing the lists of pairs failed: %s", cudaGetErrorString(err));
        if (rc == NVFP4_OK && pairs > 0)
            rc = host::launch_kernel(list_names_kernel, dim3(blocks_for((pairs + 31) / 32, kBackWarps, num_sms, 8)), dim3(kBackThreads), 0, stream, true, place,
                                     static_cast<uint32_t>(pairs), static_cast<uint32_t>(m), head, next);
        if (rc != NVFP4_OK) {
            cudaFreeAsync(head, stream);
            return rc;
        }
    }
    const int rc = with_pack(dtype, bits, [&](auto* type) {
        using P = std::remove_pointer_t<decltype(type)>;
        using Bits = typename P::Bits;
        constexpr int kN = P::kN;
        return host::launch_kernel(unsort_backward_kernel<P>, dim3(blocks_for(units, kBackWarps, num_sms, 8)), dim3(kBackThreads), 0, stream, true,
                                   static_cast<const Bits*>(dy), ldy / kN, static_cast<const Bits*>(rows), ld / kN, place, head, next, w,
                                   static_cast<uint32_t>(pairs), static_cast<uint32_t>(k), static_cast<uint32_t>(m), static_cast<uint32_t>(hidden / kN),
                                   static_cast<Bits*>(drows), dw);
    });
    if (head != nullptr) cudaFreeAsync(head, stream);
    return rc;
}

}  // namespace nvfp4
