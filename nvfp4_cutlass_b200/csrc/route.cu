// Top-k routing: the k experts of every token and their weights from the router's logits, and the gradient of the logits.
//
// One warp takes one token and keeps its row of logits in registers, value r of lane l at index 32 r + l: a load of the warp is one run
// of the row, whatever its alignment.  Logits are compared as integer keys whose order is that of the floats (NaN above +inf, -0
// equal to +0), so that the largest of the warp and the lowest index that holds it are one warp reduction each; k rounds of that, and lane j
// keeps the j-th choice.  Both score functions grow with the logit: the choice needs no score, and a tie between logits is a tie
// between scores.  A logit of -inf says that the expert is not to be had: it is never chosen, and a row with fewer than k others
// ends in ids of -1 with weight 0.  Scores, sums and weights are FP32 throughout.
// Bound by latency: the k rounds of a token are a chain of vote, compare and rescan, and the issue slots are busy 55 % of the time (16384 x 128
// BF16, 8 choices: 520 instructions a token, 10.4 us in a graph for the bytes of 0.9; backward 530, 10.3 us).  A decode step: by the launch.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "host_common.hpp"
#include "launchers.hpp"
#include "ptx.cuh"

namespace nvfp4 {
namespace {

constexpr int kRouteWarps = 8;
constexpr uint32_t kAll = 0xffffffffu;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_float(float v, float& out) { out = v; }
__device__ __forceinline__ void from_float(float v, __nv_bfloat16& out) { out = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_float(float v, __half& out) { out = __float2half_rn(v); }

// Keys in the order of the floats.  0 stands for "taken already" and for places behind the row, below the key of -inf.
__device__ __forceinline__ uint32_t key_of(float v)
{
    const uint32_t bits = __float_as_uint(v + 0.0f);                          // -0 becomes +0
    if ((bits & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key)
{
    if (key == 0xffffffffu) return __uint_as_float(0x7fc00000u);
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
constexpr uint32_t kMaskedKey = 0x007fffffu;                                  // of -inf

// A 16-bit logit's rank in 21 bits (its place among the type's 2^16 values, masked ones and NaN as above) over the index, the lowest on top.
// FP32 keys of BF16 values differ in their upper 16 bits alone; FP16 values take 10 digits and, subnormal ones included, 6 bits of
// exponent in FP32 (2^-24 to 2^15), so that bits 13 to 31 tell them apart.
constexpr uint32_t kIndexMask = 1023u;
template <typename T>
__device__ __forceinline__ uint32_t packed_key(uint32_t key, uint32_t index)
{
    constexpr uint32_t kShift = std::is_same<T, __nv_bfloat16>::value ? 16 : 13;
    return (key >> kShift << 10) + (kIndexMask - index);
}

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kAll, v, d);
    return v;
}

// Weight of lane's choice `l` (live lanes; 0 elsewhere).  `biggest`: the row's largest logit; total: the sum of exp(logit - biggest) over
// the row, read where softmax weights stay as they are.  Renormalised weights are formed from scores scaled by a common factor,
// exp(-biggest) or, for the sigmoid, exp(-min(biggest, 0)): sigmoid(l) = exp(min(l, 0)) / (1 + exp(-|l|)) keeps its digits
// where every score is too small for FP32.
template <bool kSigmoid>
__device__ __forceinline__ float choice_weight(float l, bool live, float biggest, float total, bool renormalize)
{
    float score;
    if constexpr (kSigmoid) score = expf(fminf(l, 0.0f) - (renormalize ? fminf(biggest, 0.0f) : 0.0f)) / (1.0f + expf(-fabsf(l)));
    else score = expf(l - biggest);
    if (l != l) score = l;                                                    // fminf drops a NaN
    if (!live) score = 0.0f;
    if (renormalize) total = warp_sum(score);
    else if (kSigmoid) return score;
    return live ? score / total : 0.0f;
}

template <typename T, int V, bool kSigmoid>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_kernel(const T* __restrict__ logits, int64_t ld, int64_t tokens, int experts, int k, bool renormalize, int64_t* __restrict__ ids,
             float* __restrict__ weights)
{
    const int lane = threadIdx.x & 31;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * kRouteWarps + (threadIdx.x >> 5);
    ptx::grid_dependency_wait();
    if (t >= tokens) return;
    const T* row = logits + t * ld;
    uint32_t key[V];
#pragma unroll
    for (int r = 0; r < V; ++r) key[r] = r * 32 + lane < experts ? key_of(to_float(row[r * 32 + lane])) : 0u;
    uint32_t best = 0;
#pragma unroll
    for (int r = 0; r < V; ++r) best = max(best, key[r]);
    const float biggest = value_of(__reduce_max_sync(kAll, best));
    float total = 0.0f;
    if (!kSigmoid && !renormalize) {
#pragma unroll
        for (int r = 0; r < V; ++r)
            if (r * 32 + lane < experts) total += expf(value_of(key[r]) - biggest);
        total = warp_sum(total);
    }
    int id = -1;
    uint32_t chosen = kMaskedKey;
    if constexpr (sizeof(T) == 2) {
        // A 16-bit logit's key has its digits in the upper half (both types' infinities and NaN included: the order of FP32 values that are
        // exact in them is that of their upper bits), which leaves room for the index: one reduction a round.
        best = 0;
#pragma unroll
        for (int r = 0; r < V; ++r) {
            if (r * 32 + lane < experts) key[r] = packed_key<T>(key[r], r * 32 + lane);
            best = max(best, key[r]);
        }
        for (int j = 0; j < k; ++j) {
            const uint32_t m = __reduce_max_sync(kAll, best);
            if (m <= packed_key<T>(kMaskedKey, 0)) break;                     // nothing left but masked experts
            if (lane == j) { id = static_cast<int>(kIndexMask - (m & kIndexMask)); }
            if (best == m) {
                best = 0;
#pragma unroll
                for (int r = 0; r < V; ++r) {
                    if (key[r] == m) key[r] = 0;
                    best = max(best, key[r]);
                }
            }
        }
        if (id >= 0) chosen = key_of(to_float(row[id]));
    } else {
        for (int j = 0; j < k; ++j) {
            const uint32_t m = __reduce_max_sync(kAll, best);
            if (m <= kMaskedKey) break;
            uint32_t at = 0xffffffffu;                                        // the lowest index of the lane with this key
#pragma unroll
            for (int r = V - 1; r >= 0; --r)
                if (key[r] == m) at = r * 32 + lane;
            const uint32_t winner = __reduce_min_sync(kAll, at);
            if (lane == j) { id = static_cast<int>(winner); chosen = m; }
            if ((winner & 31u) == static_cast<uint32_t>(lane)) {
                best = 0;
#pragma unroll
                for (int r = 0; r < V; ++r) {
                    if (winner == static_cast<uint32_t>(r * 32 + lane)) key[r] = 0;
                    best = max(best, key[r]);
                }
            }
        }
    }
    const float w = choice_weight<kSigmoid>(value_of(chosen), id >= 0, biggest, total, renormalize);
    if (lane < k) {
        ids[t * k + lane] = id;
        weights[t * k + lane] = w;
    }
}

// dlogits from the gradient g of the weights.  p are the softmax's scores, s the sigmoid's, w the weights, sums over a token's choices:
//   softmax                 p_j (sum_i p_i (g_j - g_i) + g_j (1 - sum_i p_i)) of a chosen one, -p_i sum g p of the others
//   softmax, renormalised   w_j sum_i w_i (g_j - g_i)     the chosen alone: the others' share falls out of the ratio
//   sigmoid                 g_j s_j (1 - s_j)
//   sigmoid, renormalised   (1 - s_j) w_j sum_i w_i (g_j - g_i)
// The sums of differences keep their digits where one weight is near 1 and g - sum(g w) would cancel; 1 - sum p is the sum of the others' scores.
template <typename T, bool kSigmoid>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_backward_kernel(const T* __restrict__ logits, int64_t ld, int64_t tokens, int experts, int k, bool renormalize,
                      const int64_t* __restrict__ ids, const float* __restrict__ grad, T* __restrict__ dlogits)
{
    __shared__ uint32_t chosen[kRouteWarps][32];
    const int lane = threadIdx.x & 31;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * kRouteWarps + (threadIdx.x >> 5);
    ptx::grid_dependency_wait();
    if (t >= tokens) return;
    const T* row = logits + t * ld;
    T* out = dlogits + t * experts;
    int64_t id = -1;
    float g = 0.0f;
    if (lane < k) { id = ids[t * k + lane]; g = grad[t * k + lane]; }
    const bool live = id >= 0 && id < experts;
    const float l = live ? to_float(row[id]) : __uint_as_float(0xff800000u);
    if (!live) g = 0.0f;
    // sum over the choices of a_i (g - g_i), by every lane for its own g
    auto weighted_differences = [&](float a) {
        float sum = 0.0f;
        for (int j = 0; j < k; ++j) sum += __shfl_sync(kAll, a, j) * (g - __shfl_sync(kAll, g, j));
        return sum;
    };
    float d, share = 0.0f, biggest = 0.0f;
    const bool dense = !kSigmoid && !renormalize;
    if (dense) {
        uint32_t* mine = chosen[threadIdx.x >> 5];                            // bit i % 32 of word i / 32: expert i was chosen
        mine[lane] = 0;
        __syncwarp();
        if (live) atomicOr(mine + (id >> 5), 1u << (id & 31));
        uint32_t best = 0;
        for (int i = lane; i < experts; i += 32) best = max(best, key_of(to_float(row[i])));
        biggest = value_of(__reduce_max_sync(kAll, best));
        __syncwarp();
        float picked = 0.0f, rest = 0.0f;                                     // scores times their total: of the chosen, of the others
        if (biggest != __uint_as_float(0xff800000u)) {
            for (int i = lane; i < experts; i += 32) {
                const float e = expf(to_float(row[i]) - biggest);
                if (mine[i >> 5] >> lane & 1u) picked += e;
                else rest += e;
            }
            rest = warp_sum(rest);
            share = 1.0f / (warp_sum(picked) + rest);
        }
        const float p = live ? expf(l - biggest) * share : 0.0f;
        const float sum = warp_sum(g * p);
        d = p * (weighted_differences(p) + g * (rest * share));
        for (int i = lane; i < experts; i += 32) {
            // a masked expert's score is 0, also in a row that has no other
            const float v = to_float(row[i]);
            from_float(v == __uint_as_float(0xff800000u) ? 0.0f : -(expf(v - biggest) * share) * sum, out[i]);
        }
    } else {
        const float top = value_of(__reduce_max_sync(kAll, key_of(l)));       // of the chosen: the row's largest is always among them
        const float rest = 1.0f / (1.0f + expf(l));                           // 1 - sigmoid(l)
        if (renormalize) {
            const float w = choice_weight<kSigmoid>(l, live, top, 0.0f, true);
            d = w * weighted_differences(w);
            if (kSigmoid) d *= rest;
        } else {
            d = g * choice_weight<kSigmoid>(l, live, top, 0.0f, false) * rest;
        }
        for (int i = lane; i < experts; i += 32) from_float(0.0f, out[i]);
    }
    __syncwarp();                                                             // the row's other values are written before the chosen ones
    if (live) from_float(d, out[id]);
}

template <typename T, bool kSigmoid>
int route(const void* logits, int64_t ld, int64_t tokens, int experts, int k, bool renormalize, int64_t* ids, float* weights, cudaStream_t stream)
{
    auto kernel = route_kernel<T, 32, kSigmoid>;
    if (experts <= 32) kernel = route_kernel<T, 1, kSigmoid>;
    else if (experts <= 64) kernel = route_kernel<T, 2, kSigmoid>;
    else if (experts <= 128) kernel = route_kernel<T, 4, kSigmoid>;
    else if (experts <= 256) kernel = route_kernel<T, 8, kSigmoid>;
    else if (experts <= 512) kernel = route_kernel<T, 16, kSigmoid>;
    const unsigned blocks = static_cast<unsigned>((tokens + kRouteWarps - 1) / kRouteWarps);
    return host::launch_kernel(kernel, dim3(blocks), dim3(kRouteWarps * 32), 0, stream, true, static_cast<const T*>(logits), ld, tokens, experts, k,
                               renormalize, ids, weights);
}

// Calls f(T*, sigmoid) for a type code and a score function.
template <typename F>
int with_type(int dtype, bool sigmoid, F&& f)
{
    auto scores = [&](auto* type) { return sigmoid ? f(type, std::true_type{}) : f(type, std::false_type{}); };
    switch (dtype) {
        case NVFP4_DTYPE_BF16: return scores(static_cast<__nv_bfloat16*>(nullptr));
        case NVFP4_DTYPE_F16: return scores(static_cast<__half*>(nullptr));
        default: return scores(static_cast<float*>(nullptr));
    }
}

}  // namespace

int launch_route(const void* logits, int64_t ld, int dtype, int64_t tokens, int experts, int k, bool sigmoid, bool renormalize, int64_t* ids,
                 float* weights, cudaStream_t stream)
{
    return with_type(dtype, sigmoid, [&](auto* type, auto s) {
        return route<std::remove_pointer_t<decltype(type)>, decltype(s)::value>(logits, ld, tokens, experts, k, renormalize, ids, weights, stream);
    });
}

int launch_route_backward(const void* logits, int64_t ld, int dtype, int64_t tokens, int experts, int k, bool sigmoid, bool renormalize,
                          const int64_t* ids, const float* grad, void* dlogits, cudaStream_t stream)
{
    const unsigned blocks = static_cast<unsigned>((tokens + kRouteWarps - 1) / kRouteWarps);
    return with_type(dtype, sigmoid, [&](auto* type, auto s) {
        using T = std::remove_pointer_t<decltype(type)>;
        return host::launch_kernel(route_backward_kernel<T, decltype(s)::value>, dim3(blocks), dim3(kRouteWarps * 32), 0, stream, true,
                                   static_cast<const T*>(logits), ld, tokens, experts, k, renormalize, ids, grad, static_cast<T*>(dlogits));
    });
}

}  // namespace nvfp4
