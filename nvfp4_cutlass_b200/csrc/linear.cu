// Dense products with bias, activation and residual in the epilogue, BF16 or FP16 operands on the tensor cores, and their gradients.
//
//   d = activation(x w^T + bias) + residual                x (M, K), w (N, K)
//   dz = dd * activation'(z)      dx = dz w      dw = dz^T x      db = sum over rows of dz
//
// Each product is D[r, c] = sum_k A[r, k] B[c, k] with an operand's memory running along k (K-major: x and w in the forward product) or
// along its own rows (MN-major: w in dx, both in dw); TMA brings 64 of k either way and the instruction descriptor says which, so
// nothing is transposed in memory.  Three kernels:
//   product_kernel       one 128 x BN tile to a CTA; up to eight CTAs of a cluster share the contraction of a tile where there are few
//                        tiles, and add their partial sums through distributed shared memory in a fixed order
//   product_pair_kernel  persistent CTA pairs, 256 x 256 tiles, two accumulators in turn: the epilogue of a tile runs under the
//                        products of the next
//   token_kernel         one or two rows of x and a small weight: no tensor cores
// Sums are FP32 from the first product to the epilogue, which rounds once.
// Every wait is bounded.  One that runs out sets the status bit, where there is a status word, and leaves NaN in what its block did not
// finish (in split form in what the cluster did not), so that nothing that was never computed passes for a result; the block leaves when its
// copies and products in flight have ended, within the same bound.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "gemm_common.cuh"
#include "host_common.hpp"
#include "launchers.hpp"

namespace nvfp4 {
namespace {

using gemm::Ring;

constexpr uint32_t BM = 128, BK = 64;                // rows of A to a CTA; contraction of a ring position (one 128-byte row of either operand)
constexpr uint32_t kRowBytes = BK * 2;
constexpr uint32_t kSlotA = BM * kRowBytes;
constexpr uint32_t kBlockMn = 64 * kRowBytes;        // an MN-major box: 64 rows of the operand x 64 of k
constexpr uint32_t kAll = 0xffffffffu;
constexpr uint32_t kMaxDepth = 8;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// ---- activations -----------------------------------------------------------------------------------------------------
// gelu(z) = z Phi(z); its tanh form 0.5 z (1 + tanh u), u = c (z + 0.044715 z^3), is z sigmoid(2 u) as silu is z sigmoid(z): none of
// them loses the digits of small values to a sum near zero.
// Two forms.  For FP32 outputs CUDA's full-precision functions (activate).  For 16-bit outputs the epilogue would be bound by them (an IEEE
// division alone takes more instructions than the rest; 16384 x 1024 x 1024 with silu took 86 us, 37 without): there (activate2) two values to
// an instruction, the hardware's base-2 exponential and reciprocal, off by 2^-21 or so of the value, and erfc by the Chebyshev fit of Press et
// al., Numerical Recipes, 6.2, erfc(x) = t exp(-x^2 + P(t)), t = 1 / (1 + x / 2), off by 1.2e-7 of its value everywhere.
constexpr float kGeluC = 0.7978845608028654f;        // sqrt(2 / pi)
constexpr float kLog2e = 1.4426950408889634f;
// y = activation(z) and, with kSlope, its derivative there.
template <int kAct, bool kSlope>
__device__ __forceinline__ void activate(float z, float& y, float& slope)
{
    if constexpr (kAct == NVFP4_ACTIVATION_RELU) {
        y = z > 0.0f || z != z ? z : 0.0f;
        slope = z > 0.0f ? 1.0f : z != z ? z : 0.0f;
    } else if constexpr (kAct == NVFP4_ACTIVATION_NONE) {
        y = z;
        slope = 1.0f;
    } else {
        const float bounded = fminf(fmaxf(z, -40.0f), 40.0f);                 // beyond, the slope is constant: no infinity times zero
        if constexpr (kAct == NVFP4_ACTIVATION_GELU) {
            const float cdf = normcdff(z);
            y = z * cdf;
            if constexpr (kSlope) slope = fmaf(bounded, 0.3989422804014327f * expf(-0.5f * bounded * bounded), cdf);
        } else {
            constexpr bool kSilu = kAct == NVFP4_ACTIVATION_SILU;
            const float u2 = kSilu ? z : 2.0f * kGeluC * z * fmaf(0.044715f * z, z, 1.0f);
            const float e = expf(-fabsf(u2)), near = 1.0f / (1.0f + e), far = e * near;
            const float sigmoid = u2 >= 0.0f ? near : far;                    // the larger of sigmoid(u2) and 1 - sigmoid(u2), or the smaller
            y = z * sigmoid;
            if constexpr (kSlope) {
                const float du2 = kSilu ? 1.0f : 2.0f * kGeluC * fmaf(3.0f * 0.044715f * bounded, bounded, 1.0f);
                slope = fmaf(bounded * du2, near * far, sigmoid);
            }
        }
    }
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 exp2_of(float2 v) { return make_float2(ptx::ex2_approx(v.x), ptx::ex2_approx(v.y)); }
__device__ __forceinline__ float2 reciprocal_of(float2 v) { return make_float2(ptx::rcp_approx(v.x), ptx::rcp_approx(v.y)); }
// min(|z|, 40), NaN for NaN: slopes are constant beyond
__device__ __forceinline__ float2 bounded_size(float2 z) { return make_float2(ptx::min_nan(fabsf(z.x), 40.0f), ptx::min_nan(fabsf(z.y), 40.0f)); }
__device__ __forceinline__ float2 with_sign(float2 size, float2 z) { return make_float2(copysignf(size.x, z.x), copysignf(size.y, z.y)); }
template <int kAct, bool kSlope>
__device__ __forceinline__ void activate2(float2 z, float2& y, float2& slope)
{
    using ptx::fma_f32x2;
    using ptx::mul_f32x2;
    if constexpr (kAct == NVFP4_ACTIVATION_RELU || kAct == NVFP4_ACTIVATION_NONE) {
        activate<kAct, kSlope>(z.x, y.x, slope.x);
        activate<kAct, kSlope>(z.y, y.y, slope.y);
    } else if constexpr (kAct == NVFP4_ACTIVATION_GELU) {
        const float2 size = bounded_size(z), t = reciprocal_of(fma_f32x2(size, both(0.35355339f), both(1.0f)));
        // -x^2 + P(t) in base 2, less one for the half of Phi(-|z|) = erfc(|z| / sqrt 2) / 2
        float2 p = both(0.17087277f * kLog2e);
        p = fma_f32x2(p, t, both(-0.82215223f * kLog2e));
        p = fma_f32x2(p, t, both(1.48851587f * kLog2e));
        p = fma_f32x2(p, t, both(-1.13520398f * kLog2e));
        p = fma_f32x2(p, t, both(0.27886807f * kLog2e));
        p = fma_f32x2(p, t, both(-0.18628806f * kLog2e));
        p = fma_f32x2(p, t, both(0.09678418f * kLog2e));
        p = fma_f32x2(p, t, both(0.37409196f * kLog2e));
        p = fma_f32x2(p, t, both(1.00002368f * kLog2e));
        p = fma_f32x2(p, t, both(-1.26551223f * kLog2e - 1.0f));
        const float2 square = mul_f32x2(mul_f32x2(size, both(-0.5f * kLog2e)), size);
        const float2 tail = mul_f32x2(t, exp2_of(fma_f32x2(square, both(1.0f), p))), body = fma_f32x2(tail, both(-1.0f), both(1.0f));
        const float2 cdf = make_float2(z.x < 0.0f ? tail.x : body.x, z.y < 0.0f ? tail.y : body.y);
        y = mul_f32x2(z, cdf);
        if constexpr (kSlope) slope = fma_f32x2(mul_f32x2(with_sign(size, z), both(0.3989422804014327f)), exp2_of(square), cdf);
    } else {
        constexpr bool kSilu = kAct == NVFP4_ACTIVATION_SILU;
        const float2 u2 = kSilu ? z : mul_f32x2(mul_f32x2(z, both(2.0f * kGeluC)), fma_f32x2(mul_f32x2(z, both(0.044715f)), z, both(1.0f)));
        const float2 e = exp2_of(mul_f32x2(make_float2(fabsf(u2.x), fabsf(u2.y)), both(-kLog2e)));
        const float2 near = reciprocal_of(fma_f32x2(e, both(1.0f), both(1.0f))), far = mul_f32x2(e, near);
        const float2 sigmoid = make_float2(u2.x >= 0.0f ? near.x : far.x, u2.y >= 0.0f ? near.y : far.y);
        y = mul_f32x2(z, sigmoid);
        if constexpr (kSlope) {
            float2 inner = with_sign(bounded_size(z), z);
            if constexpr (!kSilu) inner = mul_f32x2(mul_f32x2(inner, both(2.0f * kGeluC)), fma_f32x2(mul_f32x2(inner, both(3.0f * 0.044715f)), inner, both(1.0f)));
            slope = fma_f32x2(inner, mul_f32x2(near, far), sigmoid);
        }
    }
}
// For the backward pass a slope, all of which lie in (-0.2, 1.2), is kept in 16 bits, where z kept in BF16 would cost as much as the rounding of
// the gradient that it multiplies once more.  Two forms, told apart by the code's sign.
//   >= 0   8192 + slope * 2^14: off by 2^-15, which is at most 2^-11 of any slope that is not near zero.  Adding 2^23 + 2^22 + 8192 puts the
//          rounded number into a float's lower bits; of a NaN those are all ones, which as an FP16 number is a NaN again.
//   < 0    slopes in (-0.0622, 0), the negative tails of gelu and silu, where 2^-15 would be percents of them or all: the bits of
//          FP16(slope * 2^20), off by 2^-11 of the slope down to 2^-34 and by 2^-45 below.
// Small positive slopes lie beside the one zero of the slope, where z's own rounding counts as much, and stay in the first form.
constexpr float kSlopeScale = 16384.0f, kSlopeShift = 12582912.0f + 8192.0f, kTailScale = 1048576.0f, kTailLimit = -65216.0f;
// Codes of two slopes, by masks from comparisons of two halves at once: a training step of 8192 x 4096 x 512 with silu takes 178 us in a graph (183
// with values compared and selected one by one, 170 without the second form).
template <int kAct>
__device__ __forceinline__ uint32_t slope_codes(float2 s)
{
    const float2 c = ptx::fma_f32x2(s, both(kSlopeScale), both(kSlopeShift));
    const uint32_t codes = __byte_perm(__float_as_uint(c.x), __float_as_uint(c.y), 0x5410);
    if constexpr (kAct == NVFP4_ACTIVATION_RELU) return codes;
    const float2 t = ptx::mul_f32x2(s, both(kTailScale));
    const __half2 tails = __floats2half2_rn(t.x, t.y);
    const uint32_t in_tail = __hlt2_mask(tails, __float2half2_rn(0.0f)) & __hgt2_mask(tails, __float2half2_rn(kTailLimit));
    return (*reinterpret_cast<const uint32_t*>(&tails) & in_tail) | (codes & ~in_tail);
}
__device__ __forceinline__ float unpack_slope(int16_t c)
{
    return c < 0 ? __half2float(__ushort_as_half(static_cast<unsigned short>(c))) * (1.0f / kTailScale) : (c - 8192) * (1.0f / kSlopeScale);
}

// Calls f(std::integral_constant<int, activation>) for a code: one switch around a loop of elements.
template <typename F>
__device__ __forceinline__ void with_activation(int code, F&& f)
{
    switch (code) {
        case NVFP4_ACTIVATION_RELU: return f(std::integral_constant<int, NVFP4_ACTIVATION_RELU>{});
        case NVFP4_ACTIVATION_GELU: return f(std::integral_constant<int, NVFP4_ACTIVATION_GELU>{});
        case NVFP4_ACTIVATION_GELU_TANH: return f(std::integral_constant<int, NVFP4_ACTIVATION_GELU_TANH>{});
        case NVFP4_ACTIVATION_SILU: return f(std::integral_constant<int, NVFP4_ACTIVATION_SILU>{});
        default: return f(std::integral_constant<int, NVFP4_ACTIVATION_NONE>{});
    }
}

// ---- epilogue --------------------------------------------------------------------------------------------------------

struct Epilogue {
    void* d; int64_t ldd;                            // (rows, cols), of the operands' type or FP32
    int16_t* slopes; int64_t lds;                    // activation'(z) for the backward pass, or NULL
    const void* bias;                                // (cols) or NULL
    const void* residual; int64_t ldr;               // of d's type, or NULL
    uint32_t rows, cols;
    int activation;
    const float* scale;                              // what the sums are multiplied by, or NULL: see linear_dz_kernel
    bool staged;                                     // rows of d, residual and slopes are multiples of 16 bytes: see Stage
};

// Up to kN accumulators of a lane: output column `col`, rows row0 + i, i < count.  The lanes of a warp hold neighbouring columns, so that
// every access of the warp is one run of an output row, whatever its alignment.  T: operands and bias, D: output and residual.
// The residual's loads go out together, from rows and columns that exist (a load in a branch of its own waits for its value there: 8192 x
// 4096 x 4096 took 465 us in place of the 184 without a residual).  All of them are plain loads: __ldg is an asm statement that the
// compiler may move, and it was moved ahead of the test for a NULL bias, out of the loop over a tile's columns.
template <typename T, typename D, uint32_t kN>
__device__ __forceinline__ void finish(float (&v)[kN], uint32_t row0, uint32_t count, uint32_t col, const Epilogue& e, float factor)
{
    if (row0 >= e.rows || count == 0) return;
    const uint32_t rows = min(count, e.rows - row0), last = rows - 1, at = min(col, e.cols - 1);
    const bool mine = col < e.cols;
    D r[kN];
    if (e.residual != nullptr) {
        const D* from = static_cast<const D*>(e.residual) + static_cast<int64_t>(row0) * e.ldr + at;
#pragma unroll
        for (uint32_t i = 0; i < kN; ++i) r[i] = from[static_cast<int64_t>(min(i, last)) * e.ldr];
    }
    if (factor != 1.0f) {
#pragma unroll
        for (uint32_t i = 0; i < kN; ++i) v[i] *= factor;
    }
    if (e.bias != nullptr) {
        const float b = to_float(static_cast<const T*>(e.bias)[at]);
#pragma unroll
        for (uint32_t i = 0; i < kN; ++i) v[i] += b;
    }
    if (e.activation != NVFP4_ACTIVATION_NONE)
        with_activation(e.activation, [&](auto act) {
            constexpr int kAct = decltype(act)::value;
            auto two = [&](uint32_t i, float2& slope, auto with_slope) {
                constexpr bool kSlope = decltype(with_slope)::value;
                if constexpr (std::is_same<D, float>::value) {
                    activate<kAct, kSlope>(v[i], v[i], slope.x);
                    activate<kAct, kSlope>(v[i + 1], v[i + 1], slope.y);
                } else {
                    float2 y;
                    activate2<kAct, kSlope>(make_float2(v[i], v[i + 1]), y, slope);
                    v[i] = y.x;
                    v[i + 1] = y.y;
                }
            };
            float2 slope = make_float2(0.0f, 0.0f);
            if (e.slopes != nullptr) {
                int16_t* to = e.slopes + static_cast<int64_t>(row0) * e.lds + at;
#pragma unroll
                for (uint32_t i = 0; i < kN; i += 2) {
                    two(i, slope, std::true_type{});
                    const uint32_t codes = slope_codes<kAct>(slope);
                    if (i < rows && mine) to[i * e.lds] = static_cast<int16_t>(codes);
                    if (i + 1 < rows && mine) to[(i + 1) * e.lds] = static_cast<int16_t>(codes >> 16);
                }
            } else {
#pragma unroll
                for (uint32_t i = 0; i < kN; i += 2) two(i, slope, std::false_type{});
            }
        });
    if (e.residual != nullptr) {
#pragma unroll
        for (uint32_t i = 0; i < kN; ++i) v[i] += to_float(r[i]);
    }
    if (!mine) return;
    // eight stores in a row where there are eight rows: each in a branch of its own they took a microsecond for 32
    D* to = static_cast<D*>(e.d) + static_cast<int64_t>(row0) * e.ldd + at;
#pragma unroll
    for (uint32_t g = 0; g < kN; g += 8) {
        if (g + 8 <= rows) {
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) to[i * e.ldd] = from_float<D>(v[g + i]);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i)
                if (g + i < rows) to[i * e.ldd] = from_float<D>(v[g + i]);
        }
        to += 8 * e.ldd;
    }
}

// 32 x 32 values, lane l holding row l: afterwards lane l holds column l.  Five butterfly steps.
__device__ __forceinline__ void transpose(float (&v)[32], uint32_t lane)
{
#pragma unroll
    for (uint32_t s = 16; s > 0; s >>= 1) {
        const bool up = (lane & s) != 0;
#pragma unroll
        for (uint32_t i = 0; i < 32; ++i) {
            if ((i & s) != 0) continue;
            const float got = __shfl_xor_sync(kAll, up ? v[i] : v[i | s], s);
            if (up) v[i] = got;
            else v[i | s] = got;
        }
    }
}

template <typename T> struct Pair2;
template <> struct Pair2<__nv_bfloat16> { using type = __nv_bfloat162; };
template <> struct Pair2<__half> { using type = __half2; };
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w)
{
    const typename Pair2<T>::type h = *reinterpret_cast<const typename Pair2<T>::type*>(&w);
    if constexpr (std::is_same<T, __nv_bfloat16>::value) return __bfloat1622float2(h);
    else return __half22float2(h);
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b)
{
    typename Pair2<T>::type h;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) h = __floats2bfloat162_rn(a, b);
    else h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <uint32_t kN>
__device__ __forceinline__ void load_accumulators(uint32_t taddr, float (&v)[kN])
{
    uint32_t raw[kN];
    if constexpr (kN == 32) ptx::tmem_ld_32x32b_x32(taddr, raw);
    else ptx::tmem_ld_32x32b_x16(taddr, raw);
    ptx::tmem_ld_wait();
#pragma unroll
    for (uint32_t i = 0; i < kN; ++i) v[i] = __uint_as_float(raw[i]);
}

// An epilogue warp's way out through shared memory, where TMA can address the output: 32 rows x 64 columns (32 of FP32) at a time, a row (128
// bytes, 128-byte swizzle) to a lane as tensor memory gives them, so that nothing has to be transposed and every line of the output is
// written whole.  The residual comes into the same buffer by TMA beforehand and is replaced by the result in place.
// Slopes go the same way beside a 16-bit output.
template <typename D>
constexpr uint32_t kBox = 128 / sizeof(D);
constexpr uint32_t kBoxBytes = 32 * 128;
struct Maps {
    CUtensorMap d, residual, slopes;                 // boxes of 32 rows x 128 bytes
};
template <typename T, typename D>
struct Stage {
    uint32_t out, out_step, slopes, slopes_step;     // shared memory: buffers of the output (and residual) and of the slopes, of box 0 and from one to the next
    uint64_t* landed;                                // per box: its residual is there
    uint32_t phase = 0;
    const Maps* maps;
    long long budget;                                // of a wait, in cycles
    float factor;                                    // *e.scale, where there is one (read in front of every box it took 5 of a call's 28 us)
    uint32_t requested = 0;                          // boxes whose residual is under way
    bool withhold = false;                           // test of the expired wait: residuals are not asked for

    // Everything that the warp has given to TMA has been read: the buffers may be written.
    __device__ __forceinline__ void reclaim(uint32_t lane) const
    {
        if (lane == 0) ptx::bulk_wait_read();
        __syncwarp();
    }
    __device__ __forceinline__ void request(uint32_t box, uint32_t col, uint32_t row0, uint32_t lane)
    {
        if (withhold) return;
        requested |= 1u << box;
        if (lane == 0) {
            ptx::mbar_arrive_expect_tx(landed + box, kBoxBytes);
            tma_load(out + box * out_step, &maps->residual, landed + box, col, row0);
        }
    }
    // After a wait that expired
    __device__ __forceinline__ void settle()
    {
        const long long until = clock64() + budget;
#pragma unroll
        for (uint32_t box = 0; box < 4; ++box)
            if (requested >> box & 1u) ptx::mbar_settle(landed + box, phase >> box & 1u, until);
        requested = 0;
        __syncwarp();
    }
    static __device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int32_t c0, int32_t c1)
    {
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                     ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(ptx::smem_u32(bar)), "r"(c0), "r"(c1)
                     : "memory");
    }
    // Bias of the columns [col, col + 32), two to a word: the same for every lane
    static __device__ __forceinline__ void load_bias(const Epilogue& e, uint32_t col, uint32_t (&b)[16])
    {
        const T* from = static_cast<const T*>(e.bias) + col;
        if (col + 32 <= e.cols && (reinterpret_cast<uintptr_t>(from) & 15u) == 0) {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint4 q = reinterpret_cast<const uint4*>(from)[i];
                b[4 * i] = q.x; b[4 * i + 1] = q.y; b[4 * i + 2] = q.z; b[4 * i + 3] = q.w;
            }
        } else {
            const uint16_t* bits = reinterpret_cast<const uint16_t*>(e.bias);
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i)
                b[i] = bits[min(col + 2 * i, e.cols - 1)] | static_cast<uint32_t>(bits[min(col + 2 * i + 1, e.cols - 1)]) << 16;
        }
    }
    // One box: accumulators at taddr, columns [col, col + kBox<D>).  False: the residual never came.
    __device__ __forceinline__ bool finish(uint32_t taddr, uint32_t box, uint32_t col, uint32_t row0, uint32_t lane, const Epilogue& e,
                                           volatile uint32_t* abort_flag)
    {
        if (e.residual != nullptr) {
            if (!ptx::all_lanes(ptx::mbar_wait_budget(landed + box, phase >> box & 1u, abort_flag, budget))) return false;
            phase ^= 1u << box;
            requested &= ~(1u << box);
        }
#pragma unroll
        for (uint32_t half = 0; half < kBox<D> / 32; ++half) {
            float v[32];
            uint32_t b[16];
            if (e.bias != nullptr) load_bias(e, col + half * 32, b);
            load_accumulators(taddr + half * 32, v);
            if (factor != 1.0f) {
#pragma unroll
                for (uint32_t i = 0; i < 32; i += 2) {
                    const float2 f = ptx::mul_f32x2(make_float2(v[i], v[i + 1]), both(factor));
                    v[i] = f.x;
                    v[i + 1] = f.y;
                }
            }
            if (e.bias != nullptr) {
#pragma unroll
                for (uint32_t i = 0; i < 16; ++i) {
                    const float2 f = unpack2<T>(b[i]);
                    v[2 * i] += f.x;
                    v[2 * i + 1] += f.y;
                }
            }
            auto piece = [&](uint32_t buffer, uint32_t q) { return buffer + lane * 128 + (((half * 4 + q) ^ (lane & 7u)) << 4); };
            if constexpr (std::is_same<D, float>::value) {
                if (e.activation != NVFP4_ACTIVATION_NONE)
                    with_activation(e.activation, [&](auto act) {
                        float slope;
#pragma unroll
                        for (uint32_t i = 0; i < 32; ++i) activate<decltype(act)::value, false>(v[i], v[i], slope);
                    });
#pragma unroll
                for (uint32_t q = 0; q < 8; ++q) {
                    const uint32_t to = piece(out + box * out_step, q);
                    if (e.residual != nullptr) {
                        const uint4 r = ptx::lds128(to);
                        v[4 * q] += __uint_as_float(r.x);
                        v[4 * q + 1] += __uint_as_float(r.y);
                        v[4 * q + 2] += __uint_as_float(r.z);
                        v[4 * q + 3] += __uint_as_float(r.w);
                    }
                    ptx::sts128(to, __float_as_uint(v[4 * q]), __float_as_uint(v[4 * q + 1]), __float_as_uint(v[4 * q + 2]), __float_as_uint(v[4 * q + 3]));
                }
            } else {
                if (e.activation != NVFP4_ACTIVATION_NONE)
                    with_activation(e.activation, [&](auto act) {
                        constexpr int kAct = decltype(act)::value;
                        float2 y, slope;
                        if (e.slopes != nullptr) {
#pragma unroll
                            for (uint32_t q = 0; q < 4; ++q) {
                                uint32_t w[4];
#pragma unroll
                                for (uint32_t i = 0; i < 4; ++i) {
                                    const uint32_t at = 8 * q + 2 * i;
                                    activate2<kAct, true>(make_float2(v[at], v[at + 1]), y, slope);
                                    v[at] = y.x;
                                    v[at + 1] = y.y;
                                    w[i] = slope_codes<kAct>(slope);
                                }
                                ptx::sts128(piece(slopes + box * slopes_step, q), w[0], w[1], w[2], w[3]);
                            }
                        } else {
#pragma unroll
                            for (uint32_t i = 0; i < 32; i += 2) {
                                activate2<kAct, false>(make_float2(v[i], v[i + 1]), y, slope);
                                v[i] = y.x;
                                v[i + 1] = y.y;
                            }
                        }
                    });
#pragma unroll
                for (uint32_t q = 0; q < 4; ++q) {
                    const uint32_t to = piece(out + box * out_step, q);
                    if (e.residual != nullptr) {
                        const uint4 r = ptx::lds128(to);
                        const uint32_t rw[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i) {
                            const float2 f = unpack2<T>(rw[i]);
                            v[8 * q + 2 * i] += f.x;
                            v[8 * q + 2 * i + 1] += f.y;
                        }
                    }
                    ptx::sts128(to, pack2<T>(v[8 * q], v[8 * q + 1]), pack2<T>(v[8 * q + 2], v[8 * q + 3]), pack2<T>(v[8 * q + 4], v[8 * q + 5]),
                                pack2<T>(v[8 * q + 6], v[8 * q + 7]));
                }
            }
        }
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            ptx::tma_store_2d(&maps->d, out + box * out_step, col, row0);
            if (e.slopes != nullptr) ptx::tma_store_2d(&maps->slopes, slopes + box * slopes_step, col, row0);
            ptx::bulk_commit();
        }
        return true;
    }
};

// ---- operands --------------------------------------------------------------------------------------------------------

// The tile of an operand's rows [row0, row0 + kRows) x contraction [64 kb, 64 kb + 64) into shared memory.  What lies outside of the
// tensor arrives as zeros.  load(dst, inner, outer) is the TMA load of one box.
template <uint32_t kRows, typename Load>
__device__ __forceinline__ void load_tile(uint8_t* dst, bool mn_major, uint32_t row0, uint32_t kb, Load&& load)
{
    if (!mn_major) {
        load(dst, kb * BK, row0);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < (kRows + 63) / 64; ++i) load(dst + i * kBlockMn, row0 + i * 64, kb * BK);
    }
}
// Descriptor of the 16 of k at step `step` of a tile
__device__ __forceinline__ uint64_t operand_desc(uint32_t tile, bool mn_major, uint32_t step)
{
    return mn_major ? ptx::make_smem_desc_mn(tile + step * 16 * kRowBytes, kBlockMn, 8 * kRowBytes)
                    : ptx::make_smem_desc(tile + step * 32, 8 * kRowBytes, ptx::kSwizzle128B);
}

constexpr int kTileSmem = 216 * 1024;                // most that a block of product_kernel takes
struct Product {
    uint32_t tiles_a, tiles_b, k_blocks;
    uint32_t splits_log2, depth;                     // product_kernel: CTAs to a tile, ring positions
    bool a_mn, b_mn;
    int32_t* status;
    long long budget;                                // of every wait, in cycles
    uint32_t withhold;                               // what a test of the expired waits keeps back: kProducts, kResiduals
};
enum Withhold : uint32_t { kNothing = 0, kProducts = 1, kResiduals = 2 };
constexpr float kNan = NAN;

// ---- one tile to a CTA or cluster --------------------------------------------------------------------------------------

constexpr int kTileThreads = 192;                    // warp 0: TMA, warp 1: products, warps 2-5: epilogue
constexpr uint32_t kTileEpiWarps = 4;
constexpr uint32_t tile_stage(uint32_t bn) { return kSlotA + bn * kRowBytes; }
// Partial sums of a cluster: [source CTA][row][columns that a CTA finishes, and padding that keeps the rows on different banks].
// A row moves `partial_words` at a time; sixteen columns among eight CTAs leave two to each, which need no padding.
constexpr uint32_t partial_words(uint32_t bn) { return bn < 32 ? 2 : 4; }
__host__ __device__ constexpr uint32_t partial_pad(uint32_t bn, uint32_t splits) { return bn >= 32 ? 4 : splits == 8 ? 0 : 2; }
__host__ __device__ constexpr uint32_t partial_bytes(uint32_t bn, uint32_t splits) { return splits > 1 ? (bn + splits * partial_pad(bn, splits)) * BM * 4 : 0; }
constexpr uint32_t tile_smem(uint32_t bn, uint32_t depth, uint32_t splits)
{
    return 1024 + depth * tile_stage(bn) + partial_bytes(bn, splits) + (2 * kMaxDepth + 5) * 8 + 16 + kTileEpiWarps * 32;
}
// For an FP32 output the epilogue warps take the accumulators over every four K blocks and add them up in registers, two accumulators in
// turn: the tensor core cuts what it adds to a long sum (K = 4096 in one accumulator: off by 4.3e-6 of the result, FP32 sums by 6e-7).
// The cut goes one way and grows with the sum: over operands of one sign by 6e-9 of it for every product of FP16, 1.9e-9 of BF16 (37500 to 275000
// tokens to an accumulator).  A 16-bit output stays in its accumulator while that is less than half of the half step of its rounding, 2^-12
// and 2^-9; longer sums (a weight's gradient over very many tokens) are taken out every sixteen K blocks (kLong; dw of 65536 FP16 tokens, 4096 x
// 2048: some 1.5 ms, 0.9 on CTA pairs).
constexpr uint32_t kChunkBlocks = 4, kLongChunkBlocks = 16;
template <typename T>
constexpr uint32_t kLongestSum = std::is_same<T, __half>::value ? 16384 : 262144;

// kSwap: A is the weight and the output's columns lie on the tensor memory's lanes; else A is x and a warp's 32 x 32 accumulators are
// transposed first.  D: type of the output.
template <typename T, typename D, uint32_t BN, bool kSwap, bool kLong>
__global__ void __launch_bounds__(kTileThreads, (std::is_same<D, float>::value || kLong) && BN > 64 ? 1 : 2)
product_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ Maps maps, const Product p,
               const Epilogue e)
{
    constexpr bool kWide = std::is_same<D, float>::value || kLong;
    constexpr uint32_t kTaken = kLong ? kLongChunkBlocks : kChunkBlocks;     // K blocks after which accumulators are taken out
    constexpr uint32_t kChunk = BN < 32 ? BN : 32, kStage = tile_stage(BN), kCols = (kWide ? 2 : 1) * BN < 32 ? 32 : (kWide ? 2 : 1) * BN;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (smem - ptx::smem_u32(smem_raw));
    const uint32_t splits = 1u << p.splits_log2, depth = p.depth;
    const uint32_t partial = smem + depth * kStage;
    uint64_t* full = reinterpret_cast<uint64_t*>(gen + depth * kStage + partial_bytes(BN, splits));
    uint64_t* drained = full + kMaxDepth;
    uint64_t* tmem_full = drained + kMaxDepth;       // per accumulator
    uint64_t* tmem_empty = tmem_full + 2;
    uint64_t* landed = tmem_empty + 2;               // [epilogue warp][4] residual of a box
    uint64_t* settled = landed + 4 * kTileEpiWarps;  // the products have ended, after a wait that expired
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(settled + 1);
    volatile uint32_t* abort_flag = tmem_slot + 1;

    const uint32_t warp = ptx::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const uint32_t rank = blockIdx.x & (splits - 1), tile = blockIdx.x >> p.splits_log2;
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < depth; ++i) { ptx::mbar_init(full + i, 1); ptx::mbar_init(drained + i, 1); }
        for (uint32_t i = 0; i < 2; ++i) { ptx::mbar_init(tmem_full + i, 1); ptx::mbar_init(tmem_empty + i, kTileEpiWarps); }
        for (uint32_t i = 0; i < 4 * kTileEpiWarps + 1; ++i) ptx::mbar_init(landed + i, 1);
        *abort_flag = 0;
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&tm_a);
        ptx::prefetch_tensormap(&tm_b);
    }
    if (warp == 1) ptx::tmem_alloc<kCols>(tmem_slot);
    ptx::tcgen05_fence_before_sync();
    if (splits > 1) ptx::cluster_sync();             // every CTA of the cluster runs before anybody writes into its shared memory
    else __syncthreads();
    ptx::tcgen05_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    ptx::grid_dependency_wait();

    uint32_t a_blk, b_blk;
    gemm::tile_coords(tile, p.tiles_a, p.tiles_b, 8, a_blk, b_blk);
    const uint32_t a0 = a_blk * BM, b0 = b_blk * BN;
    const uint32_t kb0 = static_cast<uint32_t>(static_cast<uint64_t>(p.k_blocks) * rank >> p.splits_log2);
    const uint32_t kb1 = static_cast<uint32_t>(static_cast<uint64_t>(p.k_blocks) * (rank + 1) >> p.splits_log2);
    const uint32_t chunks = kWide ? (kb1 - kb0 + kTaken - 1) / kTaken : 1;
    bool ok = true;
    auto give_up = [&] {
        *abort_flag = 1;
        if (p.status != nullptr) atomicOr(p.status, 1);
        ok = false;
    };
    auto next = [&](Ring& r) {
        if (++r.slot == depth) { r.slot = 0; r.phase ^= 1; }
    };
    const uint32_t quad = warp & 3, row = quad * 32 + lane;                   // epilogue: the warp's quarter of the lanes
    const float factor = !kSwap && e.scale != nullptr ? *e.scale : 1.0f;      // (swapped: forward products alone)
    const uint32_t taddr = tmem + ((quad * 32) << 16);
    if (warp == 0) {
        const uint32_t issue = ptx::elect_one();
        Ring r;
        uint32_t loaded = 0;
        for (uint32_t kb = kb0; kb < kb1; ++kb, ++loaded) {
            if (!ptx::all_lanes(ptx::mbar_wait_budget(drained + r.slot, r.phase ^ 1, abort_flag, p.budget))) { give_up(); break; }
            uint8_t* to = gen + r.slot * kStage;
            uint64_t* bar = full + r.slot;
            ptx::mbar_arrive_expect_tx(bar, kStage, issue);
            load_tile<BM>(to, p.a_mn, a0, kb, [&](uint8_t* dst, uint32_t c0, uint32_t c1) { ptx::tma_load_2d(dst, &tm_a, bar, c0, c1, issue); });
            load_tile<BN>(to + kSlotA, p.b_mn, b0, kb, [&](uint8_t* dst, uint32_t c0, uint32_t c1) { ptx::tma_load_2d(dst, &tm_b, bar, c0, c1, issue); });
            next(r);
        }
        ptx::grid_launch_dependents();
        // the last commits arrive before the block may leave
        for (uint32_t i = 0; ok && i < depth; ++i) {
            if (!ptx::all_lanes(ptx::mbar_wait_budget(drained + r.slot, r.phase ^ 1, abort_flag, p.budget))) give_up();
            next(r);
        }
        if (!ok) {
            const long long until = clock64() + p.budget;
            for (uint32_t n = loaded > depth ? loaded - depth : 0; n < loaded; ++n) ptx::mbar_settle(full + n % depth, n / depth & 1u, until);
            __syncwarp();
        }
    } else if (warp == 1) {
        const uint32_t issue = ptx::elect_one();
        const uint32_t idesc = ptx::make_idesc_f16(BM, BN, std::is_same<T, __nv_bfloat16>::value, p.a_mn, p.b_mn);
        Ring r;
        for (uint32_t kb = kb0; kb < kb1 && p.withhold != kProducts; ++kb) {
            const uint32_t n = kb - kb0, c = kWide ? n / kTaken : 0, acc = c & 1;
            const bool first = kWide ? n % kTaken == 0 : n == 0;
            if (kWide && first && !ptx::all_lanes(ptx::mbar_wait_budget(tmem_empty + acc, ((c >> 1) & 1) ^ 1, abort_flag, p.budget))) { give_up(); break; }
            if (!ptx::all_lanes(ptx::mbar_wait_budget(full + r.slot, r.phase, abort_flag, p.budget))) { give_up(); break; }
            ptx::tcgen05_fence_after_sync();
            const uint32_t at = smem + r.slot * kStage;
#pragma unroll
            for (uint32_t s = 0; s < BK / 16; ++s)
                ptx::tcgen05_mma_f16(tmem + acc * BN, operand_desc(at, p.a_mn, s), operand_desc(at + kSlotA, p.b_mn, s), idesc, first && s == 0 ? 0u : 1u, issue);
            ptx::tcgen05_commit(drained + r.slot, issue);
            if (kb + 1 == kb1 || (kWide && n % kTaken == kTaken - 1)) ptx::tcgen05_commit(tmem_full + acc, issue);
            next(r);
        }
        if (!ok || !ptx::all_lanes(*abort_flag == 0)) {
            ptx::tcgen05_commit(settled, issue);
            ptx::mbar_settle(settled, 0, clock64() + p.budget);
            __syncwarp();
        }
    } else {
        [[maybe_unused]] float sum[kWide ? BN : 1];
        if constexpr (kWide) {
#pragma unroll
            for (uint32_t i = 0; i < BN; ++i) sum[i] = 0.0f;
        }
        for (uint32_t c = 0; c < chunks; ++c) {
            const uint32_t acc = c & 1;
            if (!ptx::all_lanes(ptx::mbar_wait_relaxed(tmem_full + acc, (c >> 1) & 1, abort_flag, 20, p.budget))) { give_up(); break; }
            ptx::tcgen05_fence_after_sync();
            if constexpr (kWide) {
#pragma unroll
                for (uint32_t c0 = 0; c0 < BN; c0 += kChunk) {
                    float v[kChunk];
                    load_accumulators(taddr + acc * BN + c0, v);
#pragma unroll
                    for (uint32_t i = 0; i < kChunk; ++i) sum[c0 + i] += v[i];
                }
                ptx::tcgen05_fence_before_sync();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(tmem_empty + acc);
            }
        }
        if constexpr (kWide) {                       // back to tensor memory, which can be indexed: what follows is there once, not once per chunk
#pragma unroll
            for (uint32_t c0 = 0; c0 < BN; c0 += kChunk) {
                uint32_t raw[kChunk];
#pragma unroll
                for (uint32_t i = 0; i < kChunk; ++i) raw[i] = __float_as_uint(sum[c0 + i]);
                ptx::tmem_st_32x32b(taddr + c0, raw);
            }
            ptx::tmem_st_wait();
        }
    }

    // epilogue: 128 rows of A in all
    const uint32_t live = kSwap ? min(BN, e.rows - b0) : min(BN, e.cols - b0);          // columns of the tile that anybody wants
    auto give = [&](float (&v)[kChunk], uint32_t column, uint32_t count) {    // columns [column, column + count) of the tile
        if constexpr (kSwap) {
            finish<T, D>(v, b0 + column, count, a0 + row, e, factor);
        } else {
            transpose(v, lane);
            finish<T, D>(v, a0 + quad * 32, 32, b0 + column + lane, e, factor);
        }
    };
    if (splits > 1) {
        const uint32_t width_log2 = __popc(BN - 1) - p.splits_log2, width = 1u << width_log2;          // columns that a CTA finishes
        constexpr uint32_t kWords = partial_words(BN);
        const uint32_t pitch = (width + partial_pad(BN, splits)) * 4, block = BM * pitch;                       // of a row, of a source's rows
        if (warp >= 2) {
            const uint32_t mine = partial + rank * block + row * pitch;
#pragma unroll 1
            for (uint32_t c0 = 0; c0 < live; c0 += kChunk) {
                float v[kChunk];
                load_accumulators(taddr + c0, v);
                if (!ok) {
#pragma unroll
                    for (uint32_t i = 0; i < kChunk; ++i) v[i] = kNan;
                }
#pragma unroll
                for (uint32_t i = 0; i < kChunk; i += kWords) {
                    const uint32_t c = c0 + i;               // columns that nobody wants included: they have their place, too
                    const uint32_t to = ptx::map_to_cta(mine + (c & (width - 1)) * 4, c >> width_log2);
                    if constexpr (kWords == 4) ptx::st_cluster_f32x4(to, v[i], v[i + 1], v[i + 2], v[i + 3]);
                    else ptx::st_cluster_f32x2(to, v[i], v[i + 1]);
                }
            }
        }
        ptx::cluster_sync();                         // partial sums have arrived; nobody touches another CTA's memory from here on
        if (warp >= 2) {
            const float* mine = reinterpret_cast<const float*>(gen + (partial - smem) + row * pitch);
#pragma unroll 1
            for (uint32_t c0 = 0; c0 < width; c0 += kChunk) {
                const uint32_t first = rank * width + c0;
                if (first >= live) break;
                const uint32_t count = min(min(width - c0, kChunk), live - first);
                float v[kChunk];
#pragma unroll
                for (uint32_t i = 0; i < kChunk; i += kWords) {
#pragma unroll
                    for (uint32_t j = 0; j < kWords; ++j) v[i + j] = 0.0f;
                    if (i >= count) continue;                // (width is a multiple of kWords)
                    // in the order of the sources, eight loads under way
                    float4 part[8];
#pragma unroll
                    for (uint32_t s = 0; s < 8; ++s) {
                        const float* from = mine + s * (block / 4) + c0 + i;
                        if (s >= splits) continue;
                        if constexpr (kWords == 4) {
                            part[s] = *reinterpret_cast<const float4*>(from);
                        } else {
                            const float2 two = *reinterpret_cast<const float2*>(from);
                            part[s] = make_float4(two.x, two.y, 0.0f, 0.0f);
                        }
                    }
#pragma unroll
                    for (uint32_t s = 0; s < 8; ++s) {
                        if (s >= splits) continue;
                        v[i] += part[s].x;
                        v[i + 1] += part[s].y;
                        if constexpr (kWords == 4) { v[i + 2] += part[s].z; v[i + 3] += part[s].w; }
                    }
                }
                give(v, first, kSwap ? count : 32);
            }
        }
    } else if (warp >= 2) {
        uint32_t done = 0;                           // columns of the tile that have left
        if constexpr (!kSwap) {
            if (e.staged && ok) {
                // the ring is at rest (the accumulators are complete): its memory takes the boxes, four for every warp: of the output, or
                // two of the output and two of the slopes
                constexpr uint32_t kColumns = kBox<D>;
                const uint32_t at = smem + (warp - 2) * 4 * kBoxBytes, row0 = a0 + quad * 32;
                Stage<T, D> stage{at, kBoxBytes, at + 2 * kBoxBytes, kBoxBytes, landed + 4 * (warp - 2), 0, &maps, p.budget, factor, 0, p.withhold == kResiduals};
                if (row0 < e.rows) {
                    if (e.residual != nullptr)
                        for (uint32_t c = 0; c < live; c += kColumns) stage.request(c / kColumns, b0 + c, row0, lane);
#pragma unroll 1
                    for (; done < live; done += kColumns)
                        if (!stage.finish(taddr + done, done / kColumns, b0 + done, row0, lane, e, abort_flag)) { give_up(); break; }
                    if (!ok) stage.settle();
                    if (lane == 0) ptx::bulk_wait();
                    __syncwarp();
                } else {
                    done = live;
                }
            }
        }
        // (unrolled, a cold call spent 3 us a chunk fetching instructions: 13 us of a router's 41)
#pragma unroll 1
        for (uint32_t c0 = done; c0 < live; c0 += kChunk) {
            float v[kChunk];
            load_accumulators(taddr + c0, v);
            if (!ok) {
#pragma unroll
                for (uint32_t i = 0; i < kChunk; ++i) v[i] = kNan;
            }
            give(v, c0, kSwap ? min(kChunk, live - c0) : 32);
        }
    }
    ptx::tcgen05_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        ptx::tcgen05_fence_after_sync();
        ptx::tmem_dealloc<kCols>(tmem);
    }
}

// ---- one or two tokens ---------------------------------------------------------------------------------------------------

// A product of one or two rows is a pass over the weight and nothing else.  While the weight is small, what counts is how soon the loads go
// out, not how many are under way: no tensor memory, barriers or clusters; some warps (a power of two) take a row of w, a lane eight
// 16-byte loads at a time, FP32 sums in a fixed order, and one lane a token finishes the element.
// This / the tensor cores, one token, BF16, in a graph: 512 x 512 1.8 / 3.6 us, 1024 x 4096 3.6 / 4.9, 4096 x 1024 3.6 / 5.2, 3000 x 2048 6.2 / 6.0,
// 2048 x 4096 6.5 / 6.3, 4096 x 4096 11.3 / 9.1: taken up to kTokenMostWeights elements of w.
constexpr uint64_t kTokenMostWeights = 5u << 20;
constexpr int kTokenThreads = 256, kTokenWarps = kTokenThreads / 32, kTokenLoads = 8;
template <typename T, typename D, int kTokens>
__global__ void __launch_bounds__(kTokenThreads)
token_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ w, int64_t ldw, uint32_t k, uint32_t warps_log2, const Epilogue e)
{
    __shared__ float part[kTokenWarps][kTokens];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = 1u << warps_log2, share = warp & (warps - 1);
    const uint32_t n = blockIdx.x * (kTokenWarps >> warps_log2) + (warp >> warps_log2);
    const bool mine = n < e.cols;
    ptx::grid_dependency_wait();
    float sum[kTokens];
#pragma unroll
    for (int t = 0; t < kTokens; ++t) sum[t] = 0.0f;
    if (mine) {
        const uint4* row = reinterpret_cast<const uint4*>(w + static_cast<int64_t>(n) * ldw);
        const uint32_t words = k / 8, step = 32 * warps;
        for (uint32_t c0 = share * 32 + lane; c0 < words; c0 += step * kTokenLoads) {
            uint4 v[kTokenLoads];
#pragma unroll
            for (int i = 0; i < kTokenLoads; ++i) v[i] = c0 + i * step < words ? row[c0 + i * step] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int i = 0; i < kTokenLoads; ++i) {
                if (c0 + i * step >= words) break;
                const uint32_t vw[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
                for (int t = 0; t < kTokens; ++t) {
                    const uint4 q = reinterpret_cast<const uint4*>(x + t * ldx)[c0 + i * step];
                    const uint32_t xw[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 a = unpack2<T>(vw[j]), b = unpack2<T>(xw[j]);
                        sum[t] = fmaf(a.x, b.x, sum[t]);
                        sum[t] = fmaf(a.y, b.y, sum[t]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum[t] += __shfl_xor_sync(kAll, sum[t], d);
        if (lane == 0) part[warp][t] = sum[t];
    }
    __syncthreads();
    if (!mine || share != 0 || lane >= kTokens) return;
    float z = 0.0f;
    for (uint32_t i = 0; i < warps; ++i) z += part[warp + i][lane];
    if (e.scale != nullptr) z *= *e.scale;
    if (e.bias != nullptr) z += to_float(static_cast<const T*>(e.bias)[n]);
    float y = z;
    with_activation(e.activation, [&](auto act) {
        constexpr int kAct = decltype(act)::value;
        float slope = 1.0f;
        activate<kAct, true>(z, y, slope);
        if (e.slopes != nullptr) e.slopes[lane * e.lds + n] = static_cast<int16_t>(slope_codes<kAct>(both(slope)));
    });
    if (e.residual != nullptr) y += to_float(static_cast<const D*>(e.residual)[lane * e.ldr + n]);
    static_cast<D*>(e.d)[lane * e.ldd + n] = from_float<D>(y);
}

// ---- persistent CTA pairs ----------------------------------------------------------------------------------------------

constexpr int kPairThreads = 320;                    // warp 0: TMA, warp 1: products (even CTA), warps 2-9: epilogue
constexpr uint32_t kPairFirstEpi = 2;
constexpr uint32_t kPairDepth = 5, kPairStage = 2 * kSlotA, kPairBN = 256, kPairEpiWarps = 8;
// behind the ring: two boxes for every epilogue warp (of the output, or of the output and the slopes), barriers
constexpr uint32_t kPairSmem = 1024 + kPairDepth * kPairStage + kPairEpiWarps * 2 * kBoxBytes + (2 * kPairDepth + 5 + 2 * kPairEpiWarps) * 8 + 16;
static_assert(kPairSmem <= 232448, "shared memory of an SM");

template <typename T>
__global__ void __launch_bounds__(kPairThreads, 1)
product_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ Maps maps,
                    const Product p, const Epilogue e)
{
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (smem - ptx::smem_u32(smem_raw));
    constexpr uint32_t kOffBoxes = kPairDepth * kPairStage;
    uint64_t* full = reinterpret_cast<uint64_t*>(gen + kOffBoxes + kPairEpiWarps * 2 * kBoxBytes);       // even CTA: both CTAs' operands have landed
    uint64_t* drained = full + kPairDepth;           // each CTA: the products that read a ring position are done
    uint64_t* tmem_full = drained + kPairDepth;      // each CTA, per accumulator: complete
    uint64_t* tmem_empty = tmem_full + 2;            // even CTA, per accumulator: read by the epilogue warps of both
    uint64_t* landed = tmem_empty + 2;               // [epilogue warp][2] residual of a box
    uint64_t* settled = landed + 2 * kPairEpiWarps;  // even CTA: the products have ended, after a wait that expired
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(settled + 1);
    volatile uint32_t* abort_flag = tmem_slot + 1;

    const uint32_t warp = ptx::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const uint32_t rank = ptx::cluster_cta_rank(), pair_id = ptx::cluster_id_x(), num_pairs = ptx::num_clusters_x();
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < kPairDepth; ++i) { ptx::mbar_init(full + i, 1); ptx::mbar_init(drained + i, 1); }
        for (uint32_t i = 0; i < 2; ++i) { ptx::mbar_init(tmem_full + i, 1); ptx::mbar_init(tmem_empty + i, 2 * kPairEpiWarps); }
        for (uint32_t i = 0; i < 2 * kPairEpiWarps + 1; ++i) ptx::mbar_init(landed + i, 1);
        *abort_flag = 0;
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&tm_a);
        ptx::prefetch_tensormap(&tm_b);
    }
    if (warp == 1) ptx::tmem_alloc_pair<512>(tmem_slot);
    ptx::tcgen05_fence_before_sync();
    ptx::cluster_sync();
    ptx::tcgen05_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    ptx::grid_dependency_wait();

    const uint32_t tiles = p.tiles_a * p.tiles_b;
    bool ok = true;
    auto give_up = [&] {
        *abort_flag = 1;
        if (p.status != nullptr) atomicOr(p.status, 1);
        ok = false;
    };
    if (warp == 0) {
        const uint32_t issue = ptx::elect_one();
        const uint32_t full_even = ptx::map_to_cta(ptx::smem_u32(full), 0);
        Ring r;
        uint32_t loaded = 0;                         // ring positions with copies in them
        for (uint32_t tile = pair_id; ok && tile < tiles; tile += num_pairs) {
            uint32_t a_blk, b_blk;
            gemm::tile_coords(tile, p.tiles_a, p.tiles_b, 8, a_blk, b_blk);
            const uint32_t a0 = (a_blk * 2 + rank) * BM, b0 = b_blk * kPairBN + rank * (kPairBN / 2);
            for (uint32_t kb = 0; kb < p.k_blocks; ++kb) {
                if (!ptx::all_lanes(ptx::mbar_wait_budget(drained + r.slot, r.phase ^ 1, abort_flag, p.budget))) { give_up(); break; }
                // the even CTA announces the bytes of both; the odd CTA's complete on its barrier
                if (rank == 0) ptx::mbar_arrive_expect_tx(full + r.slot, 2 * kPairStage, issue);
                uint8_t* to = gen + r.slot * kPairStage;
                const uint32_t bar = full_even + r.slot * 8;
                load_tile<BM>(to, p.a_mn, a0, kb, [&](uint8_t* dst, uint32_t c0, uint32_t c1) { ptx::tma_load_2d_pair(dst, &tm_a, bar, c0, c1, issue); });
                load_tile<BM>(to + kSlotA, p.b_mn, b0, kb, [&](uint8_t* dst, uint32_t c0, uint32_t c1) { ptx::tma_load_2d_pair(dst, &tm_b, bar, c0, c1, issue); });
                r.advance<kPairDepth>();
                loaded = min(loaded + 1, kPairDepth);
            }
        }
        ptx::grid_launch_dependents();
        if (ok && !gemm::drain_ring<kPairDepth>(r, [&](uint32_t i, uint32_t parity) {
                return ptx::all_lanes(ptx::mbar_wait_budget(drained + i, parity, abort_flag, p.budget)); })) give_up();
        // (the odd CTA's copies complete on the even one's barriers, and it cannot leave before that one; any that the even CTA has not
        // announced are as old as the wait that ran out in the odd one)
        if (!ok && rank == 0) {
            const long long until = clock64() + p.budget;
            for (uint32_t i = 0; i < loaded; ++i) {  // backwards from the next position: the last use of each
                if (r.slot == 0) { r.slot = kPairDepth; r.phase ^= 1; }
                --r.slot;
                ptx::mbar_settle(full + r.slot, r.phase, until);
            }
            __syncwarp();
        }
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t issue = ptx::elect_one();
            const uint32_t idesc = ptx::make_idesc_f16(2 * BM, kPairBN, std::is_same<T, __nv_bfloat16>::value, p.a_mn, p.b_mn);
            constexpr uint16_t kBoth = 3;
            Ring r;
            uint32_t n = 0;
            for (uint32_t tile = pair_id; ok && tile < tiles && p.withhold != kProducts; tile += num_pairs, ++n) {
                const uint32_t acc = n & 1;
                if (!ptx::all_lanes(ptx::mbar_wait_budget(tmem_empty + acc, ((n >> 1) & 1) ^ 1, abort_flag, p.budget))) { give_up(); break; }
                ptx::tcgen05_fence_after_sync();
                for (uint32_t kb = 0; kb < p.k_blocks; ++kb) {
                    if (!ptx::all_lanes(ptx::mbar_wait_budget(full + r.slot, r.phase, abort_flag, p.budget))) { give_up(); break; }
                    ptx::tcgen05_fence_after_sync();
                    const uint32_t at = smem + r.slot * kPairStage;
#pragma unroll
                    for (uint32_t s = 0; s < BK / 16; ++s)
                        ptx::tcgen05_mma_f16_pair(tmem + acc * kPairBN, operand_desc(at, p.a_mn, s), operand_desc(at + kSlotA, p.b_mn, s), idesc, kb | s, issue);
                    ptx::tcgen05_commit_pair(drained + r.slot, kBoth, issue);
                    r.advance<kPairDepth>();
                }
                if (ok) ptx::tcgen05_commit_pair(tmem_full + acc, kBoth, issue);
            }
            if (!ok || !ptx::all_lanes(*abort_flag == 0)) {
                ptx::tcgen05_commit_pair(settled, 1, issue);
                ptx::mbar_settle(settled, 0, clock64() + p.budget);
                __syncwarp();
            }
        }
    } else {
        const uint32_t quad = warp & 3, half = (warp - kPairFirstEpi) >> 2;   // its lanes; columns [128 half, 128 half + 128) of the tile
        const uint32_t tmem_empty_even = ptx::map_to_cta(ptx::smem_u32(tmem_empty), 0);
        const uint32_t boxes = smem + kOffBoxes + (warp - kPairFirstEpi) * 2 * kBoxBytes;
        const bool both = e.slopes != nullptr;       // the second buffer takes the slopes
        const float factor = e.scale != nullptr ? *e.scale : 1.0f;
        constexpr uint32_t kBoxColumns = kBox<T>;
        Stage<T, T> stage{boxes, both ? 0u : kBoxBytes, boxes + kBoxBytes, 0u, landed + 2 * (warp - kPairFirstEpi), 0, &maps, p.budget, factor, 0,
                          p.withhold == kResiduals};
        uint32_t n = 0;
        for (uint32_t tile = pair_id; tile < tiles; tile += num_pairs, ++n) {
            const uint32_t acc = n & 1;
            uint32_t a_blk, b_blk;
            gemm::tile_coords(tile, p.tiles_a, p.tiles_b, 8, a_blk, b_blk);
            const uint32_t row0 = (a_blk * 2 + rank) * BM + quad * 32, col0 = b_blk * kPairBN + half * 128;
            const bool wanted = row0 < e.rows && col0 < e.cols, second = col0 + kBoxColumns < e.cols;
            if (e.staged && wanted && ok) {
                stage.reclaim(lane);
                if (e.residual != nullptr) {
                    stage.request(0, col0, row0, lane);
                    if (second && !both) stage.request(1, col0 + kBoxColumns, row0, lane);
                }
            }
            if (ok && !ptx::all_lanes(ptx::mbar_wait_relaxed(tmem_full + acc, (n >> 1) & 1, abort_flag, 50, p.budget))) give_up();
            ptx::tcgen05_fence_after_sync();
            const uint32_t taddr = tmem + ((quad * 32) << 16) + acc * kPairBN + half * 128;
            uint32_t done = 0;                       // of the 128 columns, those that have left
            if (e.staged) {
#pragma unroll 1
                for (uint32_t box = 0; wanted && ok && box < (second ? 2u : 1u); ++box) {
                    if (box == 1 && both) {
                        stage.reclaim(lane);
                        if (e.residual != nullptr) stage.request(1, col0 + kBoxColumns, row0, lane);
                    }
                    if (!stage.finish(taddr + box * kBoxColumns, box, col0 + box * kBoxColumns, row0, lane, e, abort_flag)) give_up();
                    else done += kBoxColumns;
                }
                if (!ok) stage.settle();
            }
            if (wanted && (!e.staged || !ok)) {
#pragma unroll 1
                for (uint32_t c = done; c < 128; c += 32) {
                    if (col0 + c >= e.cols) break;
                    float v[32];
                    load_accumulators(taddr + c, v);
                    if (!ok) {
#pragma unroll
                        for (uint32_t i = 0; i < 32; ++i) v[i] = kNan;
                    }
                    transpose(v, lane);
                    finish<T, T>(v, row0, 32, col0 + c + lane, e, factor);
                }
            }
            if (!ok) continue;
            ptx::tcgen05_fence_before_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive_remote(tmem_empty_even + acc * 8);
        }
        if (lane == 0) ptx::bulk_wait();
    }
    // neither CTA leaves, or gives up its tensor memory, while the other can still signal it or read its operands
    ptx::tcgen05_fence_before_sync();
    ptx::cluster_sync();
    if (warp == 1) {
        ptx::tcgen05_fence_after_sync();
        ptx::tmem_dealloc_pair<512>(tmem);
    }
}

// ---- host: which kernel, which tiles -----------------------------------------------------------------------------------

template <typename T>
constexpr CUtensorMapDataType kMapType = std::is_same<T, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;

// Map of an operand with `rows` rows over a contraction of `k`; box: `tile` rows x 64, or 64 x 64 where memory runs along the rows.
template <typename T>
int operand_map(CUtensorMap* map, const void* base, int64_t ld, bool mn_major, uint64_t rows, uint64_t k, uint32_t tile)
{
    return host::encode_tensor_map_2d(map, kMapType<T>, 2, base, mn_major ? rows : k, mn_major ? k : rows, static_cast<uint64_t>(ld) * 2, BK,
                                      mn_major ? 64 : tile, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Maps of what the epilogue moves by TMA, if it can.
template <typename T, typename D>
int output_maps(Maps* maps, Epilogue* e)
{
    constexpr bool kFloat = std::is_same<D, float>::value;
    auto aligned = [](const void* p, int64_t ld, int64_t size) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld * size % 16 == 0; };
    *maps = Maps{};
    e->staged = aligned(e->d, e->ldd, sizeof(D)) && (e->residual == nullptr || aligned(e->residual, e->ldr, sizeof(D))) &&
                (e->slopes == nullptr || (!kFloat && aligned(e->slopes, e->lds, 2)));
    if (!e->staged) return NVFP4_OK;
    auto map = [&](CUtensorMap* m, CUtensorMapDataType type, const void* base, int64_t ld) {
        return host::encode_tensor_map_2d(m, type, sizeof(D), base, e->cols, e->rows, static_cast<uint64_t>(ld) * sizeof(D), kBox<D>, 32,
                                          CU_TENSOR_MAP_SWIZZLE_128B);
    };
    constexpr CUtensorMapDataType kType = kFloat ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : kMapType<T>;
    if (int rc = map(&maps->d, kType, e->d, e->ldd)) return rc;
    if (e->residual != nullptr)
        if (int rc = map(&maps->residual, kType, e->residual, e->ldr)) return rc;
    if (e->slopes != nullptr)
        if (int rc = map(&maps->slopes, CU_TENSOR_MAP_DATA_TYPE_UINT16, e->slopes, e->lds)) return rc;
    return NVFP4_OK;
}

struct Operands {
    const void* a; int64_t lda; bool a_mn; uint32_t rows_a;
    const void* b; int64_t ldb; bool b_mn; uint32_t rows_b;
    uint32_t k;
    int32_t* status;
    long long budget = ptx::kWaitBudgetCycles;
    uint32_t withhold = kNothing;
};

// CTAs that find an SM of their own: clusters of four and eight do not divide the SMs of every GPC.
int ctas_at_once(uint32_t splits_log2, int num_sms) { return splits_log2 < 2 || num_sms < 2 ? num_sms : num_sms * 13 / 15; }

template <typename T, typename D, uint32_t BN, bool kSwap, bool kLong = false>
int launch_tiles(const Operands& o, Epilogue e, uint32_t splits_log2, int num_sms, cudaStream_t stream)
{
    CUtensorMap tm_a, tm_b;
    Maps maps{};
    if constexpr (!kSwap)
        if (splits_log2 == 0)
            if (int rc = output_maps<T, D>(&maps, &e)) return rc;
    if (int rc = operand_map<T>(&tm_a, o.a, o.lda, o.a_mn, o.rows_a, o.k, BM)) return rc;
    if (int rc = operand_map<T>(&tm_b, o.b, o.ldb, o.b_mn, o.rows_b, o.k, BN)) return rc;
    Product p{};
    p.tiles_a = (o.rows_a + BM - 1) / BM;
    p.tiles_b = (o.rows_b + BN - 1) / BN;
    p.k_blocks = (o.k + BK - 1) / BK;
    p.splits_log2 = splits_log2;
    p.a_mn = o.a_mn;
    p.b_mn = o.b_mn;
    p.status = o.status;
    p.budget = o.budget;
    p.withhold = o.withhold;
    const uint64_t ctas = static_cast<uint64_t>(p.tiles_a) * p.tiles_b << splits_log2;
    // One CTA to an SM: its ring may fill the shared memory; more: two share it.  Clusters of eight, too, leave room for a second CTA: of
    // those that fill their SMs not even sixteen run at once (256 x 128 x 4096, 16 of them: 8.9 us, a second wave; 5.7 so).
    const uint32_t budget = ctas <= static_cast<uint64_t>(ctas_at_once(splits_log2, num_sms)) && splits_log2 < 3 ? kTileSmem : 112 * 1024;
    p.depth = kMaxDepth;
    while (p.depth > 2 && tile_smem(BN, p.depth, 1u << splits_log2) > budget) --p.depth;
    int dev = 0;
    NVFP4_CUDA_CHECK(cudaGetDevice(&dev));
    static bool attr_set[host::kMaxDevices] = {};
    if (!attr_set[dev]) {
        NVFP4_CUDA_CHECK(cudaFuncSetAttribute(product_kernel<T, D, BN, kSwap, kLong>, cudaFuncAttributeMaxDynamicSharedMemorySize, kTileSmem));
        attr_set[dev] = true;
    }
    NVFP4_REQUIRE(ctas <= INT32_MAX, "too many tiles (%llu)", static_cast<unsigned long long>(ctas));
    return host::launch_kernel_cluster(product_kernel<T, D, BN, kSwap, kLong>, dim3(static_cast<unsigned>(ctas)), dim3(kTileThreads),
                                       tile_smem(BN, p.depth, 1u << splits_log2), stream, true, 1u << splits_log2, tm_a, tm_b, maps, p, e);
}

template <typename T>
int launch_pairs(const Operands& o, Epilogue e, int num_sms, cudaStream_t stream)
{
    CUtensorMap tm_a, tm_b;
    Maps maps;
    if (int rc = output_maps<T, T>(&maps, &e)) return rc;
    if (int rc = operand_map<T>(&tm_a, o.a, o.lda, o.a_mn, o.rows_a, o.k, BM)) return rc;
    if (int rc = operand_map<T>(&tm_b, o.b, o.ldb, o.b_mn, o.rows_b, o.k, BM)) return rc;
    Product p{};
    p.tiles_a = (o.rows_a + 2 * BM - 1) / (2 * BM);
    p.tiles_b = (o.rows_b + kPairBN - 1) / kPairBN;
    p.k_blocks = (o.k + BK - 1) / BK;
    p.a_mn = o.a_mn;
    p.b_mn = o.b_mn;
    p.status = o.status;
    p.budget = o.budget;
    p.withhold = o.withhold;
    int dev = 0;
    NVFP4_CUDA_CHECK(cudaGetDevice(&dev));
    static bool attr_set[host::kMaxDevices] = {};
    if (!attr_set[dev]) {
        NVFP4_CUDA_CHECK(cudaFuncSetAttribute(product_pair_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem));
        attr_set[dev] = true;
    }
    const uint64_t tiles = static_cast<uint64_t>(p.tiles_a) * p.tiles_b, pairs = static_cast<uint64_t>(num_sms / 2);
    NVFP4_REQUIRE(tiles <= INT32_MAX, "too many tiles (%llu)", static_cast<unsigned long long>(tiles));
    return host::launch_kernel_cluster(product_pair_kernel<T>, dim3(static_cast<unsigned>(2 * (tiles < pairs ? tiles : pairs))), dim3(kPairThreads),
                                       kPairSmem, stream, true, 2u, tm_a, tm_b, maps, p, e);
}

// Which kernel, which tile and how many CTAs to a tile: the form with the smallest estimate, in microseconds,
//     start + splitting + |(K blocks of a CTA * time of one * CTAs to an SM, operands / HBM)|
// Measured on a B200 (BF16, alone on the GPU): a block of 64 of K takes a CTA 0.16 us at BN = 16 to 0.235 at 128, the time its bytes take into
// one SM, and a CTA pair 0.29, the time of its products.  What is left at K -> 0 is the start.  Adding partial sums over a
// cluster costs by the tile's columns.  Estimates are within a tenth or so of what was measured: 64 x 4096 x 4096 (swap 64 / 4) 10.4 for
// 11.1, 256 x 1024 x 4096 (swap 64 / 4) 7.9 for 9.9, 512 x 4096 x 4096 (normal 128) 18 for 19, 1024 x 4096 x 4096 (pairs) 24 for 26.  Against the
// best of all forms by measurement the choice loses up to 8 % over 1 to 2048 rows, 128 to 4096 columns, K 1024 and 4096.
// Tiles of 128 columns with an FP32 output have an SM to themselves (the sums in their registers): of several, nobody's products run under
// another's sums and stores, and a block costs 0.41 us.  8192 x 4096 on swapped tiles of 64 / tiles of 128: K = 64 47 / 63 us, 1024 110 / 124, 4096 321 / 354.
struct Form {
    enum Kind { kSwap, kNormal, kPairs } kind;
    uint32_t bn, splits_log2;
};
struct TileCost {
    uint32_t bn;
    double block, start_swap, start_normal, split;
};
constexpr TileCost kTileCosts[] = {{16, 0.16, 2.5, 0, 0.45}, {32, 0.17, 2.5, 0, 1.5}, {64, 0.20, 2.4, 2.6, 2.3}, {128, 0.235, 3.3, 3.0, 5.0}};
Form choose_form(const Operands& o, bool wide, int num_sms)
{
    const double hbm = (static_cast<double>(o.rows_a) + o.rows_b) * o.k * 2 / 6.0e6;
    const uint32_t k_blocks = (o.k + BK - 1) / BK;
    auto blocks = [](uint32_t rows, uint32_t tile) { return (rows + tile - 1) / tile; };
    Form best{Form::kNormal, 128, 0};
    double least = 1e30;
    auto consider = [&](Form::Kind kind, uint64_t tiles, const TileCost& c, double start, uint32_t most_log2) {
        for (uint32_t s = 0; s <= most_log2 && (s == 0 || k_blocks >> s >= 2); ++s) {
            const uint64_t at_once = ctas_at_once(s, num_sms);
            const double resident = static_cast<double>(((tiles << s) + at_once - 1) / at_once);
            const bool alone = wide && c.bn == 128 && resident > 1;
            const double loop = ((k_blocks + (1u << s) - 1) >> s) * (alone ? 0.41 : c.block) * resident;
            const double t = start * (alone ? resident : resident > 2 ? resident / 2 : 1) + (s ? c.split : 0) + std::sqrt(loop * loop + hbm * hbm);
            if (t < least) { least = t; best = Form{kind, c.bn, s}; }
            if (tiles << (s + 1) > 2 * static_cast<uint64_t>(num_sms)) break;
        }
    };
    for (const TileCost& c : kTileCosts) {
        if (!o.a_mn && !o.b_mn) consider(Form::kSwap, static_cast<uint64_t>(blocks(o.rows_b, BM)) * blocks(o.rows_a, c.bn), c, c.start_swap, c.bn <= 32 ? 3 : 2);
        if (c.start_normal > 0) consider(Form::kNormal, static_cast<uint64_t>(blocks(o.rows_a, BM)) * blocks(o.rows_b, c.bn), c, c.start_normal, c.bn / 64);
    }
    if (!wide && num_sms >= 2) {
        const uint64_t tiles = static_cast<uint64_t>(blocks(o.rows_a, 2 * BM)) * blocks(o.rows_b, kPairBN), pairs = num_sms / 2;
        const double loop = static_cast<double>((tiles + pairs - 1) / pairs) * k_blocks * 0.29, t = 5.0 + std::sqrt(loop * loop + hbm * hbm);
        if (t < least) best = Form{Form::kPairs, kPairBN, 0};
    }
    return best;
}

template <typename T, typename D>
int launch_tokens(const Operands& o, const Epilogue& e, int num_sms, cudaStream_t stream)
{
    // warps to a row: until there are sixteen to an SM, each with a batch of loads at least
    uint32_t warps_log2 = 0;
    while (warps_log2 < 3 && (static_cast<uint64_t>(o.rows_b) << warps_log2) < 16 * static_cast<uint64_t>(num_sms) && (o.k / 8 >> (warps_log2 + 1)) >= 32) ++warps_log2;
    const uint32_t rows = kTokenWarps >> warps_log2;
    auto kernel = o.rows_a == 1 ? token_kernel<T, D, 1> : token_kernel<T, D, 2>;
    return host::launch_kernel(kernel, dim3((o.rows_b + rows - 1) / rows), dim3(kTokenThreads), 0, stream, true, static_cast<const T*>(o.a), o.lda,
                               static_cast<const T*>(o.b), o.ldb, o.k, warps_log2, e);
}

// The output (rows_a, rows_b), of type D.
template <typename T, typename D>
int launch_product(const Operands& o, const Epilogue& e, int num_sms, cudaStream_t stream)
{
    if (o.rows_a <= 2 && !o.a_mn && !o.b_mn && static_cast<uint64_t>(o.rows_b) * o.k <= kTokenMostWeights) return launch_tokens<T, D>(o, e, num_sms, stream);
    const Form f = choose_form(o, !std::is_same<D, T>::value, num_sms);
    if constexpr (std::is_same<D, T>::value) {
        if (o.k >> f.splits_log2 > kLongestSum<T>) {         // CTAs of a cluster have sums of their own
            const uint64_t tiles = static_cast<uint64_t>((o.rows_a + BM - 1) / BM) * ((o.rows_b + 127) / 128);
            uint32_t splits_log2 = 0;
            while (splits_log2 < 2 && tiles << (splits_log2 + 1) <= static_cast<uint64_t>(ctas_at_once(splits_log2 + 1, num_sms))) ++splits_log2;
            return launch_tiles<T, D, 128, false, true>(o, e, splits_log2, num_sms, stream);
        }
    }
    if (f.kind == Form::kSwap) {                     // the weight's rows on the tensor memory's lanes
        const Operands s{o.b, o.ldb, false, o.rows_b, o.a, o.lda, false, o.rows_a, o.k, o.status, o.budget, o.withhold};
        switch (f.bn) {
            case 16: return launch_tiles<T, D, 16, true>(s, e, f.splits_log2, num_sms, stream);
            case 32: return launch_tiles<T, D, 32, true>(s, e, f.splits_log2, num_sms, stream);
            case 64: return launch_tiles<T, D, 64, true>(s, e, f.splits_log2, num_sms, stream);
            default: return launch_tiles<T, D, 128, true>(s, e, f.splits_log2, num_sms, stream);
        }
    }
    if constexpr (std::is_same<D, T>::value)
        if (f.kind == Form::kPairs) return launch_pairs<T>(o, e, num_sms, stream);
    return f.bn == 64 ? launch_tiles<T, D, 64, false>(o, e, f.splits_log2, num_sms, stream) : launch_tiles<T, D, 128, false>(o, e, f.splits_log2, num_sms, stream);
}

// ---- dz and the bias' gradient -----------------------------------------------------------------------------------------

// dz = dd * activation'(z), rounded once for the tensor cores, and per block of rows the sums of its columns before that rounding.
// A thread takes eight columns (16 bytes of the slopes and of dz, whose rows are padded to that) of every eighth row of its block's; a
// block 256 columns.  One pass over dd and the slopes, bound by their bytes.
// FP32 gradients of FP16 operands may lie outside of FP16: those of a mean over many tokens below its smallest number, where dz would be
// zero, others above its largest.  So every block leaves its largest finite |dz| in `peaks`, and a second pass, which is over at once if the
// largest of all is in [1/4, 65504], writes dz times a power of two that brings that to [2^14, 2^15), so that what is lost is 2^-39 of the
// largest; the products multiply their sums by that power's inverse, *scale.  (Training step of 4096 x 2048 x 2048 with silu in a graph: 158 -> 165 us
// with gradients that FP16 holds.)
__device__ __forceinline__ float dz_factor(float most)
{
    if (most == 0.0f || (most >= 0.25f && most <= 65504.0f)) return 1.0f;
    const int exponent = max(static_cast<int>(__float_as_uint(most) >> 23) - 127, -112);      // at most 2^126: its inverse is no subnormal number
    return __uint_as_float(static_cast<uint32_t>(127 + 14 - exponent) << 23);
}
constexpr int kGradThreads = 256, kGradColumns = 256, kGradRowLanes = 8;
enum DzPass { kOnlyPass, kFirstPass, kSecondPass };                          // (a 4099 x 4096 pass that need not look for the largest: 16.7 us for 18.9)
template <typename T, typename D, DzPass kPass>
__global__ void __launch_bounds__(kGradThreads)
linear_dz_kernel(const D* __restrict__ dd, int64_t ldd, bool wide, const int16_t* __restrict__ slopes, int64_t lds, T* __restrict__ dz, int64_t lddz, uint32_t rows,
                 uint32_t cols, uint32_t rows_each, float* __restrict__ sums, float* __restrict__ peaks, float* __restrict__ scale)
{
    __shared__ float part[kGradRowLanes][kGradColumns];
    const uint32_t group = threadIdx.x % 32, row_lane = threadIdx.x / 32;
    const uint32_t col0 = blockIdx.x * kGradColumns + group * 8;
    const uint32_t first = blockIdx.y * rows_each, last = min(rows, first + rows_each);
    ptx::grid_dependency_wait();
    float factor = 1.0f, most = 0.0f;
    __shared__ uint32_t largest[kGradRowLanes];
    // the largest of the block's numbers, none of them negative: their bits are in their order
    auto largest_of_block = [&](float v) {
        const uint32_t bits = __reduce_max_sync(kAll, __float_as_uint(v));
        if (threadIdx.x % 32 == 0) largest[row_lane] = bits;
        __syncthreads();
        return __uint_as_float(__reduce_max_sync(kAll, largest[threadIdx.x % kGradRowLanes]));
    };
    if constexpr (kPass == kSecondPass) {
        for (uint32_t i = threadIdx.x; i < gridDim.x * gridDim.y; i += kGradThreads) most = fmaxf(most, peaks[i]);
        factor = dz_factor(largest_of_block(most));
        if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *scale = 1.0f / factor;
        if (factor == 1.0f) return;
    }
    float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (col0 < cols) {
        const uint32_t here = min(8u, cols - col0);
        for (uint32_t r = first + row_lane; r < last; r += kGradRowLanes) {
            const D* from = dd + static_cast<int64_t>(r) * ldd + col0;
            alignas(16) D g[8];
            if (wide) {
#pragma unroll
                for (uint32_t i = 0; i < sizeof(g) / 16; ++i) reinterpret_cast<uint4*>(g)[i] = reinterpret_cast<const uint4*>(from)[i];
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) g[i] = i < here ? from[i] : from_float<D>(0.0f);
            }
            alignas(16) int16_t code[8];
            if (slopes != nullptr) *reinterpret_cast<uint4*>(code) = *reinterpret_cast<const uint4*>(slopes + static_cast<int64_t>(r) * lds + col0);
            alignas(16) T out[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                float v = to_float(g[i]);
                if (slopes != nullptr) v *= unpack_slope(code[i]);
                sum[i] += v;
                if constexpr (kPass == kSecondPass) v *= factor;
                if (kPass == kFirstPass && fabsf(v) < INFINITY && i < here) most = fmaxf(most, fabsf(v));
                out[i] = from_float<T>(v);
            }
            if (dz != nullptr) *reinterpret_cast<uint4*>(dz + static_cast<int64_t>(r) * lddz + col0) = *reinterpret_cast<const uint4*>(out);
        }
    }
    if constexpr (kPass == kFirstPass) {
        const float top = largest_of_block(most);
        if (threadIdx.x == 0) peaks[blockIdx.y * gridDim.x + blockIdx.x] = top;
    }
    if (kPass == kSecondPass || sums == nullptr) return;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) part[row_lane][group * 8 + i] = sum[i];
    __syncthreads();
    const uint32_t col = blockIdx.x * kGradColumns + threadIdx.x;
    if (col >= cols) return;
    float total = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < kGradRowLanes; ++i) total += part[i][threadIdx.x];
    sums[static_cast<int64_t>(blockIdx.y) * cols + col] = total;
}
template <typename T>
__global__ void __launch_bounds__(kGradThreads)
linear_db_kernel(const float* __restrict__ sums, uint32_t blocks, uint32_t cols, T* __restrict__ db)
{
    const uint32_t col = blockIdx.x * kGradThreads + threadIdx.x;
    ptx::grid_dependency_wait();
    if (col >= cols) return;
    float total = 0.0f;
    for (uint32_t b = 0; b < blocks; ++b) total += sums[static_cast<int64_t>(b) * cols + col];
    db[col] = from_float<T>(total);
}

template <typename T, typename D>
int launch_dz(const void* dd, int64_t ldd, const int16_t* slopes, int64_t lds, void* dz, int64_t lddz, void* db, uint32_t rows, uint32_t cols, float* scale,
              int num_sms, cudaStream_t stream)
{
    const unsigned columns = (cols + kGradColumns - 1) / kGradColumns;
    // about four blocks to an SM, at least eight rows to a block
    uint32_t blocks = (static_cast<uint32_t>(num_sms) * 4 + columns - 1) / columns;
    uint32_t rows_each = (rows + blocks - 1) / blocks;
    rows_each = (rows_each + kGradRowLanes - 1) / kGradRowLanes * kGradRowLanes;
    blocks = (rows + rows_each - 1) / rows_each;
    const bool wide = ((reinterpret_cast<uintptr_t>(dd) | static_cast<uintptr_t>(ldd * sizeof(D))) & 15u) == 0 && cols % 8 == 0;
    float *workspace = nullptr, *sums = nullptr, *peaks = nullptr;
    const size_t sum_words = db != nullptr ? static_cast<size_t>(blocks) * cols : 0, peak_words = scale != nullptr ? static_cast<size_t>(blocks) * columns : 0;
    if (sum_words + peak_words > 0) {
        int dev = 0;
        NVFP4_CUDA_CHECK(cudaGetDevice(&dev));
        cudaMemPool_t pool;
        if (int rc = host::workspace_pool(dev, &pool)) return rc;
        NVFP4_CUDA_CHECK(cudaMallocFromPoolAsync(reinterpret_cast<void**>(&workspace), (sum_words + peak_words) * sizeof(float), pool, stream));
        if (db != nullptr) sums = workspace;
        if (scale != nullptr) peaks = workspace + sum_words;
    }
    const dim3 grid(columns, blocks);
    auto pass = [&](auto kernel) {
        return host::launch_kernel(kernel, grid, dim3(kGradThreads), 0, stream, true, static_cast<const D*>(dd), ldd, wide, slopes, lds, static_cast<T*>(dz), lddz,
                                   rows, cols, rows_each, sums, peaks, scale);
    };
    int rc = NVFP4_OK;
    if (scale == nullptr) {
        rc = pass(linear_dz_kernel<T, D, kOnlyPass>);
    } else if constexpr (std::is_same<T, __half>::value && std::is_same<D, float>::value) {
        rc = pass(linear_dz_kernel<T, D, kFirstPass>);
        if (rc == NVFP4_OK) rc = pass(linear_dz_kernel<T, D, kSecondPass>);
    }
    if (rc == NVFP4_OK && db != nullptr)
        rc = host::launch_kernel(linear_db_kernel<T>, dim3((cols + kGradThreads - 1) / kGradThreads), dim3(kGradThreads), 0, stream, true, sums, blocks, cols,
                                 static_cast<T*>(db));
    if (workspace != nullptr) cudaFreeAsync(workspace, stream);
    return rc;
}

}  // namespace

template <typename T>
static int product(const Operands& o, const Epilogue& e, bool out32, int num_sms, cudaStream_t stream)
{
    return out32 ? launch_product<T, float>(o, e, num_sms, stream) : launch_product<T, T>(o, e, num_sms, stream);
}

int launch_linear(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* residual, int64_t ldr, void* d, int64_t ldd,
                  int16_t* slopes, int64_t lds, int M, int N, int K, bool bf16, bool out32, int activation, int32_t* status, int num_sms,
                  cudaStream_t stream, int64_t budget, bool withhold_residuals)
{
    Operands o{x, ldx, false, static_cast<uint32_t>(M), w, ldw, false, static_cast<uint32_t>(N), static_cast<uint32_t>(K), status};
    if (budget > 0) {                                // the test of waits that run out
        o.budget = budget;
        o.withhold = withhold_residuals ? kResiduals : kProducts;
    }
    if (activation == NVFP4_ACTIVATION_NONE) slopes = nullptr;
    const Epilogue e{d, ldd, slopes, lds, bias, residual, ldr, static_cast<uint32_t>(M), static_cast<uint32_t>(N), activation, nullptr, false};
    return bf16 ? product<__nv_bfloat16>(o, e, out32, num_sms, stream) : product<__half>(o, e, out32, num_sms, stream);
}

int launch_linear_dz(const void* dd, int64_t ldd, bool dd32, const int16_t* slopes, int64_t lds, void* dz, int64_t lddz, void* db, int M, int N,
                     bool bf16, float* scale, int num_sms, cudaStream_t stream)
{
    const uint32_t m = static_cast<uint32_t>(M), n = static_cast<uint32_t>(N);
    if (bf16)
        return dd32 ? launch_dz<__nv_bfloat16, float>(dd, ldd, slopes, lds, dz, lddz, db, m, n, scale, num_sms, stream)
                    : launch_dz<__nv_bfloat16, __nv_bfloat16>(dd, ldd, slopes, lds, dz, lddz, db, m, n, scale, num_sms, stream);
    return dd32 ? launch_dz<__half, float>(dd, ldd, slopes, lds, dz, lddz, db, m, n, scale, num_sms, stream)
                : launch_dz<__half, __half>(dd, ldd, slopes, lds, dz, lddz, db, m, n, scale, num_sms, stream);
}

int launch_linear_dx(const void* dz, int64_t lddz, const void* w, int64_t ldw, void* dx, int64_t lddx, int M, int N, int K, bool bf16,
                     const float* scale, int32_t* status, int num_sms, cudaStream_t stream)
{
    const Operands o{dz, lddz, false, static_cast<uint32_t>(M), w, ldw, true, static_cast<uint32_t>(K), static_cast<uint32_t>(N), status};
    const Epilogue e{dx, lddx, nullptr, 0, nullptr, nullptr, 0, static_cast<uint32_t>(M), static_cast<uint32_t>(K), NVFP4_ACTIVATION_NONE, scale, false};
    return bf16 ? product<__nv_bfloat16>(o, e, false, num_sms, stream) : product<__half>(o, e, false, num_sms, stream);
}

int launch_linear_dw(const void* dz, int64_t lddz, const void* x, int64_t ldx, void* dw, int64_t lddw, int M, int N, int K, bool bf16,
                     const float* scale, int32_t* status, int num_sms, cudaStream_t stream)
{
    const Operands o{dz, lddz, true, static_cast<uint32_t>(N), x, ldx, true, static_cast<uint32_t>(K), static_cast<uint32_t>(M), status};
    const Epilogue e{dw, lddw, nullptr, 0, nullptr, nullptr, 0, static_cast<uint32_t>(N), static_cast<uint32_t>(K), NVFP4_ACTIVATION_NONE, scale, false};
    return bf16 ? product<__nv_bfloat16>(o, e, false, num_sms, stream) : product<__half>(o, e, false, num_sms, stream);
}

}  // namespace nvfp4
