// Rows of 16-bit floats to rows of 8-bit floats with one FP32 scale each, optionally gathered by an index vector:
//
//     m_r  = max(2^-80, max over the finite |x[i_r][k]|)          i_r = index[r], or r without an index
//     s_r  = m_r / top                                            top = 448 (E4M3), 57344 (E5M2)
//     q[r][k] = RNE(x[i_r][k] * top / m_r)                        infinities saturate, a NaN stays a NaN
//
// so that q * s is the row again.  The operands of the row-scaled products (a_row_scale / b_row_scale) are made by it;
// i_r outside the source is a row of zeros (the padding of a fixed-capacity expert).  The floor 2^-80 keeps s_r and its
// reciprocal normal numbers for rows of zeros.
//
// Bound by HBM: 2 bytes read and 1 written per element.  A row stays in registers between the maximum and the
// conversion, so it is read once: one warp (four rows to a block, no barrier) or a block of 128 to 512 threads holds it, 4 to 12
// 16-byte pieces per thread, all loads in flight at once.  Rows of more than 16384 elements and rows that are not 16-byte aligned
// take the two-pass form at the end.
//
// Measured: 8192 rows of 4096 gathered into 16384 (67 MB read, 67 MB written) 25.2 us in a graph, 5.3 TB/s, 0.81 of a plain
// copy's rate; the two-pass form 150 us.  What is left is issue slots, about eight instructions per element.  One row of 8192:
// 1.6 us in a graph.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <cstdint>
#include "ptx_sm100.cuh"

namespace b200fp8 {

struct QuantizeArgs {
    const uint16_t* x;
    long long ldx;       // elements
    int source_rows;
    const int* index;    // source row of each output row, or nullptr
    int rows, k;
    uint8_t* q;
    long long ldq;
    float* scale;
    int q_dtype;         // 0 E4M3, 1 E5M2
};

constexpr float kQuantizeLeast = 8.271806125530277e-25f;    // 2^-80

constexpr int kQuantizeMostPieces = 2048;                   // of eight elements: the longest row that a block holds in registers

template <bool BF16>
__device__ __forceinline__ float2 unpack16(uint32_t w) {
    if constexpr (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// The quotient x / m * top, rounded so that its conversion to 8 bits is that of the exact quotient.  x and m have at most
// 11 significant bits, so an inexact quotient lies at least 2^-17 (relative) away from a border between two 8-bit values
// and any error below that is harmless; a quotient that IS such a border (a tie) has to come out exactly.  One
// residual step after the multiplication by the reciprocal does that: the residual of a product that should have been
// exact is computed without error by the fused multiply-add, and adding it lands on the representable quotient.
// x carries 2^-3, so that 1 / m is a normal number for every finite m while the residual of E5M2's smallest tie in a row of
// the least m, 2^-148, is still a number (with 2^-20 ties were lost for m of 2^-80 to 2^-76); top = 0.875 * 2^9 or 0.875 * 2^16.
struct Quotient {
    static constexpr float kUp = 0.125f;
    float m, back, inverse;
    __device__ __forceinline__ Quotient(float most, float two_power) : m(most) {
        const float a = most * kUp;
        back = a / two_power;
        inverse = two_power * __frcp_rn(a);
    }
    // an infinity as the largest finite magnitude, which becomes +-top; a NaN passes
    __device__ __forceinline__ float finite(float x) const { return fabsf(x) > m ? copysignf(m, x) : x; }
    __device__ __forceinline__ float operator()(float x) const {
        const float u = x * (0.875f * kUp);                      // exact: three more bits
        const float z = u * inverse;
        return fmaf(fmaf(-z, back, u), inverse, z);
    }
};

// The same on two numbers at once: the packed FP32 instructions round each half as the single ones do.
struct Quotient2 {
    uint64_t unit, minus_back, inverse;
    static __device__ __forceinline__ uint64_t twice(float v) { return pack(make_float2(v, v)); }
    static __device__ __forceinline__ uint64_t pack(float2 v) {
        uint64_t r;
        asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
        return r;
    }
    __device__ __forceinline__ explicit Quotient2(const Quotient& q)
        : unit(twice(0.875f * Quotient::kUp)), minus_back(twice(-q.back)), inverse(twice(q.inverse)) {}
    __device__ __forceinline__ float2 operator()(float2 x) const {
        uint64_t u, z, r;
        asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(u) : "l"(pack(x)), "l"(unit));
        asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(z) : "l"(u), "l"(inverse));
        asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(z), "l"(minus_back), "l"(u));
        asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(r), "l"(inverse), "l"(z));
        float2 v;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(r));
        return v;
    }
};

template <bool BF16>
__device__ __forceinline__ float finite_abs(uint16_t bits) {
    const uint16_t mag = bits & 0x7FFFu;
    if (mag >= (BF16 ? 0x7F80u : 0x7C00u)) return 0.0f;
    return BF16 ? __uint_as_float(static_cast<uint32_t>(mag) << 16) : __half2float(__ushort_as_half(mag));
}

// the largest of non-negative numbers (ordered like their bit patterns) over a warp, over a block
__device__ __forceinline__ float warp_max(float v) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v))); }
__device__ __forceinline__ float block_max(float v, float* shared) {
    v = warp_max(v);
    const int warps = blockDim.x >> 5;
    if (warps == 1) return v;
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_max(static_cast<int>(threadIdx.x & 31) < warps ? shared[threadIdx.x & 31] : 0.0f);
}

// The larger magnitude of two pairs of 16-bit floats; a NaN loses against a number.
template <bool BF16>
__device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b) {
    b &= 0x7FFF7FFFu;
    if constexpr (BF16) {
        const __nv_bfloat162 r = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    } else {
        const __half2 r = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
}

// THREADS == 32: four rows to a block of four warps; else one row to a block.  PIECES of 16 bytes per thread.
template <bool BF16, int Q, int THREADS, int PIECES>
__global__ void __launch_bounds__(THREADS == 32 ? 128 : THREADS) quantize_rows_kernel(const QuantizeArgs args) {
    __shared__ float shared[THREADS / 32];
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const long long r = THREADS == 32 ? blockIdx.x * 4ll + (threadIdx.x >> 5) : blockIdx.x;
    if (THREADS == 32 && r >= args.rows) return;
    const int t = THREADS == 32 ? threadIdx.x & 31 : threadIdx.x;
    const int pieces = args.k / 8;
    const int src = args.index ? __ldg(args.index + r) : static_cast<int>(r);
    const bool have = src >= 0 && src < args.source_rows;
    const uint4* x = reinterpret_cast<const uint4*>(args.x + static_cast<long long>(have ? src : 0) * args.ldx);
    uint4 v[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        v[i] = make_uint4(0u, 0u, 0u, 0u);
        if (have && t + i * THREADS < pieces) v[i] = __ldg(x + t + i * THREADS);
    }
    uint32_t both = 0u;
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
        both = max_abs2<BF16>(max_abs2<BF16>(max_abs2<BF16>(max_abs2<BF16>(both, v[i].x), v[i].y), v[i].z), v[i].w);
    const float2 two = unpack16<BF16>(both);
    auto across = [&](float m) {
        if constexpr (THREADS == 32) return warp_max(m);
        else return block_max(m, shared);
    };
    float most = across(fmaxf(two.x, two.y));
    const bool infinite = isinf(most);
    if (infinite) {                                               // rare: the largest finite magnitude, one element at a time
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) m = fmaxf(m, fmaxf(finite_abs<BF16>(static_cast<uint16_t>(w[j])), finite_abs<BF16>(static_cast<uint16_t>(w[j] >> 16))));
        }
        if constexpr (THREADS != 32) __syncthreads();            // everybody has read the first maximum
        most = across(m);
    }
    most = fmaxf(most, kQuantizeLeast);
    const Quotient quotient(most, Q == 0 ? 512.0f : 65536.0f);
    uint2* q = reinterpret_cast<uint2*>(args.q + r * args.ldq);
    auto convert = [&](auto value) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            if (t + i * THREADS >= pieces) break;
            const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
            uint32_t b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                b[j] = __nv_cvt_float2_to_fp8x2(value(unpack16<BF16>(w[j])), __NV_SATFINITE, Q == 0 ? __NV_E4M3 : __NV_E5M2);
            }
            q[t + i * THREADS] = make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
        }
    };
    // the comparison with the maximum would be a third of the instructions of a row without infinities
    const Quotient2 quotient2(quotient);
    if (infinite) convert([&](float2 f) { return quotient2(make_float2(quotient.finite(f.x), quotient.finite(f.y))); });
    else convert([&](float2 f) { return quotient2(f); });
    if (t == 0) args.scale[r] = most / (Q == 0 ? 448.0f : 57344.0f);
}

// One block per row, any K and any alignment of 2 / 1 bytes: two passes over the row.
template <bool BF16>
__global__ void __launch_bounds__(256) quantize_rows_any_kernel(const QuantizeArgs args) {
    __shared__ float shared[8];
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int r = blockIdx.x;
    const int src = args.index ? args.index[r] : r;
    const bool have = src >= 0 && src < args.source_rows;
    const uint16_t* x = args.x + static_cast<long long>(have ? src : 0) * args.ldx;
    uint8_t* q = args.q + static_cast<long long>(r) * args.ldq;
    float most = 0.0f;
    if (have)
        for (int k = threadIdx.x; k < args.k; k += blockDim.x) most = fmaxf(most, finite_abs<BF16>(x[k]));
    most = fmaxf(block_max(most, shared), kQuantizeLeast);
    const Quotient quotient(most, args.q_dtype == 0 ? 512.0f : 65536.0f);
    const __nv_fp8_interpretation_t kind = args.q_dtype == 0 ? __NV_E4M3 : __NV_E5M2;
    for (int k = threadIdx.x; k < args.k; k += blockDim.x) {
        const float v = have ? unpack16<BF16>(x[k]).x : 0.0f;
        q[k] = __nv_cvt_float_to_fp8(quotient(quotient.finite(v)), __NV_SATFINITE, kind);
    }
    if (threadIdx.x == 0) args.scale[r] = most / (args.q_dtype == 0 ? 448.0f : 57344.0f);
}

}  // namespace b200fp8
