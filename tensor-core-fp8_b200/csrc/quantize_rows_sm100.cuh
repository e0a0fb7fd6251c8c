// Rows of 16-bit floats to rows of 8-bit floats with one FP32 scale each, optionally gathered by an index vector:
//
//     m_r  = max(2^-80, max over the finite |x[i_r][k]|)          i_r = index[r], or r without an index
//     s_r  = m_r / top                                            top = 448 (E4M3), 57344 (E5M2)
//     q[r][k] = RNE(x[i_r][k] / m_r * top)                        infinities saturate, a NaN stays a NaN
//
// so that q * s is the row again.  The operands of the row-scaled products (a_row_scale / b_row_scale) are made by it;
// i_r outside the source is a row of zeros (the padding of a fixed-capacity expert).  The floor 2^-80 keeps s_r and its
// reciprocal normal numbers for rows of zeros.
//
// Bound by HBM: 2 bytes read and 1 written per element.  A row stays in registers between the maximum and the
// conversion, so it is read once.
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
// x carries 2^-20 so that 1 / m is a normal number for every finite m; top = 0.875 * 2^9 or 0.875 * 2^16.
struct Quotient {
    float m, back, inverse;
    __device__ __forceinline__ Quotient(float most, float two_power) : m(most) {
        const float a = most * 9.5367431640625e-07f;             // 2^-20
        back = a / two_power;
        inverse = two_power * __frcp_rn(a);
    }
    __device__ __forceinline__ float operator()(float x) const {
        x = fabsf(x) > m ? copysignf(m, x) : x;                  // an infinity; a NaN passes
        const float u = x * (0.875f * 9.5367431640625e-07f);     // exact: three more bits
        const float z = u * inverse;
        return fmaf(fmaf(-z, back, u), inverse, z);
    }
};

template <bool BF16>
__device__ __forceinline__ float finite_abs(uint16_t bits) {
    const uint16_t mag = bits & 0x7FFFu;
    if (mag >= (BF16 ? 0x7F80u : 0x7C00u)) return 0.0f;
    return BF16 ? __uint_as_float(static_cast<uint32_t>(mag) << 16) : __half2float(__ushort_as_half(mag));
}

__device__ __forceinline__ float block_max(float v, float* shared) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    const int warps = blockDim.x >> 5;
    if (warps == 1) return v;
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    v = static_cast<int>(threadIdx.x & 31) < warps ? shared[threadIdx.x & 31] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
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
        q[k] = __nv_cvt_float_to_fp8(quotient(v), __NV_SATFINITE, kind);
    }
    if (threadIdx.x == 0) args.scale[r] = most / (args.q_dtype == 0 ? 448.0f : 57344.0f);
}

}  // namespace b200fp8
