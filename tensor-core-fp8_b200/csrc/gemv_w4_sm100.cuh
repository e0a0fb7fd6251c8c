// Products of a matrix of 4-bit weights with a few vectors:
//
//     y[m][n] = sum over groups g of s[n][g] * sum_{k in g} (c[n][k] - z[n][g]) * x[m][k]
//
// c: codes 0..15, two to a byte, the even k in the low half; one scale (and, optionally, one zero point; 8 without) per row
// and group of 32, 64 or 128 k.  x is BF16 or FP16; y has its type or FP32.
//
// The arithmetic is exact up to the FP32 sums: c - z is a whole number of at most 15 and so exact in either 16-bit type,
// the tensor core (m16n8k16) multiplies exactly and adds in FP32, and the scale multiplies a group's FP32 sum, not the
// rounded weight.  Rows of the weights are the M index of the instruction and the vectors its N index, so up to eight
// vectors cost what one costs; the order of k inside an instruction is free, and is chosen so that a lane's eight codes
// are one aligned 32-bit word: (k, k + 4) share a 16-bit pair, which is what a mask and a shift take out of the word.
//
// By expert: row r of y takes the weights of expert[r] and row r / (rows / tokens) of x.  A block finds the experts that
// occur by itself (a bit set over `expert`), so each of them is read once whatever the routing, with no second launch.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>
#include "gemm_sm100.cuh"

namespace b200fp8 {

struct W4Args {
    const uint8_t* codes;  long long code_ld, code_stride;     // bytes: row pitch, expert pitch
    const void* scales;    long long scale_ld, scale_stride;   // elements
    const uint8_t* zeros;  long long zero_ld, zero_stride;     // elements; nullptr: 8
    int scale_dtype;       // 0 FP32, 1 BF16, 2 FP16
    const uint16_t* x;     long long ldx;
    void* y;               long long ldy;
    int y_dtype;
    int m, n, k, group;
    const int* expert;     // by expert: the expert of each row of y, else nullptr
    int experts, rows_per_x;
};

constexpr int kW4MostRows = 4096;        // rows of y of one call by expert: their list is held in shared memory
constexpr int kW4MostExperts = 4096;

template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Codes j and j + 4 of a word as a pair of 16-bit floats minus the zero point, exactly.  A code placed in the low bits of
// the number 128 (BF16: eight significant bits) or 1024 (FP16: eleven) adds itself to that number.
template <bool BF16>
__device__ __forceinline__ uint32_t w4_pair(uint32_t word, int j, uint32_t minus) {
    const uint32_t v = ((word >> (4 * j)) & 0x000F000Fu) | (BF16 ? 0x43004300u : 0x64006400u);
    if constexpr (BF16) {
        const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&minus));
        return *reinterpret_cast<const uint32_t*>(&r);
    } else {
        const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&minus));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
}
// the number 128 + z (1024 + z) in both halves
template <bool BF16>
__device__ __forceinline__ uint32_t w4_minus(uint32_t z) { return ((z & 15u) | (BF16 ? 0x4300u : 0x6400u)) * 0x00010001u; }

__device__ __forceinline__ float w4_scale(const W4Args& args, long long at) { return load_out(args.scales, at, args.scale_dtype); }

// Rows of y that this block computes together: the `slot`-th expert that occurs, in ascending order, and its rows.
// Returns the expert, or -1 when fewer experts occur.  All threads of the block call it.
__device__ __forceinline__ int w4_find_rows(const W4Args& args, int slot, uint32_t* bits, int* list, int* count) {
    for (int i = threadIdx.x; i < (args.experts + 31) / 32; i += blockDim.x) bits[i] = 0u;
    __syncthreads();
    for (int r = threadIdx.x; r < args.m; r += blockDim.x) {
        const int e = args.expert[r];
        if (e >= 0 && e < args.experts) atomicOr(bits + (e >> 5), 1u << (e & 31));
    }
    __syncthreads();
    int found = -1, left = slot;
    for (int i = 0; i < (args.experts + 31) / 32; ++i) {
        const int here = __popc(bits[i]);
        if (left < here) { found = 32 * i + static_cast<int>(__fns(bits[i], 0, left + 1)); break; }
        left -= here;
    }
    if (found < 0) return -1;
    if (threadIdx.x < 32) {                                    // one warp keeps the list in ascending order
        int n = 0;
        for (int r0 = 0; r0 < args.m; r0 += 32) {
            const int r = r0 + static_cast<int>(threadIdx.x);
            const bool mine = r < args.m && args.expert[r] == found;
            const uint32_t who = __ballot_sync(0xffffffffu, mine);
            if (mine) list[n + __popc(who & ((1u << threadIdx.x) - 1u))] = r;
            n += __popc(who);
        }
        if (threadIdx.x == 0) *count = n;
    }
    __syncthreads();
    return found;
}

constexpr int kW4SimpleWarps = 4;

// The simple form: a warp per 16 rows of the weights and eight vectors, straight from global memory.
template <bool BF16>
__global__ void __launch_bounds__(32 * kW4SimpleWarps) gemv_w4_simple_kernel(const W4Args args) {
    __shared__ uint32_t bits[kW4MostExperts / 32];
    __shared__ int list[kW4MostRows];
    __shared__ int count;
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    int e = 0, have = args.m;
    if (args.expert) {
        e = w4_find_rows(args, blockIdx.z, bits, list, &count);
        if (e < 0) return;
        have = count;
    }
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = (blockIdx.x * kW4SimpleWarps + (threadIdx.x >> 5)) * 16;
    if (n0 >= args.n) return;
    const int lo = min(n0 + g, args.n - 1), hi = min(n0 + g + 8, args.n - 1);
    const uint8_t* codes = args.codes + e * args.code_stride;
    const uint8_t *clo = codes + lo * args.code_ld, *chi = codes + hi * args.code_ld;
    const long long slo = e * args.scale_stride + lo * args.scale_ld, shi = e * args.scale_stride + hi * args.scale_ld;
    const long long zlo = e * args.zero_stride + lo * args.zero_ld, zhi = e * args.zero_stride + hi * args.zero_ld;
    for (int m0 = blockIdx.y * 8; m0 < have; m0 += 8 * gridDim.y) {
        const int col = m0 + g;
        const int row = col < have ? (args.expert ? list[col] / args.rows_per_x : col) : -1;
        const uint16_t* x = args.x + (row < 0 ? 0 : row) * args.ldx;
        float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int k0 = 0; k0 < args.k; k0 += args.group) {
            const int at = k0 / args.group;
            uint32_t mlo = w4_minus<BF16>(8), mhi = mlo;
            if (args.zeros) { mlo = w4_minus<BF16>(args.zeros[zlo + at]); mhi = w4_minus<BF16>(args.zeros[zhi + at]); }
            float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int k = k0 + t * 8; k < k0 + args.group; k += 32) {
                const uint32_t wlo = *reinterpret_cast<const uint32_t*>(clo + k / 2), whi = *reinterpret_cast<const uint32_t*>(chi + k / 2);
                uint4 v = make_uint4(0u, 0u, 0u, 0u);
                if (row >= 0) v = *reinterpret_cast<const uint4*>(x + k);
                const uint32_t b0 = __byte_perm(v.x, v.z, 0x5410), b1 = __byte_perm(v.x, v.z, 0x7632);
                const uint32_t b2 = __byte_perm(v.y, v.w, 0x5410), b3 = __byte_perm(v.y, v.w, 0x7632);
                mma_16816<BF16>(c, w4_pair<BF16>(wlo, 0, mlo), w4_pair<BF16>(whi, 0, mhi), w4_pair<BF16>(wlo, 1, mlo), w4_pair<BF16>(whi, 1, mhi), b0, b1);
                mma_16816<BF16>(c, w4_pair<BF16>(wlo, 2, mlo), w4_pair<BF16>(whi, 2, mhi), w4_pair<BF16>(wlo, 3, mlo), w4_pair<BF16>(whi, 3, mhi), b2, b3);
            }
            const float sl = w4_scale(args, slo + at), sh = w4_scale(args, shi + at);
            y[0] = fmaf(sl, c[0], y[0]);
            y[1] = fmaf(sl, c[1], y[1]);
            y[2] = fmaf(sh, c[2], y[2]);
            y[3] = fmaf(sh, c[3], y[3]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = m0 + 2 * t + (i & 1), n = n0 + g + (i >> 1) * 8;
            if (c < have && n < args.n) store_out(args.y, static_cast<long long>(args.expert ? list[c] : c) * args.ldy + n, y[i], args.y_dtype);
        }
    }
}

}  // namespace b200fp8
