// Products of a matrix of 4-bit weights with a few vectors:
//
//     y[m][n] = sum over groups g of s[n][g] * sum_{k in g} (c[n][k] - z[n][g]) * x[m][k]
//
// c: codes 0..15, two to a byte, the even k in the low half; one scale (and, optionally, one zero point; 8 without) per row
// and group of 32, 64 or 128 k.  x is BF16 or FP16; y has its type or FP32.
//
// The arithmetic is exact up to the FP32 sums: c - z is a whole number of at most 15 and so exact in x's type (over 1024 in
// FP16, over 64 in BF16), the tensor core (m16n8k16) multiplies exactly and adds in FP32, and the scale multiplies a group's
// FP32 sum, not the rounded weight.  x is taken as it is, whatever stands beside it: bringing BF16 vectors to FP16 by a power
// of two per 256 of K, as this kernel once did, lost what was 2^-32 of the largest among them, which shows where that
// one's weight is zero, and took a sum and a factor per slot more (eight vectors, 28672 x 8192: 49.6 -> 45.4 us).
// Rows of the weights are the M index of the instruction and the vectors its N index, so up to eight vectors cost what
// one costs; the order of k inside an instruction is free, and is chosen so that a lane's eight codes are one aligned
// 32-bit word: (k, k + 4) share a 16-bit pair, which is what a mask takes out of the word.
//
// Bound by the weights' bytes from HBM: 13 weights per picosecond at the measured rate, 47 per SM and clock, of which the
// instructions above take 9 per eight (a shift, four masks, four subtractions) plus the tensor core's one.  So the
// kernel is about bytes in flight and few instructions:
//
//   * a CTA owns 128 rows of weights, 16 for each of eight warps (256 and 32 where there are many CTAs), and a part of K;
//     every warp streams the codes of its rows by TMA through a ring of its own (boxes of 16 or 32 rows of 128 bytes under
//     the 128-byte swizzle, 8 KB in flight) and refills a slot as soon as
//     it has read it: no producer warp and no waiting for other warps; two CTAs per SM;
//   * its part of x lies in shared memory, in the order in which the lanes want it;
//   * the parts of K of one tile of rows form a thread-block cluster and add their FP32 sums through distributed shared
//     memory in the order of K: no scratch in HBM, no atomics, one launch.
//
// By expert: row r of y takes the weights of expert[r] and row r / (rows / tokens) of x.  A block finds its rows by itself
// in one pass over `expert`: with fewer rows than experts block z stands for row z and works if that row is the
// first of its expert, else block z stands for expert z.  Each expert's weights are read once per eight of its rows (two in the
// integer form, which calls of one or two tokens take).
//
// Measured: one vector, 8192 x 8192, groups of 128: 12.4 us (2.8 TB/s; starting and joining the parts of K is about 5 of them); eight
// vectors, 28672 x 8192, groups of 64 with zero points: 45.4 us (2.8 TB/s, 0.43 of a plain copy's rate); 16 tokens with 8 of 64
// experts each, 2048 x 4096, groups of 128: 42.0 us.  Issue slots are half used: what bounds it is a warp's chain from a slot's
// arrival over unpacking to the sums, about 380 instructions per 16 x 256 codes at 16 warps per SM (a third CTA per SM spills: 64 us).
//
// Waits on mbarriers are bounded as in the other kernels: a wait that runs out sets the status word and ends the kernel.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>
#include <type_traits>
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
    int k_blocks;          // ceil(k / 256)
    int k_unit;            // parts of K begin at multiples of this many blocks
    int vector_scales, vector_zeros;   // four scales (zero points) of a row can be loaded at once
    int splits;            // parts of K = CTAs of a cluster
    int* status;
    int debug;             // 512: the third slot of the first warp stays unloaded
};

constexpr int kW4MostRows = 4096;        // rows of y of one call by expert: their list is held in shared memory
constexpr int kW4MostExperts = 4096;
constexpr int kW4Warps = 8;
constexpr int kW4Threads = 32 * kW4Warps;
constexpr int kW4MostSplits = 8;         // portable cluster size
constexpr int kW4BoxBytes = 128;         // of codes per row and ring slot: 256 of K
constexpr int kW4BoxK = 2 * kW4BoxBytes;
constexpr int kStatusW4Timeout = 106;

// c = a b (FIRST) or c += a b, in BF16 or FP16
#define B200FP8_W4_MMA(TYPE)                                                                                                                    \
    if constexpr (FIRST)                                                                                                                        \
        asm("mma.sync.aligned.m16n8k16.row.col.f32." TYPE "." TYPE ".f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"  \
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));               \
    else                                                                                                                                        \
        asm("mma.sync.aligned.m16n8k16.row.col.f32." TYPE "." TYPE ".f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"      \
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1))
template <bool BF16, bool FIRST>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (BF16) {
        B200FP8_W4_MMA("bf16");
    } else {
        B200FP8_W4_MMA("f16");
    }
}
#undef B200FP8_W4_MMA

// Codes become numbers of x's type without a conversion: a code in the four lowest bits of a half is the subnormal number
// c * 2^-24 of FP16 or c * 2^-133 of BF16, one in the next four bits 16 times that, so that a mask alone makes it a number
// and one fused multiply-add brings it to c * kUnit and takes the zero point off.  kUnit is the largest power of two that
// the factors of both places allow; (c - z) * kUnit has four significant bits and is exact.
template <bool BF16>
struct W4Number {
    using Pair = typename std::conditional<BF16, __nv_bfloat162, __half2>::type;
    static constexpr float kBack = BF16 ? 64.0f : 1024.0f;              // 1 / kUnit
    static __device__ __forceinline__ Pair twice(uint32_t bits) {
        const uint32_t w = bits | bits << 16;
        return *reinterpret_cast<const Pair*>(&w);
    }
    // A row's zero point as what its codes lose, -z * kUnit.  `zeros` holds four zero points, one to a byte.
    static __device__ __forceinline__ Pair minus(uint32_t zeros, uint32_t place) {
        const uint32_t z = __byte_perm(zeros, 0u, 0x4040u + place * 0x0101u);
        return __hmul2(*reinterpret_cast<const Pair*>(&z), twice(BF16 ? 0xFF00u : 0xF400u));                        // -2^127, -2^14
    }
    // The eight codes of a word as four pairs (j, j + 4).
    static __device__ __forceinline__ void unpack(uint32_t word, Pair minus, uint32_t (&a)[4]) {
        const uint32_t next = word >> 8;
        const uint32_t v[4] = {word & 0x000F000Fu, word & 0x00F000F0u, next & 0x000F000Fu, next & 0x00F000F0u};
        const Pair low = twice(BF16 ? 0x7F00u : 0x7400u), high = twice(BF16 ? 0x7D00u : 0x6400u);                   // 2^127, 2^14; 2^123, 2^10
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const Pair r = __hfma2(*reinterpret_cast<const Pair*>(&v[i]), i & 1 ? high : low, minus);
            a[i] = *reinterpret_cast<const uint32_t*>(&r);
        }
    }
};

// Eight consecutive x of one vector as pairs (0, 4), (1, 5), (2, 6), (3, 7).
__device__ __forceinline__ uint4 w4_vector_piece(uint4 v) {
    return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
}

// ---- the integer form --------------------------------------------------------------------------------------------------
// A few vectors leave most of the instruction's eight columns empty, and unpacking codes to floats is what bounds the form
// above.  Here an x becomes a whole number of 30 bits and a sign (scaled by a power of two per vector and 256 of K so that
// the largest lies in [2^29, 2^30)), cut into four signed bytes that take a column each: two vectors fill a tile of eight
// columns.  The codes then go into m16n8k32 as bytes, two masks and a shift per eight, the sums are exact integers (at most
// 128 * 15 * 128 in magnitude), z enters as z times the digits' sum over the group, and the columns meet with weights 1, 256,
// 65536, 2^24.  A block of 256 of K whose numbers do not all fit (an element more than 2^22 below the largest in BF16, 2^19
// in FP16 where the largest is 64 or more, an infinity or a NaN) is multiplied as the form above does it, with one column per
// vector, so that no block loses anything: an element far below the largest is all that counts where that one's weight is zero.
constexpr int kW4Magic = 0x4B400000;     // the FP32 number 3 * 2^22: adding a small integer to its bits adds it to its value

template <bool FIRST>
__device__ __forceinline__ void mma_16832(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (FIRST)
        asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(kW4Magic));
    else
        asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight consecutive x of one vector as digits d[0..3]: .x the even k's, .y the odd ones.  A whole warp calls it with 256
// consecutive k; `back` undoes the scaling.  True where this lane's numbers are not exactly these digits.
template <bool BF16>
__device__ __forceinline__ bool w4_digits(uint4 v, float& back, uint2 (&d)[4]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t most = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) most = max(most, max(w[i] & 0x7FFFu, (w[i] >> 16) & 0x7FFFu));
    most = __reduce_max_sync(0xffffffffu, most);
    // exponent of the largest: |x| < 2^(e + 1); a subnormal FP16 number counts as the smallest exponent
    const int e = BF16 ? static_cast<int>(most >> 7) - 127 : max(static_cast<int>(most >> 10), 1) - 15;
    const int up = min(126, 29 - e);
    const float forth = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
    back = __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
    bool lost = false;
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float2 f;
        if constexpr (BF16) f = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
        else f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        const float a = f.x * forth, b = f.y * forth;
        const int n = __float2int_rn(a), o = __float2int_rn(b);              // a NaN becomes 0, infinities the ends of int: not equal either
        lost = lost || __int2float_rn(n) != a || __int2float_rn(o) != b;
        u[2 * i] = static_cast<uint32_t>(n) + 0x80808080u;                   // its bytes are the balanced digits plus 128
        u[2 * i + 1] = static_cast<uint32_t>(o) + 0x80808080u;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t pick = i | (4 + i) << 4;
        d[i].x = __byte_perm(__byte_perm(u[0], u[2], pick), __byte_perm(u[4], u[6], pick), 0x5410) ^ 0x80808080u;
        d[i].y = __byte_perm(__byte_perm(u[1], u[3], pick), __byte_perm(u[5], u[7], pick), 0x5410) ^ 0x80808080u;
    }
    return lost;
}

// Four scales in a row from group `at` on (a multiple of four) as they are stored: FP32, or 16-bit ones two to a word.
template <bool WIDE> struct W4Scales;
template <> struct W4Scales<true> {
    uint4 v;
    __device__ __forceinline__ void load(const W4Args& args, long long row, int at, int groups) {
        const uint32_t* p = static_cast<const uint32_t*>(args.scales) + row + at;
        if (args.vector_scales && at + 4 <= groups) { v = __ldg(reinterpret_cast<const uint4*>(p)); return; }
        v = make_uint4(0u, 0u, 0u, 0u);
        if (at < groups) v.x = __ldg(p);
        if (at + 1 < groups) v.y = __ldg(p + 1);
        if (at + 2 < groups) v.z = __ldg(p + 2);
        if (at + 3 < groups) v.w = __ldg(p + 3);
    }
    // scales 2 pair and 2 pair + 1 of lane `from`
    __device__ __forceinline__ float2 pair(int p, int from, int) const {
        return make_float2(__uint_as_float(__shfl_sync(0xffffffffu, p ? v.z : v.x, from)), __uint_as_float(__shfl_sync(0xffffffffu, p ? v.w : v.y, from)));
    }
};
template <> struct W4Scales<false> {
    uint2 v;
    __device__ __forceinline__ void load(const W4Args& args, long long row, int at, int groups) {
        const uint16_t* p = static_cast<const uint16_t*>(args.scales) + row + at;
        if (args.vector_scales && at + 4 <= groups) { v = __ldg(reinterpret_cast<const uint2*>(p)); return; }
        v = make_uint2(0u, 0u);
        if (at < groups) v.x = __ldg(p);
        if (at + 1 < groups) v.x |= static_cast<uint32_t>(__ldg(p + 1)) << 16;
        if (at + 2 < groups) v.y = __ldg(p + 2);
        if (at + 3 < groups) v.y |= static_cast<uint32_t>(__ldg(p + 3)) << 16;
    }
    __device__ __forceinline__ float2 pair(int p, int from, int dtype) const {
        const uint32_t w = __shfl_sync(0xffffffffu, p ? v.y : v.x, from);
        return dtype == 1 ? make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)) : __half22float2(*reinterpret_cast<const __half2*>(&w));
    }
};
// Four zero points in a row, one to a byte.
__device__ __forceinline__ uint32_t w4_zeros(const W4Args& args, const uint8_t* row, int at, int groups) {
    if (args.vector_zeros && at + 4 <= groups) return __ldg(reinterpret_cast<const uint32_t*>(row + at));
    uint32_t v = 0u;
    if (at < groups) v = __ldg(row + at);
    if (at + 1 < groups) v |= static_cast<uint32_t>(__ldg(row + at + 1)) << 8;
    if (at + 2 < groups) v |= static_cast<uint32_t>(__ldg(row + at + 2)) << 16;
    if (at + 3 < groups) v |= static_cast<uint32_t>(__ldg(row + at + 3)) << 24;
    return v;
}

// NT: tiles of eight columns; RT: tiles of 16 rows per warp
template <int NT, int RT, bool INT>
struct W4Smem {
    static constexpr int kTileRows = 16 * RT * kW4Warps;         // rows of the weights per CTA
    static constexpr int kSlotBytes = 16 * RT * kW4BoxBytes;
    static constexpr int kStages = 4 / RT;                       // 8 KB in flight per warp
    static constexpr int kVectors = INT ? 2 * NT : 8 * NT;        // of x that share a pass over the weights
    static constexpr int kXK = INT ? 2048 : 2048 / NT;           // of K whose x is staged at a time
    static constexpr int kXPitch = kXK * (INT ? 1 : 2) + 64;     // bytes; two columns' lanes meet different banks
    static constexpr int kPartPitch = kTileRows + 4;           // floats
    static constexpr int kXOff = kW4Warps * kStages * kSlotBytes;
    static constexpr int kBackOff = kXOff + 8 * NT * kXPitch;     // powers of two [blocks][columns]
    static constexpr int kSumOff = kBackOff + kXK / kW4BoxK * 8 * NT * 4;               // INT: digits' sums [groups][columns]
    static constexpr int kPartOff = kSumOff + (INT ? kXK / 32 * 8 * NT * 4 : 0);
    static constexpr int kBarOff = kPartOff + 8 * NT * kPartPitch * 4;   // full[warp][stage], ready, done
    static constexpr int kMiscOff = kBarOff + 8 * (kW4Warps * kStages + 2);   // abort flag, INT: blocks of the chunk that go as floats
    static constexpr int kListOff = kMiscOff + 48;                       // by expert: rows of y (the call's row count)
    static constexpr int kFixedBytes = kListOff + 1024;                  // with the slack for 1024-byte alignment
};

// Rows of y for this block by expert, in ascending order into `list` (written by warp 0; every warp learns expert and
// count).  Returns the expert, -1 when the block has none.
__device__ __forceinline__ int w4_find_rows(const W4Args& args, int slot, int* list, bool write, int& count) {
    const int lane = threadIdx.x & 31;
    const bool by_row = args.m < args.experts;
    const int e = by_row ? __ldg(args.expert + slot) : slot;
    count = 0;
    constexpr int kAtOnce = 8;                                   // loads in flight: one round trip for up to 256 rows
    for (int r0 = 0; r0 < args.m; r0 += 32 * kAtOnce) {
        int id[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) id[i] = r0 + 32 * i + lane < args.m ? __ldg(args.expert + r0 + 32 * i + lane) : -1;
        if (e < 0 || e >= args.experts) return -1;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const uint32_t who = __ballot_sync(0xffffffffu, id[i] == e);
            if (by_row && count == 0 && who != 0 && r0 + 32 * i + __ffs(who) - 1 < slot) return -1;   // an earlier row stands for it
            if (write && id[i] == e) list[count + __popc(who & ((1u << lane) - 1u))] = r0 + 32 * i + lane;
            count += __popc(who);
        }
    }
    return count > 0 ? e : -1;
}

template <bool BF16, int G, int NT, int RT, bool WIDE, bool INT>           // WIDE: FP32 scales
__global__ void __launch_bounds__(kW4Threads, 2)
gemv_w4_kernel(const __grid_constant__ CUtensorMap tmap, const W4Args args)      // codes [experts][N][K/2], box 128 bytes x 16 RT rows
{
    using L = W4Smem<NT, RT, INT>;
    constexpr int kStages = L::kStages;
    static_assert((!INT && RT == 1) || NT == 1, "the integer form and the one with two row tiles have one tile of columns");
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (ptx::smem_addr(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - ptx::smem_addr(smem_raw));
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
    const int lane = threadIdx.x & 31;
    const uint32_t bar_full = smem_base + L::kBarOff + warp * 8 * kStages;     // this warp's
    const uint32_t bar_ready = smem_base + L::kBarOff + 8 * kW4Warps * kStages, bar_done = bar_ready + 8;
    const uint32_t ring = smem_base + warp * kStages * L::kSlotBytes;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem_gen + L::kMiscOff);
    int* as_floats = reinterpret_cast<int*>(smem_gen + L::kMiscOff + 8);               // INT: [block of the chunk]
    int* list = reinterpret_cast<int*>(smem_gen + L::kListOff);
    const bool clustered = args.splits > 1;

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < kW4Warps * kStages; ++s) ptx::mbar_init(smem_base + L::kBarOff + 8 * s, 1);
        ptx::mbar_init(bar_ready, args.splits);
        ptx::mbar_init(bar_done, args.splits);
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&tmap);
    }
    __syncthreads();
    if (clustered) ptx::cluster_arrive();                        // the wait comes before the first remote arrival
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();

    int e = 0, have = args.m;
    if (args.expert) e = w4_find_rows(args, blockIdx.z, list, warp == 0, have);
    if (e < 0) {                                                 // the same for all CTAs of the cluster
        if (clustered) ptx::cluster_wait();
        return;
    }
    const int n0 = blockIdx.y * L::kTileRows;
    const int split = blockIdx.x;
    const int units = (args.k_blocks + args.k_unit - 1) / args.k_unit;
    const int kb0 = static_cast<int>(static_cast<long long>(units) * split / args.splits) * args.k_unit;
    const int kb1 = min(args.k_blocks, static_cast<int>(static_cast<long long>(units) * (split + 1) / args.splits) * args.k_unit);
    const int batches = (have + L::kVectors - 1) / L::kVectors;
    long long to_fill = static_cast<long long>(batches) * (kb1 - kb0);                         // blocks of this warp's rows still to be asked for
    int fill_kb = kb0;
    // one lane: the next block into slot s
    auto fill = [&](int s) {
        if (!(args.debug && warp == 0 && fill_kb == kb0 + 2) && ptx::elect_one()) {
            ptx::mbar_arrive_expect_tx(bar_full + 8 * s, L::kSlotBytes);
            ptx::tma_load_3d(ring + s * L::kSlotBytes, &tmap, fill_kb * kW4BoxBytes, n0 + warp * 16 * RT, e, bar_full + 8 * s);
        }
        --to_fill;
        if (++fill_kb == kb1) fill_kb = kb0;
    };
    for (int s = 0; s < kStages && to_fill > 0; ++s) fill(s);

    constexpr int kGroups = kW4BoxK / G;                         // groups per ring slot: 2, 4 or 8
    constexpr int kWords = 8 / kGroups;                          // 32-bit words of codes per lane, row and group
    const int g = lane >> 2, t = lane & 3;
    // Which of the warp's rows stands at place g of the instruction is free; these orders keep the reads of codes free of
    // bank conflicts: the rows that one pass of a shared-memory read takes (two of 64 bytes, four of 32, eight of 16)
    // differ in the bits of the swizzle that the bytes of one row do not.
    const int row_of = G == 128 ? (g >> 1) | ((g & 1) << 2) : G == 64 ? (2 * g) % 8 + g / 4 : g;
    const int groups = args.k / G;
    // this lane's rows: two in each tile of 16, eight apart
    auto row = [&](int h, int i) { return warp * 16 * RT + 16 * h + 8 * i + row_of; };
    auto row_n = [&](int h, int i) { return static_cast<long long>(min(n0 + row(h, i), args.n - 1)); };
    auto scale_at = [&](int h, int i) { return e * args.scale_stride + row_n(h, i) * args.scale_ld; };
    auto zero_at = [&](int h, int i) { return args.zeros + e * args.zero_stride + row_n(h, i) * args.zero_ld; };
    // 16-byte chunk ^ row mod 8, the same for all its rows: the bits that depend on the lane; the others are xor'ed in
    const uint32_t lane_at = row_of * kW4BoxBytes + ((G == 128 ? t ^ row_of : G == 64 ? (t >> 1) ^ row_of : row_of) << 4) + (G == 64 ? (t & 1) * 8 : G == 32 ? t * 4 : 0);
    const uint32_t x_lane = smem_base + L::kXOff + g * L::kXPitch + t * 16;
    // Scales and zero points: the four lanes of a row hold those of 16 groups in a row, four each (a whole sector of
    // 16-bit scales), fetched 16 groups ahead and handed round by shuffles.  Fetched one by one, just before their use,
    // they bound the kernel: every load missed to HBM and kept the load unit busy with eight rows' lines.
    W4Scales<WIDE> s_now[RT][2], s_next[RT][2];
    uint32_t z_now[RT][2], z_next[RT][2];
    const int g_first = kb0 * kGroups;
    long long s_row[RT][2];
    const uint8_t* z_row[RT][2];
#pragma unroll
    for (int h = 0; h < RT; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            s_row[h][i] = scale_at(h, i);
            z_row[h][i] = args.zeros ? zero_at(h, i) : nullptr;
            z_next[h][i] = 0x08080808u;
        }
    auto fetch = [&](int window) {
        const int at = g_first + 16 * window + 4 * t;
#pragma unroll
        for (int h = 0; h < RT; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                s_next[h][i].load(args, s_row[h][i], at, groups);
                if (args.zeros) z_next[h][i] = w4_zeros(args, z_row[h][i], at, groups) & 0x0F0F0F0Fu;
            }
    };
    int s = 0;
    uint32_t ph = 0, round = 0;
    bool ok = true;                                              // after a wait that ran out: no more waits, no more copies, and on to the end
    for (int b = 0; b < batches; ++b) {
        const int m0 = b * L::kVectors, cols = min(L::kVectors, have - m0);   // vectors of this batch
        float y[RT][NT][4];
#pragma unroll
        for (int h = 0; h < RT; ++h)
#pragma unroll
            for (int j = 0; j < NT; ++j) y[h][j][0] = y[h][j][1] = y[h][j][2] = y[h][j][3] = 0.0f;
        fetch(0);
        for (int kc = kb0; kc < kb1; kc += L::kXK / kW4BoxK) {
            const int kend = min(kb1, kc + L::kXK / kW4BoxK);
            // x of these k-blocks: a warp takes one block, a lane eight of its k, for every vector (four loads in flight), and
            // places them so that the four lanes of a row of fragments read 64 bytes.  Vectors that are not there are zeros,
            // written once per batch.
            __syncthreads();
            constexpr int kBlocks = L::kXK / kW4BoxK;             // a chunk's: eight, or four
            const int block = warp % kBlocks;
            const int limit = kc == kb0 ? 8 * NT : cols;
            const int rest = lane % (4 * kWords);                 // piece within the group: lane rest / kWords's word rest % kWords
            if (INT && (kc + block < kend || kc == kb0)) {
                const int k = (kc + block) * kW4BoxK + lane * 8;
                const int word = (lane - rest) / 4 + rest % kWords;
                const uint32_t to = smem_base + L::kXOff + block * kW4BoxK + (word >> 1) * 64 + rest / kWords * 16 + (word & 1) * 8;
                float* sums = reinterpret_cast<float*>(smem_gen + L::kSumOff) + (block * kGroups + lane / (4 * kWords)) * 8 * NT;
                float* backs = reinterpret_cast<float*>(smem_gen + L::kBackOff) + block * 8 * NT;
                uint4 v[L::kVectors];
#pragma unroll
                for (int i = 0; i < L::kVectors; ++i) {
                    v[i] = make_uint4(0u, 0u, 0u, 0u);
                    if (i < cols && k < args.k && kc + block < kend) {
                        const int row = args.expert ? list[m0 + i] / args.rows_per_x : m0 + i;
                        v[i] = __ldg(reinterpret_cast<const uint4*>(args.x + row * args.ldx + k));
                    }
                }
                bool lost = false;
#pragma unroll
                for (int i = 0; i < L::kVectors; ++i) {
                    if (i >= cols && kc != kb0) break;            // columns of a vector that is not there: zeros, written once per batch
                    float back;
                    uint2 d[4];
                    lost = w4_digits<BF16>(v[i], back, d) || lost;
#pragma unroll
                    for (int q = 0; q < 4; q += 2) {              // two digits' sums in one word: at most 2^14 in magnitude each
                        int two = 0;
#pragma unroll
                        for (int u = q; u < q + 2; ++u) {
                            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to + (4 * i + u) * L::kXPitch), "r"(d[u].x), "r"(d[u].y) : "memory");
                            two += __dp4a(static_cast<int>(d[u].x), 0x01010101, __dp4a(static_cast<int>(d[u].y), 0x01010101, 0)) * (u == q ? 1 : 65536);
                        }
#pragma unroll
                        for (int o = 1; o < 4 * kWords; o <<= 1) two += __shfl_xor_sync(0xffffffffu, two, o);
                        const int low = static_cast<short>(two);
                        if (rest == 0) *reinterpret_cast<float2*>(sums + 4 * i + q) = make_float2(static_cast<float>(low), static_cast<float>((two - low) >> 16));
                    }
                    if (lane == 0) *reinterpret_cast<float4*>(backs + 4 * i) = make_float4(back, 256.0f * back, 65536.0f * back, 16777216.0f * back);
                }
                lost = __any_sync(0xffffffffu, lost);
                if (lane == 0) as_floats[block] = lost;
                if (lost) {                                       // as floats: 512 bytes per vector, in the place of its first two columns
                    const int piece = lane - rest + rest % kWords * 4 + rest / kWords;
                    const uint32_t to_floats = smem_base + L::kXOff + (piece >> 4) * L::kXPitch + block * kW4BoxK + (piece & 15) * 16;
                    __syncwarp();                                 // behind the other lanes' digits
#pragma unroll
                    for (int i = 0; i < L::kVectors; ++i) {
                        const uint4 h = w4_vector_piece(v[i]);
                        ptx::st_shared_v4(to_floats + 4 * i * L::kXPitch, h.x, h.y, h.z, h.w);
                    }
                }
            }
            if (!INT && (kc + block < kend || kc == kb0)) {
                const int k = (kc + block) * kW4BoxK + lane * 8;
                const int pos = lane - rest + rest % kWords * 4 + rest / kWords;
                const uint32_t to = smem_base + L::kXOff + (block * (kW4BoxK / 8) + pos) * 16;
                for (int c0 = warp / kBlocks * 4; c0 < limit; c0 += 4 * NT) {
                    uint4 v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        v[i] = make_uint4(0u, 0u, 0u, 0u);
                        if (c0 + i < cols && k < args.k && kc + block < kend) {
                            const int row = args.expert ? list[m0 + c0 + i] / args.rows_per_x : m0 + c0 + i;
                            v[i] = __ldg(reinterpret_cast<const uint4*>(args.x + row * args.ldx + k));
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (c0 + i >= limit) break;
                        const uint4 h = w4_vector_piece(v[i]);
                        ptx::st_shared_v4(to + (c0 + i) * L::kXPitch, h.x, h.y, h.z, h.w);
                    }
                }
            }
            __syncthreads();
            const uint32_t floats = INT ? __ballot_sync(0xffffffffu, lane < kend - kc && as_floats[lane % kBlocks] != 0) : 0u;   // a bit per block
            // The slots of the chunk; `mixed`: some of the integer form's blocks are floats.  Two copies of the loop, since the
            // choice inside it cost every call of the integer form 2 to 4 % (16384 x 16384: 36.3 -> 34.8 us).
            auto slots = [&](auto mixed) {
                for (int kb = kc; kb < kend; ++kb) {
                    const int rel = (kb - kb0) * kGroups & 15;        // first group of the slot within its 16
                    if (rel == 0) {
#pragma unroll
                        for (int h = 0; h < RT; ++h)
#pragma unroll
                            for (int i = 0; i < 2; ++i) { s_now[h][i] = s_next[h][i]; z_now[h][i] = z_next[h][i]; }
                        if (kb + 16 / kGroups < kb1) fetch(((kb - kb0) * kGroups >> 4) + 1);
                    }
                    if (ok && !wait_bounded(bar_full + 8 * s, ph, abort_flag, false)) {
                        record_failure(args.status, abort_flag, kStatusW4Timeout);
                        ok = false;
                    }
                    __syncwarp();
                    const uint32_t at = ring + s * L::kSlotBytes + lane_at;
                    uint32_t lo[RT][8], hi[RT][8];
#pragma unroll
                    for (int h = 0; h < RT; ++h) {
                        const uint32_t from = at + h * 16 * kW4BoxBytes;
                        if constexpr (G == 128) {
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const uint4 a = ptx::ld_shared_v4(from ^ (i << 6)), c = ptx::ld_shared_v4((from ^ (i << 6)) + 8 * kW4BoxBytes);
                                lo[h][4 * i] = a.x; lo[h][4 * i + 1] = a.y; lo[h][4 * i + 2] = a.z; lo[h][4 * i + 3] = a.w;
                                hi[h][4 * i] = c.x; hi[h][4 * i + 1] = c.y; hi[h][4 * i + 2] = c.z; hi[h][4 * i + 3] = c.w;
                            }
                        } else if constexpr (G == 64) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(lo[h][2 * i]), "=r"(lo[h][2 * i + 1]) : "r"(from ^ (i << 5)) : "memory");
                                asm volatile("ld.shared.v2.b32 {%0, %1}, [%2+1024];" : "=r"(hi[h][2 * i]), "=r"(hi[h][2 * i + 1]) : "r"(from ^ (i << 5)) : "memory");
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                lo[h][i] = ptx::ld_shared_u32(from ^ (i << 4));
                                hi[h][i] = ptx::ld_shared_u32((from ^ (i << 4)) + 8 * kW4BoxBytes);
                            }
                        }
                    }
                    // The slot may be refilled once these reads are done.  The refill is a write of another proxy (TMA), and nothing
                    // but a proxy fence orders it behind them: without it a warp read codes of the ring's next turn.
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (ok && to_fill > 0) fill(s);
                    __syncwarp();
                    if (++s == kStages) { s = 0; ph ^= 1u; }
                    const uint32_t x_at = x_lane + (kb - kc) * (INT ? 1 : 2) * kW4BoxK;
                    // The slot's products, by group; `ints`: in the integer form.
                    auto multiply = [&](auto ints) {
                        constexpr bool kInts = decltype(ints)::value;
                        float2 two[RT][2];                            // scales of two groups
                        uint32_t zeros[RT][2];                        // zero points of four groups
                        uint4 digits[NT];
                        float ys[RT][NT][4];                          // kInts: this slot's sums, in the scaling of its x
#pragma unroll
                        for (int h = 0; h < RT; ++h) {
                            zeros[h][0] = zeros[h][1] = 0x08080808u;
#pragma unroll
                            for (int j = 0; j < NT; ++j) ys[h][j][0] = ys[h][j][1] = ys[h][j][2] = ys[h][j][3] = 0.0f;
                        }
#pragma unroll
                        for (int i = 0; i < kGroups; ++i) {
                            // group rel + i of the 16: lane (rel + i) / 4 of the row holds it, at place (rel + i) % 4
                            const int from = (lane & ~3) | ((rel + i) >> 2);
#pragma unroll
                            for (int h = 0; h < RT; ++h)
#pragma unroll
                                for (int u = 0; u < 2; ++u) {
                                    if ((i & 1) == 0) two[h][u] = s_now[h][u].pair(((kGroups == 2 ? rel : i) >> 1) & 1, from, args.scale_dtype);
                                    if (args.zeros && (i & 3) == 0) zeros[h][u] = __shfl_sync(0xffffffffu, z_now[h][u], from);
                                }
                            auto scale = [&](int h, int u) { return i & 1 ? two[h][u].y : two[h][u].x; };
                            const uint32_t place = kGroups == 2 ? (rel + i) & 3 : i & 3;
                            if constexpr (kInts) {
                                int c[RT][NT][4];
#pragma unroll
                                for (int w = i * kWords; w < (i + 1) * kWords; ++w) {
#pragma unroll
                                    for (int j = 0; j < NT; ++j)
                                        if ((w & 1) == 0) digits[j] = ptx::ld_shared_v4(x_at + 8 * j * L::kXPitch + (w >> 1) * 64);   // two words'
#pragma unroll
                                    for (int h = 0; h < RT; ++h) {
                                        const uint32_t le = lo[h][w] & 0x0F0F0F0Fu, lo4 = (lo[h][w] >> 4) & 0x0F0F0F0Fu;
                                        const uint32_t he = hi[h][w] & 0x0F0F0F0Fu, hi4 = (hi[h][w] >> 4) & 0x0F0F0F0Fu;
#pragma unroll
                                        for (int j = 0; j < NT; ++j) {
                                            const uint32_t b0 = w & 1 ? digits[j].z : digits[j].x, b1 = w & 1 ? digits[j].w : digits[j].y;
                                            if (w == i * kWords) mma_16832<true>(c[h][j], le, he, lo4, hi4, b0, b1);
                                            else mma_16832<false>(c[h][j], le, he, lo4, hi4, b0, b1);
                                        }
                                    }
                                }
                                const float* sums = reinterpret_cast<const float*>(smem_gen + L::kSumOff) + ((kb - kc) * kGroups + i) * 8 * NT + 2 * t;
#pragma unroll
                                for (int j = 0; j < NT; ++j) {
                                    const float2 d = *reinterpret_cast<const float2*>(sums + 8 * j);
#pragma unroll
                                    for (int h = 0; h < RT; ++h)
#pragma unroll
                                        for (int u = 0; u < 2; ++u) {
                                            // z as a number: its byte below the bits of 2^23; all exact: whole numbers below 2^24
                                            const float z = __uint_as_float(__byte_perm(zeros[h][u], 0x4B000000u, 0x7540u | place)) - 8388608.0f;
                                            const float even = fmaf(-z, d.x, __int_as_float(c[h][j][2 * u])) - 12582912.0f;
                                            const float odd = fmaf(-z, d.y, __int_as_float(c[h][j][2 * u + 1])) - 12582912.0f;
                                            ys[h][j][2 * u] = fmaf(scale(h, u), even, ys[h][j][2 * u]);
                                            ys[h][j][2 * u + 1] = fmaf(scale(h, u), odd, ys[h][j][2 * u + 1]);
                                        }
                                }
                            } else {
                                float c[RT][NT][4];
                                using Number = W4Number<BF16>;
                                typename Number::Pair minus[RT][2];
#pragma unroll
                                for (int h = 0; h < RT; ++h) { minus[h][0] = Number::minus(zeros[h][0], place); minus[h][1] = Number::minus(zeros[h][1], place); }
#pragma unroll
                                for (int w = i * kWords; w < (i + 1) * kWords; ++w) {
                                    uint4 v[NT];
                                    if constexpr (INT) {              // a vector's first column has all of it
                                        v[0] = make_uint4(0u, 0u, 0u, 0u);
                                        if ((g & 3) == 0) v[0] = ptx::ld_shared_v4(x_at + (w >> 2) * L::kXPitch + (w & 3) * 64);
                                    } else {
#pragma unroll
                                        for (int j = 0; j < NT; ++j) v[j] = ptx::ld_shared_v4(x_at + 8 * j * L::kXPitch + w * 64);
                                    }
#pragma unroll
                                    for (int h = 0; h < RT; ++h) {
                                        uint32_t a[4], b[4];
                                        Number::unpack(lo[h][w], minus[h][0], a);
                                        Number::unpack(hi[h][w], minus[h][1], b);
#pragma unroll
                                        for (int j = 0; j < NT; ++j) {
                                            if (w == i * kWords) mma_16816<BF16, true>(c[h][j], a[0], b[0], a[1], b[1], v[j].x, v[j].y);
                                            else mma_16816<BF16, false>(c[h][j], a[0], b[0], a[1], b[1], v[j].x, v[j].y);
                                            mma_16816<BF16, false>(c[h][j], a[2], b[2], a[3], b[3], v[j].z, v[j].w);
                                        }
                                    }
                                }
#pragma unroll
                                for (int h = 0; h < RT; ++h)
#pragma unroll
                                    for (int j = 0; j < NT; ++j) {
#pragma unroll
                                        for (int q = 0; q < 4; ++q) y[h][j][q] = fmaf(scale(h, q >> 1), (INT ? Number::kBack : 1.0f) * c[h][j][q], y[h][j][q]);
                                    }
                            }
                        }
                        if constexpr (kInts) {
                            const float* back = reinterpret_cast<const float*>(smem_gen + L::kBackOff) + (kb - kc) * 8 * NT + 2 * t;
#pragma unroll
                            for (int j = 0; j < NT; ++j) {
                                const float2 p = *reinterpret_cast<const float2*>(back + 8 * j);
#pragma unroll
                                for (int h = 0; h < RT; ++h)
#pragma unroll
                                    for (int q = 0; q < 4; ++q) y[h][j][q] = fmaf(q & 1 ? p.y : p.x, ys[h][j][q], y[h][j][q]);
                            }
                        }
                    };
                    if constexpr (!INT) multiply(std::false_type{});
                    else if constexpr (!decltype(mixed)::value) multiply(std::true_type{});
                    else if (floats >> (kb - kc) & 1) multiply(std::false_type{});
                    else multiply(std::true_type{});
                }
            };
            if (INT && floats != 0) slots(std::true_type{});
            else slots(std::false_type{});
        }
        // the parts of K meet: every CTA lays its sums out in its shared memory and adds a share of the rows
        float* part = reinterpret_cast<float*>(smem_gen + L::kPartOff);
#pragma unroll
        for (int h = 0; h < RT; ++h)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    part[(8 * j + 2 * t + (i & 1)) * L::kPartPitch + row(h, i >> 1)] = (INT ? 1.0f : W4Number<BF16>::kBack) * y[h][j][i];
        if (clustered) {
            if (b == 0) ptx::cluster_wait();                     // every CTA of the cluster has its barriers
            __syncthreads();
            if (threadIdx.x < args.splits) ptx::mbar_arrive_cluster(ptx::mapa(bar_ready, threadIdx.x));
            if (ok && !wait_bounded(bar_ready, round & 1u, abort_flag, true)) { record_failure(args.status, abort_flag, kStatusW4Timeout); ok = false; }
        } else {
            __syncthreads();
        }
        const int share = L::kTileRows / args.splits;
        const uint32_t part_addr = smem_base + L::kPartOff;
        for (int i = threadIdx.x; i < cols * share && ok; i += 32 * kW4Warps) {
            const int c = i / share, r = split * share + i - c * share;
            float sum = 0.0f;
#pragma unroll
            for (int q = 0; q < (INT ? 4 : 1); ++q) {
                const int column = (INT ? 4 : 1) * c + q;
                if (clustered) {
                    const uint32_t at = part_addr + (column * L::kPartPitch + r) * 4;
                    float v[kW4MostSplits];                       // all loads in flight, then added in the order of K
#pragma unroll
                    for (int p = 0; p < kW4MostSplits; ++p) v[p] = p < args.splits ? __uint_as_float(ptx::ld_shared_cluster_u32(ptx::mapa(at, p))) : 0.0f;
#pragma unroll
                    for (int p = 0; p < kW4MostSplits; ++p) sum += v[p];
                } else {
                    sum += part[column * L::kPartPitch + r];
                }
            }
            if (n0 + r < args.n) store_out(args.y, static_cast<long long>(args.expert ? list[m0 + c] : m0 + c) * args.ldy + n0 + r, sum, args.y_dtype);
        }
        __syncthreads();
        if (clustered && b + 1 < batches) {                      // the next batch may overwrite the sums once all have read them
            if (threadIdx.x < args.splits) ptx::mbar_arrive_cluster(ptx::mapa(bar_done, threadIdx.x));
            if (ok && !wait_bounded(bar_done, round & 1u, abort_flag, true)) { record_failure(args.status, abort_flag, kStatusW4Timeout); ok = false; }
        }
        ++round;
    }
    if (!ok && lane == 0) {                                       // leave no copy in flight into this CTA's shared memory
        for (int i = 0; i < kStages; ++i) {
            const uint64_t t0 = ptx::globaltimer_ns();
            while (!ptx::mbar_try_wait(bar_full + 8 * s, ph) && ptx::globaltimer_ns() - t0 < kWaitLimitNs / 8) {}
            if (++s == kStages) { s = 0; ph ^= 1u; }
        }
    }
    __syncwarp();
    if (clustered) { ptx::cluster_arrive(); ptx::cluster_wait(); }   // no CTA leaves while another reads its shared memory
}

}  // namespace b200fp8
