// FP8 products grouped by expert with ragged sizes, forward and backward, on the tensor cores (tcgen05):
//
//   forward   D[r][n]    = ep( sum_k A[r][k] B[e][n][k] )    r in group e     A [rows][K]  B [E][N][K]  D [rows][N]
//   dgrad     D[r][k]    = ep( sum_n A[r][n] B[e][n][k] )    r in group e     A [rows][N]  B [E][N][K]  D [rows][K]
//   wgrad     D[e][n][k] = ep( sum_{r in e} A[r][n] B[r][k] )                 A [rows][N]  B [rows][K]  D [E][N][K]
//
// Group e holds the rows [end of group e-1, ends[e]); `ends` is read by the kernel (device memory), so a router on the same
// stream may have written it just before.  Ends are clamped to [0, rows] and to their running maximum, so that no
// content of `ends` makes the kernel touch anything outside the operands.  Rows of no group are left as they were.
//
// Operands are read as they are stored, in all three products: the tensor core takes an operand whose contraction index
// is contiguous (A and B forward, A of dgrad) or whose row index is (B of dgrad, both of wgrad; the descriptor's MN-major
// form), so training needs no transposed copies.
//
// Structure: that of the dense kernel (gemm_sm100.cuh) -- a persistent CTA or CTA pair per SM, warp 0 TMA producer into a
// ring of k-blocks (128 bytes of contraction each), warp 1 MMA issue, warps 2-9 epilogue out of two TMEM accumulator
// slots -- with two differences:
//
//   * The walk over tiles: every warp derives it from `ends` by itself (32 groups at a time in the lanes of a warp, one scan
//     and one ballot per tile), so there is no schedule to build, no workspace and no second launch.
//   * The accumulator is D transposed: the columns of D (128 per CTA, contiguous in memory) are the tensor core's M index
//     = the lanes of TMEM, the ragged rows its N index.  N is set per tile to the tile's rows rounded up to 16 (32 for a
//     pair), so a group's last tile costs what its rows cost: with 256-row tiles and groups of about a thousand rows,
//     tiles of full height wasted an eighth of the multiplications (and, in a power-limited run, of the energy); a decode
//     step's few rows per expert cost few bytes and cycles next to the weights (a tile loads the shortest of four boxes,
//     16 to 128 rows, that covers them).  In the epilogue a lane owns columns, so the vectors per column (b_row_scale,
//     bias) are a few registers.  FP32 rows go out as they are, 128 bytes per instruction.  16-bit ones are read from TMEM
//     in the matrix-fragment distribution, packed in pairs along the rows and transposed on the way through shared memory
//     by stmatrix, then stored 16 bytes per lane, or a row's 64 bytes from 32 lanes where the alignment allows no more
//     (swapping columns between neighbouring lanes instead took four times the instructions, and the epilogue bounds
//     products with a short contraction).  8-bit ones are packed four rows to a word and transposed 4 x 4 between four
//     lanes, then stored 4 bytes per lane.  Rows behind a group's end are simply not stored, and D needs no TMA.
//
// Rows behind a group's end inside a tile belong to the next group.  Forward and dgrad may load and multiply them (each
// row of a product depends on its own row of A only) and do not store them.  wgrad contracts over the rows, so the block
// across a group's end must not see the next group: it is loaded as 32-row TMA boxes, and the last, ragged 32 rows
// with ordinary loads that put zeros behind the end (a product with zero would not do: the other operand's foreign rows
// may hold infinities or NaN).  The MMA issues only as many K = 32 steps as there are rows.  A group without rows stores
// zeros (or beta * D).
//
// Measured (per call, BF16 outputs; one launch - a long run, which the power limit slows): 32 rows over 16 experts of 4096 x
// 4096, 12 hit: 33.4 us, 6.0 TB/s of weights.  16384 rows, 16 experts of 8192 x 4096, bias and GELU: 412 - 526 us (1.04 GHz),
// 2.6 - 2.0 PFLOP/s, tensor pipe 81 % in the former.  dgrad of 8192 rows, 8 experts of 8192 x 4096: 202 - 262 us (1.09 GHz), 2.7 -
// 2.1 PFLOP/s, tensor pipe 79 %.  wgrad of 8192 rows, 8 experts of 4096 x 4096: 138 - 166 us (1.43 GHz), tensor pipe 52 %.
//
// Every wait on an mbarrier is bounded, as in the dense kernel.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cstdint>
#include "gemm_sm100.cuh"

namespace b200fp8 {

enum GroupedMode : int { kGroupedForward = 0, kGroupedDgrad = 1, kGroupedWgrad = 2 };

// The operand whose index becomes the columns of D (W: the weights; wgrad: the input X) and the one whose index becomes its
// rows (R: the ragged rows; wgrad: the output's gradient, N columns).
struct GroupedMaps {
    CUtensorMap w;        // 128 x 128 boxes
    CUtensorMap r[4];     // forward, dgrad: boxes of 16, 32, 64, 128 rows; wgrad: [3] 128 x 128
    CUtensorMap w32, r32; // wgrad: 32 rows of 128 bytes
};

struct GroupedArgs {
    int experts;
    int rows;             // rows of the ragged operands
    int d_rows;           // wgrad: rows of D per expert (N)
    int cols;             // columns of D
    int depth;            // contraction extent: K forward, N dgrad (wgrad: the group's rows)
    const int* ends;
    int row_tiles;        // wgrad: tiles along the rows of D[e]
    int col_tiles;
    int group_rows;       // tiles are walked down this many row tiles before the next column tile
    uint32_t idesc;       // without N
    int wide_store;       // 16-bit D: eight neighbouring columns can be stored as 16 bytes; 8-bit D: four as 4
    void* d;
    long long ldd, stride_d;
    const uint8_t* w;     // wgrad: base pointers of the ragged rows' ordinary loads
    const uint8_t* r;
    long long ldw, ldr;
    int* status;
    int debug;            // 512: the third k-block of every CTA's first tile stays unloaded
    Epilogue epi;
};

// One tile: expert, position, and what it multiplies.
struct GroupedTile {
    int e;
    int row0;        // forward, dgrad: first row of the tile in R and D; wgrad: first row of the tile in D[e]
    int rows;        // rows of the tile (>= 1)
    int col0;        // first column of the tile (of the pair)
    int k0, k_end;   // contraction range (wgrad: rows of the group)
};

// Walk over the tiles of all groups in order.  All 32 lanes call it together.
template <int MODE, int TILE_ROWS, int TILE_COLS>
struct GroupedWalk {
    const GroupedArgs& args;
    int lane;
    int chunk;             // first expert of the 32 in the lanes
    int carry;             // cleaned end of the last expert before the chunk
    long long base;        // tiles before the chunk
    int start, end;        // this lane's group
    int upto;              // tiles of the chunk up to and including this lane's
    int total;             // tiles of the chunk

    __device__ __forceinline__ explicit GroupedWalk(const GroupedArgs& a) : args(a), lane(threadIdx.x & 31), chunk(0), carry(0), base(0) { load(); }

    __device__ __forceinline__ void load() {
        const int e = chunk + lane;
        end = e < args.experts ? min(max(__ldg(args.ends + e), 0), args.rows) : 0;
        end = max(end, carry);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o) end = max(end, other);
        }
        start = __shfl_up_sync(0xffffffffu, end, 1);
        if (lane == 0) start = carry;
        carry = __shfl_sync(0xffffffffu, end, 31);
        if (MODE == kGroupedWgrad) upto = e < args.experts ? args.row_tiles * args.col_tiles : 0;
        else upto = (end - start + TILE_ROWS - 1) / TILE_ROWS * args.col_tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += other;
        }
        total = __shfl_sync(0xffffffffu, upto, 31);
    }

    // tile t (t never decreases between calls); false behind the last one
    __device__ __forceinline__ bool seek(long long t, GroupedTile& w) {
        while (t >= base + total) {
            base += total;
            chunk += 32;
            if (chunk >= args.experts) { total = 0; return false; }
            load();
        }
        const int local = static_cast<int>(t - base);
        const int who = __ffs(__ballot_sync(0xffffffffu, local < upto)) - 1;
        const int s = __shfl_sync(0xffffffffu, start, who), f = __shfl_sync(0xffffffffu, end, who);
        const int before = who == 0 ? 0 : __shfl_sync(0xffffffffu, upto, who - 1);
        const int r = local - before;
        w.e = chunk + who;
        const int extent = MODE == kGroupedWgrad ? args.d_rows : f - s;
        const int row_tiles = MODE == kGroupedWgrad ? args.row_tiles : (extent + TILE_ROWS - 1) / TILE_ROWS;
        const int per_group = args.group_rows * args.col_tiles;
        const int g = r / per_group;
        const int first = g * args.group_rows;
        const int size = min(args.group_rows, row_tiles - first);
        const int in_group = r - g * per_group;
        const int at = (first + in_group % size) * TILE_ROWS;
        w.col0 = in_group / size * TILE_COLS;
        w.rows = min(TILE_ROWS, extent - at);
        if (MODE == kGroupedWgrad) {
            w.row0 = at;
            w.k0 = s;
            w.k_end = f;
        } else {
            w.row0 = s + at;
            w.k0 = 0;
            w.k_end = args.depth;
        }
        return true;
    }
};

// The formula of gelu_tanh (gemm_sm100.cuh) for two neighbours, t / (1 + exp2(t (a + b t^2))): packed where the hardware
// packs, subnormals of the exponential and the reciprocal flushed (they are below the last bit of 1 + e, and of no weight in t times
// a number below 2^-126).  Two special-function results per element are what is left (16 per SM and
// clock): 37 of the 99 us that 10629 x 7792 x 448 takes in two groups, 57 without an activation and 108 with the scalar form.
__device__ __forceinline__ void grouped_gelu_tanh(uint32_t& t0, uint32_t& t1) {
    constexpr float kA = -2.3022081985f, kB = -0.1029432396f;     // -2 sqrt(2 / pi) log2(e), times 0.044715
    uint64_t t, a, b, u;
    asm("mov.b64 %0, {%1, %2};" : "=l"(t) : "r"(t0), "r"(t1));
    asm("mov.b64 %0, {%1, %1};" : "=l"(a) : "f"(kA));
    asm("mov.b64 %0, {%1, %1};" : "=l"(b) : "f"(kB));
    asm("mul.rn.f32x2 %0, %1, %1;" : "=l"(u) : "l"(t));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(u) : "l"(u), "l"(b), "l"(a));
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(u) : "l"(u), "l"(t));
    float e0, e1;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(e0), "=f"(e1) : "l"(u));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e0));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e1));
    e0 += 1.0f;
    e1 += 1.0f;
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(e0));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(e1));
    t0 = __float_as_uint(__uint_as_float(t0) * e0);
    t1 = __float_as_uint(__uint_as_float(t1) * e1);
}

// the low half of a word as BF16 (out_dtype 1) or FP16
__device__ __forceinline__ float wide16(uint32_t bits, int out_dtype) {
    return out_dtype == 1 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
}

// 32 numbers to bytes, four to a word
template <__nv_fp8_interpretation_t TYPE>
__device__ __forceinline__ void grouped_pack8(const uint32_t (&v)[32], uint32_t (&b)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1])), __NV_SATFINITE, TYPE);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(__uint_as_float(v[4 * j + 2]), __uint_as_float(v[4 * j + 3])), __NV_SATFINITE, TYPE);
        b[j] = lo | hi << 16;
    }
}

// ROWS: rows of D per tile (of the pair), the largest N of the MMA
template <int ROWS, int CTAS>
struct GroupedSmem {
    static constexpr int kWBytes = 128 * kBlockK;
    static constexpr int kRRows = ROWS / CTAS;
    static constexpr int kRBytes = kRRows * kBlockK;
    static constexpr int kStageBytes = kWBytes + kRBytes;
    static constexpr int kScaleBytes = kEpiWarps * ROWS / 2 * 4;             // row scales of a warp's rows
    static constexpr int kTurnBytes = 32 * 64;                              // 32 rows x 32 columns of 16 bits, per epilogue warp
    static constexpr int kStages = (227 * 1024 - 1024 - 384 - kScaleBytes - kEpiWarps * kTurnBytes) / kStageBytes;   // the rest is the ring
    static constexpr int kScaleOff = kStages * kStageBytes;
    static constexpr int kTurnOff = kScaleOff + kScaleBytes;
    static constexpr int kBarOff = kTurnOff + kEpiWarps * kTurnBytes;
    static constexpr int kNumBars = 3 * kStages + 4;                        // full[] empty[] tfull[2] tempty[2] ragged[]
    static constexpr int kTmemSlotOff = kBarOff + 8 * kNumBars;
    static constexpr int kAbortOff = kTmemSlotOff + 8;
    static constexpr int kDynamicBytes = kAbortOff + 8 + 1024;
    static constexpr int kTmemCols = 2 * ROWS;                              // two accumulator slots
    static_assert(8 * kNumBars + 16 <= 384 && kTmemCols <= 512, "layout");
};

// `rows` (< 32) rows of 128 bytes of a row-contiguous operand into a 32-row piece of a swizzled box, zeros behind them and
// behind the last column.  One warp.  columns is a multiple of 16.
__device__ __forceinline__ void grouped_load_ragged(uint32_t dst, const uint8_t* src, long long ld, int rows, int columns) {
    const int lane = threadIdx.x & 31;
    uint4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = i * 4 + (lane >> 3), c = (lane & 7) * 16;
        v[i] = make_uint4(0u, 0u, 0u, 0u);
        if (r < rows && c < columns) v[i] = __ldg(reinterpret_cast<const uint4*>(src + r * ld + c));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = i * 4 + (lane >> 3);
        ptx::st_shared_v4(dst + r * 128 + (((lane & 7) ^ (r & 7)) << 4), v[i].x, v[i].y, v[i].z, v[i].w);
    }
}

// OB: bytes of an element of D.  BETA: D is read too (a kernel of its own: its registers and code cost the others 8 %).
template <int MODE, int ROWS, int CTAS, int OB, bool BETA>
__global__ void __launch_bounds__(kGemmThreads, 1)
gemm_fp8_grouped_kernel(const __grid_constant__ GroupedMaps maps, const GroupedArgs args)
{
    using L = GroupedSmem<ROWS, CTAS>;
    constexpr int STAGES = L::kStages;
    constexpr bool kPair = CTAS == 2;
    constexpr bool kWMn = MODE != kGroupedForward;            // W's row index (of memory) is the contraction
    constexpr bool kRMn = MODE == kGroupedWgrad;              // ... and R's
    constexpr bool kRagged = MODE == kGroupedWgrad;           // the contraction ends inside a block
    constexpr int kStep = kPair ? 32 : 16;                    // granularity of N
    constexpr int kRBoxes = kRMn ? L::kRRows / 128 : 1;       // boxes of 128 columns of R per block (wgrad)
    static_assert(ROWS % 64 == 0 && ROWS <= 256 && (!kRMn || L::kRRows % 128 == 0), "tile");
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (ptx::smem_addr(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - ptx::smem_addr(smem_raw));

    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);   // provably warp-uniform
    const int lane = threadIdx.x & 31;
    const uint32_t rank = kPair ? ptx::cluster_ctarank() : 0u;

    const uint32_t bar_full = smem_base + L::kBarOff;
    const uint32_t bar_empty = bar_full + 8 * STAGES;
    const uint32_t bar_tfull = bar_empty + 8 * STAGES;
    const uint32_t bar_tempty = bar_tfull + 16;
    const uint32_t bar_ragged = bar_tempty + 16;
    const uint32_t tmem_slot = smem_base + L::kTmemSlotOff;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem_gen + L::kAbortOff);
    volatile uint32_t* tmem_slot_gen = reinterpret_cast<volatile uint32_t*>(smem_gen + L::kTmemSlotOff);

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < STAGES; ++s) {
            ptx::mbar_init(bar_full + 8 * s, 1);
            ptx::mbar_init(bar_empty + 8 * s, 1);
            // ragged pairs: the second CTA announces its ordinary stores to the leader, for blocks that have some only (an
            // arrival in the other CTA for every block, as a second arrival on the full barrier, halved the rate)
            ptx::mbar_init(bar_ragged + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            ptx::mbar_init(bar_tfull + 8 * b, 1);
            ptx::mbar_init(bar_tempty + 8 * b, kEpiWarps * CTAS);
        }
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&maps.w);
        ptx::prefetch_tensormap(&maps.r[3]);
    }
    if (warp == 1) {
        ptx::tmem_alloc<CTAS>(tmem_slot, L::kTmemCols);
        ptx::tmem_relinquish<CTAS>();
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (kPair) { ptx::cluster_arrive(); ptx::cluster_wait(); }
    ptx::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot_gen;
    // everything above touched only this CTA's own resources; global memory only from here on
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();

    const int step = gridDim.x / CTAS;
    const int first = blockIdx.x / CTAS;
    using Walk = GroupedWalk<MODE, ROWS, 128 * CTAS>;

    if (warp == 0) {
        // ---------------- TMA producer: warp-uniform loop, one elected lane issues ----------------
        const uint32_t full0 = kPair ? ptx::mapa(bar_full, 0) : bar_full;   // the leader's barriers
        const uint32_t ragged0 = kPair ? ptx::mapa(bar_ragged, 0) : bar_ragged;
        int s = 0, issued = 0;
        uint32_t ph = 0;
        bool ok = true;
        Walk walk(args);
        GroupedTile w;
        for (long long t = first; ok && walk.seek(t, w); t += step) {
            const int n = (w.rows + kStep - 1) / kStep * kStep;              // the MMA's N
            const int mine = n / CTAS;                                       // rows of R in this CTA
            const int col0 = w.col0 + static_cast<int>(rank) * 128, row0 = w.row0 + static_cast<int>(rank) * mine;
            const int box = kRMn ? 3 : mine > 64 ? 3 : mine > 32 ? 2 : mine > 16 ? 1 : 0;   // boxes of 16 << box rows
            const int boxes = kRMn ? kRBoxes : (mine + 127) / 128;           // one box, two for more than 128 rows
            const uint32_t block_bytes = L::kWBytes + boxes * ((16 << box) * kBlockK);
            for (int k = w.k0; k < w.k_end; k += kBlockK) {
                if (!wait_bounded(bar_empty + 8 * s, ph ^ 1u, abort_flag, kPair)) {
                    record_failure(args.status, abort_flag, kStatusProducerTimeout);
                    ok = false;
                    break;
                }
                const uint32_t w_dst = smem_base + s * L::kStageBytes;
                const uint32_t r_dst = w_dst + L::kWBytes;
                const uint32_t fullb = bar_full + 8 * s, fullr = full0 + 8 * s;
                auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y, int z) {
                    if (kPair) ptx::tma_load_3d_pair(dst, map, x, y, z, fullr);
                    else ptx::tma_load_3d(dst, map, x, y, z, fullb);
                };
                const int valid = w.k_end - k;                               // contraction left from this block on
                if (args.debug && t == first && k - w.k0 == 2 * kBlockK) {
                    // failure-path test: a slot that is never armed nor loaded, so the wait on it must run out
                } else if (kRagged && valid < kBlockK) {
                    // the block across the group's end: whole 32-row pieces by TMA, the ragged one with ordinary loads
                    const int whole = valid / 32, rest = valid % 32;
                    if (rest) {
                        const long long at = static_cast<long long>(k) + whole * 32;
                        grouped_load_ragged(w_dst + whole * 4096, args.w + at * args.ldw + col0, args.ldw, rest, args.cols - col0);
#pragma unroll
                        for (int j = 0; j < kRBoxes; ++j)
                            grouped_load_ragged(r_dst + j * 16384 + whole * 4096, args.r + at * args.ldr + row0 + j * 128, args.ldr, rest,
                                                args.d_rows - row0 - j * 128);
                        ptx::fence_proxy_async_smem();
                        __syncwarp();
                    }
                    if (ptx::elect_one()) {
                        const uint32_t bytes = whole * 4096 * (1 + kRBoxes) * CTAS;
                        if (rank != 0) { if (rest) ptx::mbar_arrive_cluster(ragged0 + 8 * s); }
                        else if (bytes) ptx::mbar_arrive_expect_tx(fullb, bytes);
                        else ptx::mbar_arrive(fullb);
                        for (int p = 0; p < whole; ++p) {
                            load(w_dst + p * 4096, &maps.w32, col0, k + p * 32, 0);
#pragma unroll
                            for (int j = 0; j < kRBoxes; ++j)
                                load(r_dst + j * 16384 + p * 4096, &maps.r32, row0 + j * 128, k + p * 32, 0);
                        }
                    }
                } else if (ptx::elect_one()) {
                    if (rank == 0) ptx::mbar_arrive_expect_tx(fullb, block_bytes * CTAS);
                    if (kWMn) load(w_dst, &maps.w, col0, k, MODE == kGroupedWgrad ? 0 : w.e);
                    else load(w_dst, &maps.w, k, col0, w.e);
                    if (kRMn) {
#pragma unroll
                        for (int j = 0; j < kRBoxes; ++j) load(r_dst + j * 16384, &maps.r[3], row0 + j * 128, k, 0);
                    } else {
                        load(r_dst, &maps.r[box], k, row0, 0);
                        if (L::kRRows > 128 && boxes > 1) load(r_dst + 16384, &maps.r[3], k, row0 + 128, 0);
                    }
                }
                __syncwarp();
                ++issued;
                if (++s == STAGES) { s = 0; ph ^= 1u; }
            }
        }
        if (!ok && rank == 0) {
            // leave no copy in flight into this CTA's shared memory: wait (bounded) for the stages armed last
            const int pending = issued < STAGES ? issued : STAGES;
            for (int i = 0; i < pending; ++i) {
                if (s == 0) { s = STAGES; ph ^= 1u; }
                --s;
                const uint64_t t0 = ptx::globaltimer_ns();
                while (!ptx::mbar_try_wait(bar_full + 8 * s, ph) && ptx::globaltimer_ns() - t0 < kWaitLimitNs) {}
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer: leader CTA, warp-uniform loop, one elected lane issues ----------------
        if (rank == 0) {
            int s = 0, it = 0;                                    // `it` counts tiles that have an accumulator
            uint32_t ph = 0, ragged_ph = 0;                       // the latter one bit per slot
            bool ok = true;
            Walk walk(args);
            GroupedTile w;
            for (long long t = first; ok && walk.seek(t, w); t += step) {
                if (w.k0 >= w.k_end) continue;                    // a group without rows: the epilogue stores zeros
                const int slot = it & 1;
                if (!wait_bounded(bar_tempty + 8 * slot, static_cast<uint32_t>((it >> 1) & 1) ^ 1u, abort_flag, kPair)) {
                    record_failure(args.status, abort_flag, kStatusMmaTimeout);
                    break;
                }
                ptx::tc_fence_after();
                const uint32_t d_tmem = tmem_base + slot * ROWS;
                const uint32_t idesc = args.idesc | (static_cast<uint32_t>((w.rows + kStep - 1) / kStep * kStep) >> 3) << 17;
                for (int k = w.k0; k < w.k_end; k += kBlockK) {
                    if (!wait_bounded(bar_full + 8 * s, ph, abort_flag, kPair)) {
                        record_failure(args.status, abort_flag, kStatusMmaTimeout);
                        ok = false;
                        break;
                    }
                    if (kRagged && kPair && w.k_end - k < kBlockK && (w.k_end - k) % 32 != 0) {
                        if (!wait_bounded(bar_ragged + 8 * s, (ragged_ph >> s) & 1u, abort_flag, true)) {
                            record_failure(args.status, abort_flag, kStatusMmaTimeout);
                            ok = false;
                            break;
                        }
                        ragged_ph ^= 1u << s;
                    }
                    ptx::tc_fence_after();
                    const uint32_t w_src = smem_base + s * L::kStageBytes;
                    const uint32_t r_src = w_src + L::kWBytes;
                    const uint64_t wdesc = kWMn ? ptx::umma_desc_mn128(w_src, 16384) : ptx::umma_desc_k128(w_src);
                    const uint64_t rdesc = kRMn ? ptx::umma_desc_mn128(r_src, 16384) : ptx::umma_desc_k128(r_src);
                    const int steps = min(kBlockK / 32, (w.k_end - k + 31) / 32);
                    if (ptx::elect_one()) {
#pragma unroll
                        for (int i = 0; i < kBlockK / 32; ++i)    // 32 of the contraction per instruction: 32 bytes or 32 rows
                            if (i < steps)
                                ptx::umma_f8<CTAS>(d_tmem, wdesc + (kWMn ? 256 : 2) * i, rdesc + (kRMn ? 256 : 2) * i, idesc, k != w.k0 || i != 0);
                        if (kPair) ptx::umma_commit_pair(bar_empty + 8 * s, 0x3);
                        else ptx::umma_commit(bar_empty + 8 * s);
                    }
                    __syncwarp();
                    if (++s == STAGES) { s = 0; ph ^= 1u; }
                }
                if (ok && ptx::elect_one()) {
                    if (kPair) ptx::umma_commit_pair(bar_tfull + 8 * slot, 0x3);
                    else ptx::umma_commit(bar_tfull + 8 * slot);
                }
                __syncwarp();
                ++it;
            }
        }
    } else {
        // ---------------- epilogue warps: a lane owns a column, the registers run along the rows ----------------
        const int q = warp & 3;                                   // TMEM lane quarter this warp may read
        const int grp = (warp - 2) >> 2;                          // 0 or 1: every second chunk of 32 rows
        const uint32_t tempty0 = kPair ? ptx::mapa(bar_tempty, 0) : bar_tempty;
        const uint32_t turn = smem_base + L::kTurnOff + (warp - 2) * L::kTurnBytes;
        float* row_scales = reinterpret_cast<float*>(smem_gen + L::kScaleOff) + (warp - 2) * (ROWS / 2);
        const int out_dtype = args.epi.out_dtype;
        float alpha0 = args.epi.alpha, dscale = 1.0f, amax = 0.0f;
        if (args.epi.a_scale) alpha0 *= *args.epi.a_scale;
        if (args.epi.b_scale) alpha0 *= *args.epi.b_scale;
        if (args.epi.d_scale) dscale = *args.epi.d_scale;
        // what few calls ask for sits behind one branch
        const bool more = BETA || args.epi.activation != 0 || args.epi.amax != nullptr || args.epi.d_scale != nullptr;
        // This lane's columns of a tile: one, or four for 16-bit outputs.
        constexpr int kCols = OB == 2 ? 4 : 1;
        auto col_of = [&](const GroupedTile& w, int m) {
            return w.col0 + static_cast<int>(rank) * 128 + q * 32 + (OB == 2 ? 8 * m + (lane >> 2) : lane);
        };
        // A tile's scales and bias are asked for one tile ahead and converted when its turn comes: their latency, once per
        // tile, cost 10629 x 7792 x 448 in two groups 79 us where 57 are enough.
        float next_scale[kCols], next_row[ROWS / 64];
        uint32_t next_bias[kCols];
        auto ask = [&](const GroupedTile& w) {
#pragma unroll
            for (int m = 0; m < kCols; ++m) {
                const long long vec = static_cast<long long>(w.e) * args.cols + col_of(w, m);   // b_row_scale, bias: [E][cols]
                const bool in = col_of(w, m) < args.cols;
                next_scale[m] = in && args.epi.b_row_scale != nullptr ? __ldg(args.epi.b_row_scale + vec) : 1.0f;
                next_bias[m] = 0u;
                if (in && args.epi.bias != nullptr)
                    next_bias[m] = args.epi.bias_dtype == 0 ? __ldg(static_cast<const unsigned int*>(args.epi.bias) + vec)
                                                            : __ldg(static_cast<const unsigned short*>(args.epi.bias) + vec);
            }
#pragma unroll
            for (int i = 0; i < ROWS / 64; ++i) {                 // this warp's chunks: grp, grp + 2, ...
                const int r = (2 * i + grp) * 32 + lane;
                next_row[i] = args.epi.a_row_scale != nullptr && r < w.rows ? __ldg(args.epi.a_row_scale + w.row0 + r) : 0.0f;
                if (BETA && r < w.rows && w.col0 + static_cast<int>(rank) * 128 + q * 32 < args.cols)
                    ptx::prefetch_l2(static_cast<const char*>(args.d) + OB * ((MODE == kGroupedWgrad ? w.e * args.stride_d : 0) +
                                     (static_cast<long long>(w.row0) + r) * args.ldd + w.col0 + static_cast<int>(rank) * 128 + q * 32));
            }
        };
        int it = 0;
        Walk walk(args);
        GroupedTile w, next;
        bool have = walk.seek(first, next);
        if (have) ask(next);
        for (long long t = first; have; t += step) {
            w = next;
            const bool empty = w.k0 >= w.k_end;
            const int slot = it & 1;
            const int chunks = (w.rows + 31) / 32;
            const int col_base = w.col0 + static_cast<int>(rank) * 128 + q * 32;         // of this warp
            auto col = [&](int m) { return col_of(w, m); };
            float factor[kCols], bias[kCols];
#pragma unroll
            for (int m = 0; m < kCols; ++m) {
                factor[m] = alpha0 * next_scale[m];
                bias[m] = args.epi.bias_dtype == 0 ? __uint_as_float(next_bias[m])
                        : args.epi.bias_dtype == 1 ? __uint_as_float(next_bias[m] << 16)
                                                   : __half2float(__ushort_as_half(static_cast<unsigned short>(next_bias[m])));
            }
            if (args.epi.a_row_scale != nullptr) {                // chunk c at 16 c in this warp's own array
                __syncwarp();
#pragma unroll
                for (int i = 0; i < ROWS / 64; ++i) row_scales[i * 32 + lane] = next_row[i];
                __syncwarp();
            }
            have = walk.seek(t + step, next);
            if (have) ask(next);
            if (!empty) {
                if (!wait_bounded(bar_tfull + 8 * slot, static_cast<uint32_t>((it >> 1) & 1), abort_flag, kPair)) {
                    record_failure(args.status, abort_flag, kStatusEpilogueTimeout);
                    break;
                }
                __syncwarp();
                ptx::tc_fence_after();
                ++it;
            }
            const uint32_t t_addr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + slot * ROWS;
            const long long d_base = (MODE == kGroupedWgrad ? w.e * args.stride_d : 0) + static_cast<long long>(w.row0) * args.ldd;   // elements

            // Element i of a lane: its row within the chunk and which of its columns.  16-bit outputs: register 16 h + 4 j + 2 u + s
            // is row 8 j + 2 (lane % 4) + s of column block 2 h + u.
            auto row_of = [&](int i) { return OB == 2 ? 8 * ((i >> 2) & 3) + 2 * (lane & 3) + (i & 1) : i; };
            auto block_of = [&](int i) { return OB == 2 ? 2 * (i >> 4) + ((i >> 1) & 1) : 0; };
            uint32_t v[32];
#pragma unroll 1
            for (int c = grp; c < chunks; c += 2) {
                const int rows = min(32, w.rows - c * 32);
                const long long at = d_base + static_cast<long long>(c) * 32 * args.ldd;
                // What D holds, for beta: all loads in flight at once (one by one they took ten times as long as the rest of wgrad),
                // from L2, where they were asked for a tile ahead.  16-bit rows come 16 bytes per lane, as they go.
                [[maybe_unused]] uint32_t old[32];
                if constexpr (BETA) {
                    if (OB == 2 && args.wide_store) {
                        const bool in = col_base + 8 * (lane & 3) < args.cols;
                        const uint16_t* from = static_cast<const uint16_t*>(args.d) + at + (lane >> 2) * args.ldd + col_base + 8 * (lane & 3);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            uint4 four = make_uint4(0u, 0u, 0u, 0u);
                            if (in && 8 * i + (lane >> 2) < rows) four = __ldcg(reinterpret_cast<const uint4*>(from + 8 * i * args.ldd));
                            old[4 * i] = four.x; old[4 * i + 1] = four.y; old[4 * i + 2] = four.z; old[4 * i + 3] = four.w;
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const long long from = at + row_of(i) * args.ldd + col(block_of(i));
                            old[i] = 0u;
                            if (row_of(i) < rows && col(block_of(i)) < args.cols) {
                                if constexpr (OB == 4) old[i] = __ldcg(static_cast<const unsigned int*>(args.d) + from);
                                else if constexpr (OB == 2) old[i] = __ldcg(static_cast<const unsigned short*>(args.d) + from);
                                else old[i] = __ldcg(static_cast<const unsigned char*>(args.d) + from);
                            }
                        }
                    }
                }
                if (empty) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = 0u;
                } else {
                    if constexpr (OB == 2) {
                        ptx::tmem_ld_16x32(t_addr + c * 32, v);
                        ptx::tmem_ld_16x32(t_addr + (16u << 16) + c * 32, v + 16);
                    } else {
                        ptx::tmem_ld_32x32(t_addr + c * 32, v);
                    }
                    ptx::tmem_ld_wait();
                }
                if (args.epi.a_row_scale != nullptr) {
                    const float* ra = row_scales + (c >> 1) * 32;
                    if constexpr (OB == 2) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float2 f = *reinterpret_cast<const float2*>(ra + 8 * j + 2 * (lane & 3));
#pragma unroll
                            for (int m = 0; m < 4; ++m) {
                                uint32_t* p = v + 16 * (m >> 1) + 4 * j + 2 * (m & 1);
                                p[0] = __float_as_uint(__uint_as_float(p[0]) * f.x);
                                p[1] = __float_as_uint(__uint_as_float(p[1]) * f.y);
                            }
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float4 f = reinterpret_cast<const float4*>(ra)[i];   // one address for all lanes
                            v[4 * i] = __float_as_uint(__uint_as_float(v[4 * i]) * f.x);
                            v[4 * i + 1] = __float_as_uint(__uint_as_float(v[4 * i + 1]) * f.y);
                            v[4 * i + 2] = __float_as_uint(__uint_as_float(v[4 * i + 2]) * f.z);
                            v[4 * i + 3] = __float_as_uint(__uint_as_float(v[4 * i + 3]) * f.w);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(fmaf(factor[block_of(i)], __uint_as_float(v[i]), bias[block_of(i)]));
                if (more) {
                    if constexpr (BETA) {
                        auto add = [&](uint32_t& sum, float d) { sum = __float_as_uint(fmaf(args.epi.beta, d, __uint_as_float(sum))); };
                        if (OB == 2 && args.wide_store) {
                            __syncwarp();                         // the chunk before has been read
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int r = 8 * i + (lane >> 2);
                                ptx::st_shared_v4(turn + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4), old[4 * i], old[4 * i + 1], old[4 * i + 2], old[4 * i + 3]);
                            }
                            __syncwarp();
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                uint32_t p[4];
                                ptx::ldmatrix_x4_trans(turn + 512 * j + (lane & 7) * 64 + (((lane >> 3) ^ ((lane >> 1) & 3)) << 4), p);
#pragma unroll
                                for (int m = 0; m < 4; ++m) {
                                    uint32_t* s = v + 16 * (m >> 1) + 4 * j + 2 * (m & 1);
                                    add(s[0], wide16(p[m], out_dtype));
                                    add(s[1], wide16(p[m] >> 16, out_dtype));
                                }
                            }
                        } else if constexpr (OB == 4) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) add(v[i], __uint_as_float(old[i]));
                        } else if constexpr (OB == 2) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) add(v[i], wide16(old[i], out_dtype));
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(old[i]), out_dtype == 3 ? __NV_E4M3 : __NV_E5M2);
                                add(v[i], __half2float(__half(h)));
                            }
                        }
                    }
                    if (args.epi.activation == 1) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(relu(__uint_as_float(v[i])));
                    } else if (args.epi.activation == 2) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(gelu_erf(__uint_as_float(v[i])));
                    } else if (args.epi.activation == 3) {
#pragma unroll
                        for (int i = 0; i < 32; i += 2) grouped_gelu_tanh(v[i], v[i + 1]);
                    }
                    if (args.epi.amax != nullptr) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (row_of(i) < rows && col(block_of(i)) < args.cols) amax = fmaxf(amax, fabsf(__uint_as_float(v[i])));
                    }
                    if (args.epi.d_scale != nullptr) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(dscale * __uint_as_float(v[i]));
                    }
                }
                if constexpr (OB == 2) {
                    // rows of 64 bytes, 16-byte chunk ^ (row / 2) mod 4: neither side has bank conflicts
                    __syncwarp();                                 // the chunk before has been read
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t p[4];
#pragma unroll
                        for (int m = 0; m < 4; ++m) {
                            const uint32_t* s = v + 16 * (m >> 1) + 4 * j + 2 * (m & 1);
                            p[m] = pack16(__uint_as_float(s[0]), __uint_as_float(s[1]), out_dtype);
                        }
                        ptx::stmatrix_x4_trans(turn + 512 * j + (lane & 7) * 64 + (((lane >> 3) ^ ((lane >> 1) & 3)) << 4), p[0], p[1], p[2], p[3]);
                    }
                    __syncwarp();
                    if (args.wide_store) {
                        const int chunk = lane & 3;                   // eight columns
                        const bool in = col_base + 8 * chunk < args.cols;
                        char* to = reinterpret_cast<char*>(static_cast<uint16_t*>(args.d) + at + (lane >> 2) * args.ldd + col_base + 8 * chunk);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int r = 8 * i + (lane >> 2);
                            const uint4 two = ptx::ld_shared_v4(turn + r * 64 + ((chunk ^ ((r >> 1) & 3)) << 4));
                            if (in && r < rows) *reinterpret_cast<uint4*>(to) = two;
                            to += 16 * args.ldd;                      // eight rows, in bytes
                        }
                    } else {                                      // a row's 64 bytes from 32 lanes
                        const bool in = col_base + lane < args.cols;
                        uint16_t* to = static_cast<uint16_t*>(args.d) + at + col_base + lane;
#pragma unroll 8
                        for (int r = 0; r < rows; ++r, to += args.ldd) {
                            const uint16_t one = ptx::ld_shared_u16(turn + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) << 4) + 2 * (lane & 7));
                            if (in) *to = one;
                        }
                    }
                } else if (OB == 1 && args.wide_store) {
                    // four rows of this lane's column to a word, 4 x 4 bytes transposed between four lanes: row 4 j + lane % 4, four columns
                    uint32_t b[8];
                    if (out_dtype == 3) grouped_pack8<__NV_E4M3>(v, b);
                    else grouped_pack8<__NV_E5M2>(v, b);
                    const uint32_t first = lane & 1 ? 0x3715u : 0x6240u, second = lane & 2 ? 0x3276u : 0x5410u;
                    const bool in = col_base + (lane & ~3) < args.cols;
                    uint8_t* to = static_cast<uint8_t*>(args.d) + at + (lane & 3) * args.ldd + col_base + (lane & ~3);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        b[j] = __byte_perm(b[j], __shfl_xor_sync(0xffffffffu, b[j], 1), first);
                        b[j] = __byte_perm(b[j], __shfl_xor_sync(0xffffffffu, b[j], 2), second);
                        if (in && 4 * j + (lane & 3) < rows) *reinterpret_cast<uint32_t*>(to) = b[j];
                        to += 4 * args.ldd;
                    }
                } else if (OB == 4 && rows == 32) {
                    if (col_base + lane < args.cols) {
                        float* to = static_cast<float*>(args.d) + at + col_base + lane;
#pragma unroll
                        for (int i = 0; i < 32; ++i, to += args.ldd) *to = __uint_as_float(v[i]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (row_of(i) < rows && col(block_of(i)) < args.cols)
                            store_out(args.d, at + row_of(i) * args.ldd + col(block_of(i)), __uint_as_float(v[i]), OB == 4 ? 0 : out_dtype);
                }
            }
            if (!empty) {                                         // this warp's part of the accumulator has been read
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (kPair) ptx::mbar_arrive_cluster(tempty0 + 8 * slot);
                    else ptx::mbar_arrive(bar_tempty + 8 * slot);
                }
            }
        }
        __syncwarp();
        if (args.epi.amax != nullptr) amax_merge_warp(args.epi.amax, amax);
    }

    // ---------------- teardown ----------------
    ptx::tc_fence_before();
    __syncthreads();
    if (kPair) { ptx::cluster_arrive(); ptx::cluster_wait(); }
    if (warp == 1) {
        __syncwarp();
        ptx::tc_fence_after();
        ptx::tmem_dealloc<CTAS>(tmem_base, L::kTmemCols);
    }
}

}  // namespace b200fp8
