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
// slots -- with a walk over tiles that every warp derives from `ends` by itself (32 groups at a time in the lanes of a
// warp, one scan and one ballot per tile), so there is no schedule to build, no workspace and no second launch.
//
//   * Rows behind a group's end inside a tile belong to the next group.  Forward and dgrad multiply them (each row of a
//     product depends on its own row of A only) and do not store them: 32-row boxes that lie inside the group go out
//     by TMA, the box across the end by masked stores.  A one-CTA tile picks the shortest of four A boxes (16, 32, 64,
//     128 rows) that covers its rows, so a decode step's few rows per expert cost few bytes next to the weights.
//   * wgrad contracts over the rows, so the block across a group's end must not see the next group: it is loaded as 32-row
//     TMA boxes, and the last, ragged 32 rows with ordinary loads that put zeros behind the end (a product with
//     zero would not do: the other operand's foreign rows may hold infinities or NaN).  The MMA issues only as many
//     K = 32 steps as there are rows.  A group without rows stores zeros (or beta * D).
//
// Every wait on an mbarrier is bounded, as in the dense kernel.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cstdint>
#include "gemm_sm100.cuh"

namespace b200fp8 {

enum GroupedMode : int { kGroupedForward = 0, kGroupedDgrad = 1, kGroupedWgrad = 2 };

struct GroupedMaps {
    CUtensorMap a[4];     // forward, dgrad: boxes of 16, 32, 64, 128 rows; wgrad: [1] 32 rows, [3] 128 rows
    CUtensorMap b;        // forward: BN / CTAS rows of 128 bytes; dgrad, wgrad: 128 rows of 128 bytes
    CUtensorMap b32;      // wgrad: 32 rows
    CUtensorMap d;        // 32 x 32 boxes of D
};

struct GroupedArgs {
    int experts;
    int rows;             // rows of the ragged operands
    int tile_rows_all;    // wgrad: rows of D per expert (N)
    int cols;             // columns of D
    int depth;            // contraction extent: K forward, N dgrad (wgrad: the group's rows)
    const int* ends;
    int m_tiles;          // wgrad: tiles along the rows of D[e]
    int n_tiles;
    int group_m;          // forward, dgrad: tiles are walked down `group_m` M-tiles before moving along the columns
    uint32_t idesc;
    int tma_store;
    void* d;
    long long ldd, stride_d;
    const uint8_t* a;     // wgrad: base pointers of the ragged rows' ordinary loads
    const uint8_t* b;
    long long lda, ldb;
    int a_cols;
    int* status;
    Epilogue epi;
};

// One tile: expert, position, and what it multiplies.
struct GroupedTile {
    int e;
    int row0;     // forward, dgrad: first row of the tile in A and D; wgrad: first row of the tile in D[e]
    int row_end;  // first row that is not the tile's to store
    int n0;
    int k0, k_end;   // contraction range (wgrad: rows of the group)
};

// Walk over the tiles of all groups in order.  All 32 lanes call it together.
template <int MODE, int TILE_M, int BN>
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
        if (MODE == kGroupedWgrad) upto = e < args.experts ? args.m_tiles * args.n_tiles : 0;
        else upto = (end - start + TILE_M - 1) / TILE_M * args.n_tiles;
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
        const int m_tiles = MODE == kGroupedWgrad ? args.m_tiles : (f - s + TILE_M - 1) / TILE_M;
        const int per_group = args.group_m * args.n_tiles;
        const int g = r / per_group;
        const int first_m = g * args.group_m;
        const int gsz = min(args.group_m, m_tiles - first_m);
        const int in_group = r - g * per_group;
        const int m0 = (first_m + in_group % gsz) * TILE_M;
        w.n0 = in_group / gsz * BN;
        if (MODE == kGroupedWgrad) {
            w.row0 = m0;
            w.row_end = args.tile_rows_all;
            w.k0 = s;
            w.k_end = f;
        } else {
            w.row0 = s + m0;
            w.row_end = f;
            w.k0 = 0;
            w.k_end = args.depth;
        }
        return true;
    }
};

// OB: bytes of an output element
template <int BN, int CTAS, int OB>
struct GroupedSmem {
    static constexpr int kABytes = kTileM * kBlockK;
    static constexpr int kBRows = BN / CTAS;
    static constexpr int kBBytes = kBRows * kBlockK;
    static constexpr int kStageBytes = kABytes + kBBytes;
    // An epilogue warp stores 32 rows x BN / 2 columns as boxes of 32 rows x 128 bytes (64 for 8-bit outputs), through two
    // staging buffers where it has two boxes or more: a box is written while the one before it is still read.
    static constexpr int kBoxCols = OB == 4 ? 32 : 64;
    static constexpr int kBoxes = BN / 2 / kBoxCols;
    static constexpr int kBuffers = kBoxes >= 2 ? 2 : 1;
    static constexpr int kEpiBufBytes = 4096;
    static constexpr int kEpiBytes = kEpiWarps * kBuffers * kEpiBufBytes;
    static constexpr int kStages = (227 * 1024 - 1024 - 256 - kEpiBytes) / kStageBytes;   // what is left is the ring
    static constexpr int kEpiOff = kStages * kStageBytes;
    static constexpr int kBarOff = kEpiOff + kEpiBytes;
    static constexpr int kNumBars = 3 * kStages + 4;          // full[] empty[] tfull[2] tempty[2] ragged[]
    static constexpr int kTmemSlotOff = kBarOff + 8 * kNumBars;
    static constexpr int kAbortOff = kTmemSlotOff + 8;
    static constexpr int kDynamicBytes = kAbortOff + 8 + 1024;
    static constexpr int kTmemCols = 2 * BN;
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

template <int MODE, int BN, int CTAS, int OB>
__global__ void __launch_bounds__(kGemmThreads, 1)
gemm_fp8_grouped_kernel(const __grid_constant__ GroupedMaps maps, const GroupedArgs args)
{
    using L = GroupedSmem<BN, CTAS, OB>;
    constexpr int STAGES = L::kStages;
    constexpr bool kPair = CTAS == 2;
    constexpr bool kAMn = MODE == kGroupedWgrad;              // A's row index is the contiguous one
    constexpr bool kBMn = MODE != kGroupedForward;
    constexpr bool kRagged = MODE == kGroupedWgrad;           // the contraction ends inside a block
    static_assert(BN % 64 == 0 && BN <= 256 && (!kBMn || L::kBRows % 128 == 0), "tile");
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
        ptx::prefetch_tensormap(&maps.a[3]);
        ptx::prefetch_tensormap(&maps.b);
        ptx::prefetch_tensormap(&maps.d);
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
    using Walk = GroupedWalk<MODE, kTileM * CTAS, BN>;

    if (warp == 0) {
        // ---------------- TMA producer: warp-uniform loop, one elected lane issues ----------------
        const uint32_t full0 = kPair ? ptx::mapa(bar_full, 0) : bar_full;   // the leader's full barriers
        const uint32_t ragged0 = kPair ? ptx::mapa(bar_ragged, 0) : bar_ragged;
        int s = 0, issued = 0;
        uint32_t ph = 0;
        bool ok = true;
        Walk walk(args);
        GroupedTile w;
        for (long long t = first; ok && walk.seek(t, w); t += step) {
            const int row0 = w.row0 + static_cast<int>(rank) * kTileM;       // this CTA's rows of the tile
            const int nb0 = w.n0 + static_cast<int>(rank) * L::kBRows;
            int box = 3;                                                     // A boxes of 16 << box rows
            if (!kPair && !kRagged) {
                const int have = w.row_end - row0;
                box = have > 64 ? 3 : have > 32 ? 2 : have > 16 ? 1 : 0;
            }
            const uint32_t block_bytes = kRagged ? L::kStageBytes : (16 << box) * kBlockK + L::kBBytes;
            for (int k = w.k0; k < w.k_end; k += kBlockK) {
                if (!wait_bounded(bar_empty + 8 * s, ph ^ 1u, abort_flag, kPair)) {
                    record_failure(args.status, abort_flag, kStatusProducerTimeout);
                    ok = false;
                    break;
                }
                const uint32_t a_dst = smem_base + s * L::kStageBytes;
                const uint32_t b_dst = a_dst + L::kABytes;
                const uint32_t fullb = bar_full + 8 * s, fullr = full0 + 8 * s;
                auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y, int z) {
                    if (kPair) ptx::tma_load_3d_pair(dst, map, x, y, z, fullr);
                    else ptx::tma_load_3d(dst, map, x, y, z, fullb);
                };
                const int valid = w.k_end - k;                               // contraction left from this block on
                if (kRagged && valid < kBlockK) {
                    // the block across the group's end: whole 32-row pieces by TMA, the ragged one with ordinary loads
                    const int whole = valid / 32, rest = valid % 32;
                    if (rest) {
                        grouped_load_ragged(a_dst + whole * 4096, args.a + (static_cast<long long>(k) + whole * 32) * args.lda + row0, args.lda, rest, args.a_cols - row0);
#pragma unroll
                        for (int j = 0; j < L::kBRows / 128; ++j)
                            grouped_load_ragged(b_dst + j * 16384 + whole * 4096, args.b + (static_cast<long long>(k) + whole * 32) * args.ldb + nb0 + j * 128,
                                                args.ldb, rest, args.cols - nb0 - j * 128);
                        ptx::fence_proxy_async_smem();
                        __syncwarp();
                    }
                    if (ptx::elect_one()) {
                        const uint32_t bytes = whole * 4096 * (1 + L::kBRows / 128) * CTAS;
                        if (rank != 0) { if (rest) ptx::mbar_arrive_cluster(ragged0 + 8 * s); }
                        else if (bytes) ptx::mbar_arrive_expect_tx(fullb, bytes);
                        else ptx::mbar_arrive(fullb);
                        for (int p = 0; p < whole; ++p) {
                            load(a_dst + p * 4096, &maps.a[1], row0, k + p * 32, 0);
#pragma unroll
                            for (int j = 0; j < L::kBRows / 128; ++j)
                                load(b_dst + j * 16384 + p * 4096, &maps.b32, nb0 + j * 128, k + p * 32, 0);
                        }
                    }
                } else if (ptx::elect_one()) {
                    if (rank == 0) ptx::mbar_arrive_expect_tx(fullb, block_bytes * CTAS);
                    if (kAMn) load(a_dst, &maps.a[3], row0, k, 0);
                    else load(a_dst, &maps.a[box], k, row0, 0);
                    if (!kBMn) load(b_dst, &maps.b, k, nb0, w.e);
                    else {
#pragma unroll
                        for (int j = 0; j < L::kBRows / 128; ++j)
                            load(b_dst + j * 16384, &maps.b, nb0 + j * 128, k, MODE == kGroupedWgrad ? 0 : w.e);
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
                const uint32_t d_tmem = tmem_base + slot * BN;
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
                    const uint32_t a_src = smem_base + s * L::kStageBytes;
                    const uint32_t b_src = a_src + L::kABytes;
                    const uint64_t adesc = kAMn ? ptx::umma_desc_mn128(a_src, L::kABytes) : ptx::umma_desc_k128(a_src);
                    const uint64_t bdesc = kBMn ? ptx::umma_desc_mn128(b_src, 16384) : ptx::umma_desc_k128(b_src);
                    const int steps = min(kBlockK / 32, (w.k_end - k + 31) / 32);
                    if (ptx::elect_one()) {
#pragma unroll
                        for (int i = 0; i < kBlockK / 32; ++i)    // 32 of the contraction per instruction: 32 bytes or 32 rows
                            if (i < steps)
                                ptx::umma_f8<CTAS>(d_tmem, adesc + (kAMn ? 256 : 2) * i, bdesc + (kBMn ? 256 : 2) * i, args.idesc,
                                                   k != w.k0 || i != 0);
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
        // ---------------- epilogue warps ----------------
        const int q = warp & 3;                                   // TMEM lane quarter this warp may read
        const int grp = (warp - 2) >> 2;                          // 0 or 1: which half of the tile's columns
        const uint32_t staging = smem_base + L::kEpiOff + (warp - 2) * L::kBuffers * L::kEpiBufBytes;
        const uint32_t tempty0 = kPair ? ptx::mapa(bar_tempty, 0) : bar_tempty;
        const bool issuer = ptx::elect_one();                    // this lane owns the warp's bulk-store groups
        constexpr int kChunks = BN / 64;                          // 32-column chunks this warp drains per tile
        constexpr int kChunksPerBox = L::kBoxCols / 32;
        const int out_dtype = args.epi.out_dtype;
        float alpha0 = args.epi.alpha, dscale = 1.0f, amax = 0.0f;
        if (args.epi.a_scale) alpha0 *= *args.epi.a_scale;
        if (args.epi.b_scale) alpha0 *= *args.epi.b_scale;
        if (args.epi.d_scale) dscale = *args.epi.d_scale;
        // what few calls ask for sits behind one branch
        const bool more = args.epi.beta != 0.0f || args.epi.activation != 0 || args.epi.amax != nullptr || args.epi.d_scale != nullptr;
        int box = 0;                                              // boxes stored so far: they take turns in the staging buffers
        int it = 0;
        Walk walk(args);
        GroupedTile w;
        for (long long t = first; walk.seek(t, w); t += step) {
            const bool empty = w.k0 >= w.k_end;
            const int row0 = w.row0 + static_cast<int>(rank) * kTileM + q * 32;
            const int rows = min(32, w.row_end - row0);          // rows of this warp's boxes to store (may be <= 0)
            const int slot = it & 1;
            if (!empty) {
                if (!wait_bounded(bar_tfull + 8 * slot, static_cast<uint32_t>((it >> 1) & 1), abort_flag, kPair)) {
                    record_failure(args.status, abort_flag, kStatusEpilogueTimeout);
                    break;
                }
                __syncwarp();
                ptx::tc_fence_after();
                ++it;
            }
            const uint32_t t_addr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + slot * BN + grp * (BN / 2);
            const long long d_base = MODE == kGroupedWgrad ? w.e * args.stride_d : 0;   // elements
            const long long vec_base = static_cast<long long>(w.e) * args.cols;         // b_row_scale, bias: [E][cols]
            const int z = MODE == kGroupedWgrad ? w.e : 0;
            const float alpha = (args.epi.a_row_scale != nullptr && lane < rows) ? alpha0 * __ldg(args.epi.a_row_scale + row0 + lane) : alpha0;

            // a box across a group's end must not reach the next group's rows: masked stores; a box across the end of D
            // itself (wgrad: of D[e]) is clipped by the hardware
            const bool by_tma = args.tma_store && (rows == 32 || (MODE == kGroupedWgrad && rows > 0));
            auto scale = [&](uint32_t (&v)[32], int col0) {
                if (args.epi.b_row_scale != nullptr) {
                    const float mine = (col0 + lane < args.cols) ? __ldg(args.epi.b_row_scale + vec_base + col0 + lane) : 1.0f;
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__shfl_sync(0xffffffffu, mine, i) * __uint_as_float(v[i]));
                }
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(alpha * __uint_as_float(v[i]));
                if (more && args.epi.beta != 0.0f && lane < rows) {
                    const long long at = d_base + static_cast<long long>(row0 + lane) * args.ldd + col0;
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (col0 + i < args.cols) v[i] = __float_as_uint(fmaf(args.epi.beta, load_out(args.d, at + i, out_dtype), __uint_as_float(v[i])));
                }
                if (args.epi.bias != nullptr) {
                    const float mine = (col0 + lane < args.cols) ? load_out(args.epi.bias, vec_base + col0 + lane, args.epi.bias_dtype) : 0.0f;
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) + __shfl_sync(0xffffffffu, mine, i));
                }
                if (!more) return;
                if (args.epi.activation == 1) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(relu(__uint_as_float(v[i])));
                } else if (args.epi.activation == 2) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(gelu_erf(__uint_as_float(v[i])));
                } else if (args.epi.activation == 3) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(gelu_tanh(__uint_as_float(v[i])));
                }
                if (args.epi.amax != nullptr && lane < rows) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (col0 + i < args.cols) amax = fmaxf(amax, fabsf(__uint_as_float(v[i])));
                }
                if (args.epi.d_scale != nullptr) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(dscale * __uint_as_float(v[i]));
                }
            };
            // Chunk c in registers -> its box; `next` starts the load of the chunk behind it as soon as the registers are free.
            auto emit = [&](uint32_t (&v)[32], int c, auto next) {
                const int col0 = w.n0 + grp * (BN / 2) + c * 32;
                const uint32_t sb = staging + (L::kBuffers == 2 ? (box & 1) * L::kEpiBufBytes : 0);
                const int part = c % kChunksPerBox;
                if (by_tma) {
                    constexpr int kWords = 8 * OB;                // of this chunk per row
                    uint32_t p[kWords];
                    if constexpr (OB == 4) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) p[i] = v[i];
                    } else if constexpr (OB == 2) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) p[i] = pack16(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]), out_dtype);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            p[i] = pack8(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]), __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]), out_dtype);
                    }
                    next();
                    if (part == 0) {                              // the box that used this buffer before has been read
                        if (issuer) ptx::bulk_wait_group_read<L::kBuffers - 1>();
                        __syncwarp();
                    }
                    // rows of 128 bytes under the 128-byte swizzle, of 64 under the 64-byte one: no bank conflicts
                    const uint32_t at = sb + lane * (L::kBoxCols * OB);
                    const int swizzle = OB == 1 ? (lane >> 1) & 3 : lane & 7;
#pragma unroll
                    for (int i = 0; i < kWords / 4; ++i)
                        ptx::st_shared_v4(at + (((part * (kWords / 4) + i) ^ swizzle) << 4), p[4 * i], p[4 * i + 1], p[4 * i + 2], p[4 * i + 3]);
                    if (part == kChunksPerBox - 1) {
                        ptx::fence_proxy_async_smem();
                        __syncwarp();
                        const int box0 = col0 - part * 32;
                        if (issuer) {
                            if (box0 < args.cols) ptx::tma_store_3d(&maps.d, sb, box0, row0, z);
                            ptx::bulk_commit_group();
                        }
                        ++box;
                    }
                } else {
                    if (issuer) ptx::bulk_wait_group_read<0>();
                    __syncwarp();
                    const uint32_t at = sb + lane * 128;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        ptx::st_shared_v4(at + ((i ^ (lane & 7)) << 4), v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                    next();
                    __syncwarp();
                    const int col = col0 + lane;                  // one instruction writes 32 elements of one row
                    if (col < args.cols) {
                        long long to = d_base + static_cast<long long>(row0) * args.ldd + col;
                        for (int r = 0; r < rows; ++r, to += args.ldd) {
                            const uint32_t bits = ptx::ld_shared_u32(sb + r * 128 + ((((lane >> 2) ^ (r & 7)) << 4) | ((lane & 3) << 2)));
                            store_out(args.d, to, __uint_as_float(bits), out_dtype);
                        }
                    }
                    __syncwarp();
                }
            };

            if (!empty && rows <= 0) {                            // nothing of this quarter belongs to the group
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (kPair) ptx::mbar_arrive_cluster(tempty0 + 8 * slot);
                    else ptx::mbar_arrive(bar_tempty + 8 * slot);
                }
                continue;
            }
            uint32_t v[32];
            if (!empty) ptx::tmem_ld_32x32(t_addr, v);
#pragma unroll 1
            for (int c = 0; c < kChunks; ++c) {
                if (empty) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = 0u;
                } else {
                    ptx::tmem_ld_wait();
                    if (c == kChunks - 1) {                       // the accumulator's columns of this warp are in registers
                        ptx::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            if (kPair) ptx::mbar_arrive_cluster(tempty0 + 8 * slot);
                            else ptx::mbar_arrive(bar_tempty + 8 * slot);
                        }
                    }
                }
                scale(v, w.n0 + grp * (BN / 2) + c * 32);
                emit(v, c, [&]() { if (!empty && c + 1 < kChunks) ptx::tmem_ld_32x32(t_addr + (c + 1) * 32, v); });
            }
        }
        // the staging box must outlive the stores' reads of it; the writes themselves complete with the grid
        if (issuer) ptx::bulk_wait_group_read<0>();
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
