// Host side of the expert-layer entry points of include/b200fp8.h: argument checks, tensor maps, kernel choice, launch.
#include <cuda.h>
#include <cuda_runtime.h>
#include <atomic>
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>

#include "../../include/b200fp8.h"
#include "host_sm100.h"
#include "gemm_grouped_sm100.cuh"
#include "gemv_w4_sm100.cuh"
#include "quantize_rows_sm100.cuh"

namespace b200fp8 {
namespace {

constexpr int kDevices = 64;
constexpr int kMaxRows = 1 << 30;        // and columns: index arithmetic in 32 bits has room for a tile beyond them
constexpr int kMaxExperts = 1 << 16;

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
// elements from the first to behind the last of a matrix; in floating point, where no pitch overflows
double span(int rows, long long pitch, int columns) { return (rows - 1.0) * static_cast<double>(pitch) + columns; }
bool fp8(int d) { return d == B200FP8_E4M3 || d == B200FP8_E5M2; }

// dynamic shared memory above the default has to be asked for once per kernel and device
template <auto kKernel>
cudaError_t allow_smem(int bytes) {
    static std::atomic<bool> done[kDevices] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= kDevices) return cudaErrorInvalidDevice;
    if (done[dev].load(std::memory_order_relaxed)) return cudaSuccess;
    e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done[dev].store(true, std::memory_order_relaxed);
    return e;
}

template <class... Params, class... Args>
cudaError_t launch(void (*kernel)(Params...), bool pdl, dim3 grid, int threads, int smem, int cluster, cudaStream_t stream, Args&&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = static_cast<unsigned>(cluster);
        attr[n].val.clusterDim.y = 1;
        attr[n++].val.clusterDim.z = 1;
    }
    if (pdl) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // see griddep_wait in the kernels
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = static_cast<unsigned>(n);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<Args&&>(args)...);
    if (e == cudaSuccess) count_launch();
    return e;
}

// A tensor map over `count` matrices of rows x cols elements, row pitch ld, matrix pitch `stride` (elements); the box is
// one matrix deep.  A map is a pure function of these numbers, so each host thread keeps the last ones it encoded.
cudaError_t encode_3d(const HostDevice& dev, CUtensorMap* map, CUtensorMapDataType type, int elem, const void* base, uint64_t cols,
                      uint64_t rows, uint64_t count, uint64_t ld, uint64_t stride, uint32_t box_cols, uint32_t box_rows, CUtensorMapSwizzle swizzle) {
    struct Key {
        const void* base; uint64_t cols, rows, count, ld, stride; uint32_t box_cols, box_rows; int type, swizzle;
        bool operator==(const Key& o) const {
            return base == o.base && cols == o.cols && rows == o.rows && count == o.count && ld == o.ld && stride == o.stride &&
                   box_cols == o.box_cols && box_rows == o.box_rows && type == o.type && swizzle == o.swizzle;
        }
    };
    constexpr int kSlots = 64;
    struct Cache { Key key[kSlots]; CUtensorMap map[kSlots]; bool used[kSlots]; };
    static thread_local Cache cache = {};
    const Key key{base, cols, rows, count, ld, stride, box_cols, box_rows, static_cast<int>(type), static_cast<int>(swizzle)};
    const uint64_t h = ((reinterpret_cast<uintptr_t>(base) >> 8) + cols * 31 + rows * 131 + box_rows * 7 + box_cols) * 0x9E3779B97F4A7C15ull;
    const int slot = static_cast<int>(h >> 58);
    if (cache.used[slot] && cache.key[slot] == key) { *map = cache.map[slot]; return cudaSuccess; }
    const cuuint64_t dims[3] = {cols, rows, count};
    const cuuint64_t strides[2] = {ld * elem, stride * elem};
    const cuuint32_t box[3] = {box_cols, box_rows, 1};
    const cuuint32_t estr[3] = {1, 1, 1};
    if (dev.encode(map, type, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return cudaErrorInvalidValue;
    cache.key[slot] = key; cache.map[slot] = *map; cache.used[slot] = true;
    return cudaSuccess;
}

struct GroupedCall {
    int experts, rows, k, n;
    const int* ends;
    const void* a; int a_dtype; long long lda;
    const void* b; int b_dtype; long long ldb, stride_b;
    void* d; int d_dtype; long long ldd, stride_d;
    int max_ctas;
    Epilogue epi;
};

template <int MODE, int ROWS, int CTAS, int OB, bool BETA>
cudaError_t launch_grouped_form(const HostDevice& dev, const GroupedCall& c, cudaStream_t stream) {
    using L = GroupedSmem<ROWS, CTAS>;
    constexpr bool wgrad = MODE == kGroupedWgrad;
    cudaError_t e = allow_smem<gemm_fp8_grouped_kernel<MODE, ROWS, CTAS, OB, BETA>>(L::kDynamicBytes);
    if (e != cudaSuccess) return e;
    GroupedArgs args{};
    args.experts = c.experts;
    args.rows = c.rows;
    args.cols = MODE == kGroupedForward ? c.n : c.k;
    args.depth = MODE == kGroupedForward ? c.k : c.n;
    args.d_rows = c.n;                                            // wgrad
    args.ends = c.ends;
    args.row_tiles = (c.n + ROWS - 1) / ROWS;                     // wgrad
    args.col_tiles = (args.cols + 128 * CTAS - 1) / (128 * CTAS);
    args.group_rows = 16;
    // the operand of D's columns is the instruction's A, that of D's rows its B; bits 15 and 16: MN-major
    const void* w = c.b;
    const int w_dtype = c.b_dtype, r_dtype = c.a_dtype;
    args.idesc = make_idesc_f8(w_dtype, r_dtype, 128 * CTAS, 0) | (MODE != kGroupedForward ? 1u << 15 : 0u) | (wgrad ? 1u << 16 : 0u);
    args.d = c.d; args.ldd = c.ldd; args.stride_d = c.stride_d;
    args.w = static_cast<const uint8_t*>(w); args.ldw = c.ldb;
    args.r = static_cast<const uint8_t*>(c.a); args.ldr = c.lda;
    args.status = dev.status;
    args.debug = dev.debug;
    args.epi = c.epi;
    constexpr int kWide = OB == 2 ? 8 : 4;                        // columns per store
    args.wide_store = OB != 4 && args.cols % kWide == 0 && c.ldd % kWide == 0 && (!wgrad || c.stride_d % kWide == 0) && aligned(c.d, kWide * OB);

    GroupedMaps maps;
    const CUtensorMapDataType u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
    const CUtensorMapSwizzle s128 = CU_TENSOR_MAP_SWIZZLE_128B;
    const uint64_t rows = static_cast<uint64_t>(std::max(1, c.rows));
    auto ragged = [&](CUtensorMap* map, const void* base, uint64_t cols, long long ld, uint32_t box) {
        return encode_3d(dev, map, u8, 1, base, cols, rows, 1, ld, ld * rows, kBlockK, box, s128);
    };
    const uint64_t r_cols = MODE == kGroupedForward ? c.k : c.n;
    if (wgrad) {
        if ((e = ragged(&maps.w, w, c.k, c.ldb, 128)) != cudaSuccess) return e;
        if ((e = ragged(&maps.w32, w, c.k, c.ldb, 32)) != cudaSuccess) return e;
        if ((e = ragged(&maps.r[3], c.a, r_cols, c.lda, 128)) != cudaSuccess) return e;
        if ((e = ragged(&maps.r32, c.a, r_cols, c.lda, 32)) != cudaSuccess) return e;
        maps.r[0] = maps.r[1] = maps.r[2] = maps.r[3];            // not used
    } else {
        if ((e = encode_3d(dev, &maps.w, u8, 1, w, c.k, c.n, c.experts, c.ldb, c.stride_b, kBlockK, 128, s128)) != cudaSuccess) return e;
        for (int i = 0; i < 4; ++i)
            if ((e = ragged(&maps.r[i], c.a, r_cols, c.lda, 16u << i)) != cudaSuccess) return e;
        maps.w32 = maps.w;                                        // not used
        maps.r32 = maps.r[3];
    }
    // no more CTAs than there can be tiles: the sizes of the groups are known on the device only
    const long long groups = wgrad ? c.experts : std::min(c.experts, c.rows);
    const long long tiles = (wgrad ? groups * args.row_tiles : groups + c.rows / ROWS) * args.col_tiles;
    if (tiles > (1LL << 30)) return cudaErrorInvalidValue;
    int units = dev.sm_count / CTAS;
    if (c.max_ctas > 0) units = std::max(1, std::min(units, c.max_ctas / CTAS));
    units = static_cast<int>(std::min<long long>(units, tiles));
    return launch(gemm_fp8_grouped_kernel<MODE, ROWS, CTAS, OB, BETA>, dev.pdl, dim3(static_cast<unsigned>(units * CTAS), 1, 1), kGemmThreads, L::kDynamicBytes,
                  CTAS, stream, maps, args);
}

template <int MODE, int ROWS, int CTAS, int OB>
cudaError_t launch_grouped(const HostDevice& dev, const GroupedCall& c, cudaStream_t stream) {
    return c.epi.beta != 0.0f ? launch_grouped_form<MODE, ROWS, CTAS, OB, true>(dev, c, stream) : launch_grouped_form<MODE, ROWS, CTAS, OB, false>(dev, c, stream);
}

// The automatic choice.  The sizes of the groups are known on the device only, so it goes by their average.
int choose_grouped(int sm_count, int mode, const GroupedCall& c) {
    const double experts = std::max(1, std::min(c.experts, c.rows)), average = c.rows / experts;
    if (mode == kGroupedWgrad) {
        // Tiles are of equal size and their contraction is the group.  With few rows per group the product is a store of D and
        // twice as many CTAs store it faster; from about 600 on the pair's lower operand traffic decides (8 experts of
        // 4096 x 4096: 74.9 us with one CTA, 93.6 with pairs at 48 rows; 89 / 103 at 400; 118.8 / 115.8 at 700).
        if (c.n <= 128) return B200FP8_KERNEL_CTA1_N128;
        return average >= 600 ? B200FP8_KERNEL_PAIR_N256 : B200FP8_KERNEL_CTA1_N256;
    }
    // Rounds of tiles that each shape needs (whole ones while they are few) times what a round costs: a round of 256 x 256 pair
    // tiles takes about 1.3 times one of 128 x 128 tiles (one group of 256 rows, 8192 x 8192: 25.4 against 20.4 us in one round
    // each; 400 rows: 27.6 in one round against 32.3 in two), one of 64-row tiles, with more of the weights in flight, 0.88
    // (100 rows: 17.0 against 19.2 us).  A short contraction leaves the epilogue to decide, and 256-row tiles of one CTA keep it
    // busier than pairs do (8 groups of 1000 rows, 4096 columns: 22.4 / 25.9 / 37.6 / 63.5 us against 28.1 / 31.6 / 37.9 / 56.4
    // for depths of 128 / 512 / 1024 / 2048).
    const double cols = mode == kGroupedForward ? c.n : c.k;
    auto cost = [&](int tile_rows, int tile_cols, int units, double per_round) {
        const double per_group = experts == 1 ? std::ceil(average / tile_rows) : 2 * average <= tile_rows ? 1.0 : average / tile_rows + 0.5;
        const double rounds = experts * per_group * std::ceil(cols / tile_cols) / units;
        return per_round * (rounds < 4 ? std::ceil(rounds) : rounds);
    };
    const double low = cost(64, 128, sm_count, 0.88), mid = cost(128, 128, sm_count, 1.0), pair = cost(256, 256, sm_count / 2, 1.3);
    const int depth = mode == kGroupedForward ? c.k : c.n;
    if (pair <= mid && pair <= low) return depth < 1024 ? B200FP8_KERNEL_CTA1_N256 : B200FP8_KERNEL_PAIR_N256;
    return mid <= low ? B200FP8_KERNEL_CTA1_N128 : B200FP8_KERNEL_CTA1_N64;
}

template <int MODE, int OB>
cudaError_t dispatch_grouped_to(const HostDevice& dev, const GroupedCall& c, int kernel, cudaStream_t stream) {
    if (kernel == B200FP8_KERNEL_AUTO) kernel = choose_grouped(dev.sm_count, MODE, c);
    switch (kernel) {
        case B200FP8_KERNEL_PAIR_N256: return launch_grouped<MODE, 256, 2, OB>(dev, c, stream);
        case B200FP8_KERNEL_CTA1_N256: return launch_grouped<MODE, 256, 1, OB>(dev, c, stream);
        case B200FP8_KERNEL_CTA1_N128: return launch_grouped<MODE, 128, 1, OB>(dev, c, stream);
        case B200FP8_KERNEL_CTA1_N64:
            if constexpr (MODE != kGroupedWgrad) return launch_grouped<MODE, 64, 1, OB>(dev, c, stream);
            return cudaErrorInvalidValue;
        default: return cudaErrorInvalidValue;
    }
}

template <int MODE>
cudaError_t dispatch_grouped(const HostDevice& dev, const GroupedCall& c, int kernel, cudaStream_t stream) {
    switch (out_dtype_bytes(c.d_dtype)) {
        case 4: return dispatch_grouped_to<MODE, 4>(dev, c, kernel, stream);
        case 2: return dispatch_grouped_to<MODE, 2>(dev, c, kernel, stream);
        default: return dispatch_grouped_to<MODE, 1>(dev, c, kernel, stream);
    }
}

// What the three products check alike.  `a_cols` / `d_cols`: extents along the contiguous index of A and D.
cudaError_t grouped(int mode, int experts, int rows, int k, int n, const int* ends, const void* a, int a_dtype, long long lda, const void* b,
                    int b_dtype, long long ldb, long long stride_b, void* d, int d_dtype, long long ldd, long long stride_d,
                    const b200fp8_epilogue* ep, const b200fp8_options* options, cudaStream_t stream) {
    if (options && options->struct_bytes != static_cast<int>(sizeof(b200fp8_options))) return cudaErrorInvalidValue;
    if (options && (options->depth != 0 || options->split_k != 0 || options->max_ctas < 0)) return cudaErrorInvalidValue;
    if (ep && ep->struct_bytes != static_cast<int>(sizeof(b200fp8_epilogue)) && ep->struct_bytes != B200FP8_EPILOGUE_V1_BYTES) return cudaErrorInvalidValue;
    const bool extended = ep && ep->struct_bytes == static_cast<int>(sizeof(b200fp8_epilogue));
    if (extended && (ep->activation < B200FP8_ACT_NONE || ep->activation > B200FP8_ACT_GELU_TANH)) return cudaErrorInvalidValue;
    if (experts < 0 || rows < 0 || k <= 0 || n <= 0 || experts > kMaxExperts || rows > kMaxRows || k > kMaxRows || n > kMaxRows) return cudaErrorInvalidValue;
    if (!fp8(a_dtype) || !fp8(b_dtype)) return cudaErrorInvalidValue;
    if (d_dtype < B200FP8_OUT_F32 || d_dtype > B200FP8_OUT_E5M2) return cudaErrorInvalidValue;
    const bool wgrad = mode == kGroupedWgrad;
    if (ep && ep->bias && (ep->bias_dtype < B200FP8_OUT_F32 || ep->bias_dtype > B200FP8_OUT_F16)) return cudaErrorInvalidValue;
    if (ep && ep->bias && !aligned(ep->bias, out_dtype_bytes(ep->bias_dtype))) return cudaErrorInvalidValue;
    if (ep && (!aligned(ep->amax_d, 4) || !aligned(ep->a_scale, 4) || !aligned(ep->b_scale, 4) || !aligned(ep->d_scale, 4))) return cudaErrorInvalidValue;
    if (extended && (!aligned(ep->a_row_scale, 4) || !aligned(ep->b_row_scale, 4))) return cudaErrorInvalidValue;
    // a bias, an activation or a scale of one row has no place in a sum over the rows
    if (wgrad && ep && (ep->bias || (extended && (ep->activation || ep->a_row_scale || ep->b_row_scale)))) return cudaErrorInvalidValue;
    const long long a_cols = mode == kGroupedForward ? k : n, d_cols = mode == kGroupedForward ? n : k;
    // the contiguous extents that TMA and the tensor core walk: whole 16-byte pieces
    if (k % 16 || (mode != kGroupedForward && n % 16) || lda % 16 || ldb % 16) return cudaErrorInvalidValue;
    if (lda < a_cols || ldb < k || ldd < d_cols) return cudaErrorInvalidValue;
    constexpr long long kMostStride = 1LL << 39;                  // a tensor map's strides are below 2^40 bytes
    if (lda > kMostStride || ldb > kMostStride || ldd > kMostStride / 4) return cudaErrorInvalidValue;
    if (experts > 1) {                                            // one expert's matrix has no next one
        if (!wgrad && (stride_b % 16 || stride_b < span(n, ldb, k) || stride_b > kMostStride)) return cudaErrorInvalidValue;
        if (wgrad && (stride_d < span(n, ldd, k) || stride_d > kMostStride / 4)) return cudaErrorInvalidValue;
    }
    const int out_bytes = out_dtype_bytes(d_dtype);
    const bool nothing = experts == 0 || (rows == 0 && !wgrad);
    if (!nothing) {
        if (!ends || !aligned(ends, 4) || !d || !aligned(d, out_bytes)) return cudaErrorInvalidValue;
        if ((rows > 0 && !a) || ((!wgrad || rows > 0) && !b) || !aligned(a, 16) || !aligned(b, 16)) return cudaErrorInvalidValue;
        // a matrix of all rows has to be addressable as one tensor map
        const double height = rows;
        if (height * static_cast<double>(lda) > 5e11 || height * static_cast<double>(wgrad ? ldb : ldd) * out_bytes > 1e12) return cudaErrorInvalidValue;
    }
    const int kernel = options ? options->kernel : B200FP8_KERNEL_AUTO;
    if (kernel != B200FP8_KERNEL_AUTO && kernel != B200FP8_KERNEL_PAIR_N256 && kernel != B200FP8_KERNEL_CTA1_N256 &&
        kernel != B200FP8_KERNEL_CTA1_N128 && (wgrad || kernel != B200FP8_KERNEL_CTA1_N64))
        return cudaErrorInvalidValue;
    HostDevice dev;
    cudaError_t e = host_device(&dev);
    if (e != cudaSuccess) return e;
    if (ep && ep->amax_d && (e = cudaMemsetAsync(ep->amax_d, 0, sizeof(float), stream)) != cudaSuccess) return e;
    if (nothing) return cudaSuccess;

    GroupedCall c{};
    c.experts = experts; c.rows = rows; c.k = k; c.n = n; c.ends = ends;
    c.a = a; c.a_dtype = a_dtype; c.lda = lda;
    c.b = b; c.b_dtype = b_dtype; c.ldb = ldb; c.stride_b = experts > 1 ? stride_b : static_cast<long long>(n) * ldb;
    c.d = d; c.d_dtype = d_dtype; c.ldd = ldd; c.stride_d = experts > 1 ? stride_d : static_cast<long long>(n) * ldd;
    if (rows == 0) {
        // wgrad without any row: every group is empty and nothing of A or B is read; the maps need some valid base
        c.a = c.b = reinterpret_cast<const void*>(reinterpret_cast<uintptr_t>(d) & ~static_cast<uintptr_t>(15));
    }
    c.max_ctas = options ? options->max_ctas : 0;
    c.epi.active = 1;
    c.epi.out_dtype = d_dtype;
    c.epi.alpha = 1.0f;
    if (ep) {
        c.epi.alpha = ep->alpha; c.epi.beta = ep->beta;
        c.epi.a_scale = ep->a_scale; c.epi.b_scale = ep->b_scale; c.epi.d_scale = ep->d_scale;
        c.epi.amax = ep->amax_d;
        c.epi.bias = ep->bias; c.epi.bias_dtype = ep->bias_dtype;
        if (extended) { c.epi.activation = ep->activation; c.epi.a_row_scale = ep->a_row_scale; c.epi.b_row_scale = ep->b_row_scale; }
    }
    switch (mode) {
        case kGroupedForward: return dispatch_grouped<kGroupedForward>(dev, c, kernel, stream);
        case kGroupedDgrad: return dispatch_grouped<kGroupedDgrad>(dev, c, kernel, stream);
        default: return dispatch_grouped<kGroupedWgrad>(dev, c, kernel, stream);
    }
}

template <bool BF16, int Q, int THREADS, int PIECES>
cudaError_t launch_quantize_form(const HostDevice& dev, const QuantizeArgs& args, cudaStream_t stream) {
    constexpr unsigned kRows = THREADS == 32 ? 4 : 1;             // of a block
    return launch(quantize_rows_kernel<BF16, Q, THREADS, PIECES>, dev.pdl, dim3((static_cast<unsigned>(args.rows) + kRows - 1) / kRows, 1, 1),
                  kRows * THREADS, 0, 1, stream, args);
}

template <bool BF16, int Q>
cudaError_t launch_quantize(const HostDevice& dev, const QuantizeArgs& args, cudaStream_t stream) {
    const bool whole = args.k % 8 == 0 && args.ldx % 8 == 0 && args.ldq % 8 == 0 && aligned(args.x, 16) && aligned(args.q, 8);
    const int pieces = (args.k + 7) / 8;
    if (!whole || pieces > kQuantizeMostPieces)
        return launch(quantize_rows_any_kernel<BF16>, dev.pdl, dim3(static_cast<unsigned>(args.rows), 1, 1), 256, 0, 1, stream, args);
    // Many rows: few blocks with much to do each, since the GPU starts about one block per nanosecond and every thread that has a
    // piece too few still takes its instructions (67 million elements, a row of 1040 by 128 threads 67.8 us, by one warp 31.3; 2080
    // 35.5 / 26.8; 10240 by 512 threads 32.5, by 256 with six pieces 27.0).  Few rows: more threads finish one earlier (1040 elements
    // 1.2 against 1.4 us).
    if (pieces <= 128) return launch_quantize_form<BF16, Q, 32, 4>(dev, args, stream);
    if (args.rows > 8 * dev.sm_count && pieces <= 256) return launch_quantize_form<BF16, Q, 32, 8>(dev, args, stream);
    if (args.rows > 8 * dev.sm_count && pieces <= 384) return launch_quantize_form<BF16, Q, 32, 12>(dev, args, stream);
    if (pieces <= 512) return launch_quantize_form<BF16, Q, 128, 4>(dev, args, stream);
    if (pieces <= 768) return launch_quantize_form<BF16, Q, 128, 6>(dev, args, stream);
    if (pieces <= 1024) return launch_quantize_form<BF16, Q, 256, 4>(dev, args, stream);
    if (pieces <= 1536) return launch_quantize_form<BF16, Q, 256, 6>(dev, args, stream);
    return launch_quantize_form<BF16, Q, 512, 4>(dev, args, stream);
}

template <bool BF16, int G, int NT, int RT, bool WIDE, bool INT>
cudaError_t launch_w4(const HostDevice& dev, W4Args args, cudaStream_t stream) {
    using L = W4Smem<NT, RT, INT>;
    const int list_bytes = args.expert ? 4 * args.m : 0;
    const int bytes = L::kFixedBytes + list_bytes;
    cudaError_t e = allow_smem<gemv_w4_kernel<BF16, G, NT, RT, WIDE, INT>>(L::kFixedBytes + 4 * kW4MostRows);
    if (e != cudaSuccess) return e;
    const int slots = args.expert ? std::min(args.experts, args.m) : 1;
    const int tiles = (args.n + L::kTileRows - 1) / L::kTileRows;
    args.k_blocks = (args.k + kW4BoxK - 1) / kW4BoxK;
    args.status = dev.status;
    args.debug = dev.debug;
    args.k_unit = G == 128 ? 2 : 1;
    const int units = (args.k_blocks + args.k_unit - 1) / args.k_unit;
    const int scale_bytes = out_dtype_bytes(args.scale_dtype);
    args.vector_scales = args.scale_ld % 4 == 0 && args.scale_stride % 4 == 0 && aligned(args.scales, 4 * scale_bytes);
    args.vector_zeros = args.zero_ld % 4 == 0 && args.zero_stride % 4 == 0 && aligned(args.zeros, 4);
    // K is parted until three CTAs share two SMs: every part costs its CTA a start and a meeting with the others (about 5 us in
    // all), so more of them lose (8192 x 8192, one vector: 25.3 / 16.5 / 15.0 / 21.9 us in 1 / 2 / 4 / 8 parts; 28672 x 8192, eight
    // vectors: 47 / 53 / 55 / 74)
    int splits = 1;
    while (splits < kW4MostSplits && 2 * splits <= units && static_cast<long long>(slots) * tiles * splits < (dev.sm_count * 3) / 2) splits *= 2;
    args.splits = splits;
    CUtensorMap map;
    const uint64_t experts = args.expert ? args.experts : 1;
    if ((e = encode_3d(dev, &map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, args.codes, args.k / 2, args.n, experts, args.code_ld,
                       experts > 1 ? args.code_stride : args.code_ld * static_cast<long long>(args.n), kW4BoxBytes, 16 * RT,
                       CU_TENSOR_MAP_SWIZZLE_128B)) != cudaSuccess)
        return e;
    const dim3 grid(static_cast<unsigned>(splits), static_cast<unsigned>(tiles), static_cast<unsigned>(slots));
    return launch(gemv_w4_kernel<BF16, G, NT, RT, WIDE, INT>, dev.pdl, grid, kW4Threads, bytes, splits, stream, map, args);
}

template <bool BF16, int G, bool WIDE>
cudaError_t launch_w4_form(const HostDevice& dev, const W4Args& args, cudaStream_t stream) {
    // One or two vectors (a token's experts are usually different ones, so two tokens give an expert two rows) of weights beyond
    // 2^25 take the integer form.  Groups of 128: 8192 x 8192 12.8 us against 14.2, 28672 x 8192 32.2 against 39.0, but 4096 x 4096
    // 9.0 against 8.3 and, at the border, 16384 x 2048 10.5 against 10.7; groups of 64: 28672 x 8192 37.6 against 41.8, 4096 x 4096
    // 9.6 against 8.4.  With groups of 32 its work per group outweighs the rest (8192 x 8192 18.2 against 17.9, 4096 x 4096 9.5
    // against 8.5).  Filling two tiles of columns with the digits of more vectors lost to the other form everywhere.
    const int vectors = args.expert ? args.m / args.rows_per_x : args.m;
    const long long matrices = args.expert ? std::min(args.experts, args.m) : 1;
    if constexpr (G > 32)
        if (vectors <= 2 && matrices * args.n * args.k > (1LL << 25)) return launch_w4<BF16, G, 1, 1, WIDE, true>(dev, args, stream);
    // The form in x's type takes eight vectors to a pass, or sixteen.  By expert the number of rows that share an expert is known on
    // the device only: their average.
    const long long shared = args.expert ? args.experts : 1;
    if (args.m <= 8 * shared) {
        // With more CTAs than fit at once, half as many with 32 rows per warp stage x half as often and have twice the
        // independent work per warp.  16 tokens, 8 of 64 experts each, groups of 128: 2048 x 4096 52.4 -> 44.8 us,
        // 4096 x 1024 63.2 -> 48.7, 1024 x 1024 22.1 -> 16.9 (1.7 CTAs of 256 rows per SM); 4 of 32 experts, 1024 x 1024
        // (0.9) 11.5 -> 13.3.
        const long long blocks = static_cast<long long>(args.expert ? std::min(args.experts, args.m) : 1) * ((args.n + 255) / 256);
        if (blocks > dev.sm_count) return launch_w4<BF16, G, 1, 2, WIDE, false>(dev, args, stream);
        return launch_w4<BF16, G, 1, 1, WIDE, false>(dev, args, stream);
    }
    return launch_w4<BF16, G, 2, 1, WIDE, false>(dev, args, stream);
}

template <bool BF16, int G>
cudaError_t launch_w4_group(const HostDevice& dev, const W4Args& args, cudaStream_t stream) {
    if (args.scale_dtype == B200FP8_OUT_F32) return launch_w4_form<BF16, G, true>(dev, args, stream);
    return launch_w4_form<BF16, G, false>(dev, args, stream);
}

template <bool BF16>
cudaError_t launch_w4_type(const HostDevice& dev, const W4Args& args, cudaStream_t stream) {
    switch (args.group) {
        case 32: return launch_w4_group<BF16, 32>(dev, args, stream);
        case 64: return launch_w4_group<BF16, 64>(dev, args, stream);
        default: return launch_w4_group<BF16, 128>(dev, args, stream);
    }
}

cudaError_t w4(const W4Args& args, int x_dtype, cudaStream_t stream) {
    if (args.n < 0 || args.k <= 0 || args.m < 0 || args.n > 65535 * 128 || args.k > kMaxRows || args.m > kMaxRows || args.code_ld > (1LL << 39))
        return cudaErrorInvalidValue;
    if (x_dtype != B200FP8_OUT_BF16 && x_dtype != B200FP8_OUT_F16) return cudaErrorInvalidValue;
    if (args.y_dtype != x_dtype && args.y_dtype != B200FP8_OUT_F32) return cudaErrorInvalidValue;
    if (args.scale_dtype < B200FP8_OUT_F32 || args.scale_dtype > B200FP8_OUT_F16) return cudaErrorInvalidValue;
    if ((args.group != 32 && args.group != 64 && args.group != 128) || args.k % args.group) return cudaErrorInvalidValue;
    if (args.code_ld < args.k / 2 || args.code_ld % 16 || args.scale_ld < args.k / args.group || args.ldx < args.k || args.ldx % 8 || args.ldy < args.n)
        return cudaErrorInvalidValue;
    if (args.zeros && args.zero_ld < args.k / args.group) return cudaErrorInvalidValue;
    if (args.m == 0 || args.n == 0) return cudaSuccess;
    const int y_bytes = out_dtype_bytes(args.y_dtype);
    if (!args.y || !aligned(args.y, y_bytes)) return cudaErrorInvalidValue;
    if (args.k > 0 && (!args.codes || !args.scales || !args.x || !aligned(args.codes, 16) || !aligned(args.x, 16) ||
                       !aligned(args.scales, out_dtype_bytes(args.scale_dtype))))
        return cudaErrorInvalidValue;
    HostDevice dev;
    const cudaError_t e = host_device(&dev);
    if (e != cudaSuccess) return e;
    if (x_dtype == B200FP8_OUT_BF16) return launch_w4_type<true>(dev, args, stream);
    return launch_w4_type<false>(dev, args, stream);
}

}  // namespace
}  // namespace b200fp8

using namespace b200fp8;

extern "C" {

int b200fp8_gemm_grouped(int experts, int rows, int k, int n, const int* ends, const void* a, int a_dtype, long long lda, const void* b,
                         int b_dtype, long long ldb, long long stride_b, void* d, int d_dtype, long long ldd, const b200fp8_epilogue* epilogue,
                         const b200fp8_options* options, void* stream) {
    return grouped(kGroupedForward, experts, rows, k, n, ends, a, a_dtype, lda, b, b_dtype, ldb, stride_b, d, d_dtype, ldd, 0, epilogue, options,
                   static_cast<cudaStream_t>(stream));
}

int b200fp8_gemm_grouped_dgrad(int experts, int rows, int k, int n, const int* ends, const void* a, int a_dtype, long long lda, const void* b,
                               int b_dtype, long long ldb, long long stride_b, void* d, int d_dtype, long long ldd,
                               const b200fp8_epilogue* epilogue, const b200fp8_options* options, void* stream) {
    return grouped(kGroupedDgrad, experts, rows, k, n, ends, a, a_dtype, lda, b, b_dtype, ldb, stride_b, d, d_dtype, ldd, 0, epilogue, options,
                   static_cast<cudaStream_t>(stream));
}

int b200fp8_gemm_grouped_wgrad(int experts, int rows, int k, int n, const int* ends, const void* a, int a_dtype, long long lda, const void* b,
                               int b_dtype, long long ldb, void* d, int d_dtype, long long ldd, long long stride_d,
                               const b200fp8_epilogue* epilogue, const b200fp8_options* options, void* stream) {
    return grouped(kGroupedWgrad, experts, rows, k, n, ends, a, a_dtype, lda, b, b_dtype, ldb, 0, d, d_dtype, ldd, stride_d, epilogue, options,
                   static_cast<cudaStream_t>(stream));
}

int b200fp8_quantize_rows(int source_rows, int rows, int k, const void* x, int x_dtype, long long ldx, const int* index, void* q, int q_dtype,
                          long long ldq, float* scale, void* stream) {
    if (source_rows < 0 || rows < 0 || k < 0 || k > kMaxRows) return cudaErrorInvalidValue;
    if (!fp8(q_dtype) || (x_dtype != B200FP8_OUT_BF16 && x_dtype != B200FP8_OUT_F16)) return cudaErrorInvalidValue;
    if (ldx < k || ldq < k || (!index && rows > source_rows)) return cudaErrorInvalidValue;
    if (rows == 0) return cudaSuccess;
    if (!scale || !aligned(scale, 4) || !aligned(index, 4) || !aligned(x, 2)) return cudaErrorInvalidValue;
    if (k > 0 && (!q || (!x && source_rows > 0))) return cudaErrorInvalidValue;
    HostDevice dev;
    const cudaError_t e = host_device(&dev);
    if (e != cudaSuccess) return e;
    QuantizeArgs args{static_cast<const uint16_t*>(x), ldx, source_rows, index, rows, k, static_cast<uint8_t*>(q), ldq, scale, q_dtype};
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (x_dtype == B200FP8_OUT_BF16) return q_dtype == B200FP8_E4M3 ? launch_quantize<true, 0>(dev, args, st) : launch_quantize<true, 1>(dev, args, st);
    return q_dtype == B200FP8_E4M3 ? launch_quantize<false, 0>(dev, args, st) : launch_quantize<false, 1>(dev, args, st);
}

int b200fp8_gemv_w4(int m, int k, int n, int group, const void* codes, long long code_ld, const void* scales, int scale_dtype,
                    long long scale_ld, const unsigned char* zeros, long long zero_ld, const void* x, int x_dtype, long long ldx, void* y,
                    int y_dtype, long long ldy, void* stream) {
    W4Args args{};
    args.codes = static_cast<const uint8_t*>(codes); args.code_ld = code_ld;
    args.scales = scales; args.scale_dtype = scale_dtype; args.scale_ld = scale_ld;
    args.zeros = zeros; args.zero_ld = zero_ld;
    args.x = static_cast<const uint16_t*>(x); args.ldx = ldx;
    args.y = y; args.y_dtype = y_dtype; args.ldy = ldy;
    args.m = m; args.n = n; args.k = k; args.group = group;
    return w4(args, x_dtype, static_cast<cudaStream_t>(stream));
}

int b200fp8_gemv_w4_experts(int tokens, int rows, int experts, int k, int n, int group, const void* codes, long long code_ld,
                            long long code_stride, const void* scales, int scale_dtype, long long scale_ld, long long scale_stride,
                            const unsigned char* zeros, long long zero_ld, long long zero_stride, const int* expert, const void* x,
                            int x_dtype, long long ldx, void* y, int y_dtype, long long ldy, void* stream) {
    if (tokens < 0 || rows < 0 || experts < 0 || rows > kW4MostRows || experts > kW4MostExperts) return cudaErrorInvalidValue;
    if (rows > 0 && (tokens == 0 || rows % tokens || !expert || !aligned(expert, 4))) return cudaErrorInvalidValue;
    if (experts > 1 && k > 0 && n > 0 &&
        (code_stride % 16 || code_stride > (1LL << 39) || code_stride < span(n, code_ld, k / 2) ||
         scale_stride < span(n, scale_ld, k / std::max(group, 1)) || (zeros && zero_stride < span(n, zero_ld, k / std::max(group, 1)))))
        return cudaErrorInvalidValue;
    if (experts == 1) code_stride = scale_stride = zero_stride = 0;             // not read
    W4Args args{};
    args.codes = static_cast<const uint8_t*>(codes); args.code_ld = code_ld; args.code_stride = code_stride;
    args.scales = scales; args.scale_dtype = scale_dtype; args.scale_ld = scale_ld; args.scale_stride = scale_stride;
    args.zeros = zeros; args.zero_ld = zero_ld; args.zero_stride = zero_stride;
    args.x = static_cast<const uint16_t*>(x); args.ldx = ldx;
    args.y = y; args.y_dtype = y_dtype; args.ldy = ldy;
    args.m = experts == 0 ? 0 : rows; args.n = n; args.k = k; args.group = group;
    args.expert = expert; args.experts = experts;
    args.rows_per_x = tokens > 0 ? std::max(1, rows / tokens) : 1;
    return w4(args, x_dtype, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
