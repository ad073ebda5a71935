// The experts of a layer and the dense products beside them: argument checks, tensor maps and launches.
//
// All of them are product_tiles.cuh's kernel.
#include <algorithm>
#include <atomic>
#include <cstring>

#include "product_device.cuh"
#include "product_tiles.cuh"

namespace {

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                CUtensorMapFloatOOBfill);

// The driver's encoder of tensor maps, looked up through the runtime, so that the library needs no driver to be loaded.
EncodeTiled encoder() {
    static std::atomic<void*> found{nullptr};
    void* fn = found.load(std::memory_order_acquire);
    if (fn == nullptr) {
        cudaDriverEntryPointQueryResult how;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &how) != cudaSuccess ||
            how != cudaDriverEntryPointSuccess)
            return nullptr;
        found.store(fn, std::memory_order_release);
    }
    return reinterpret_cast<EncodeTiled>(fn);
}

CUtensorMapDataType map_type(int dtype) {
    return dtype == A2A_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

// Rows [rows][inner], `stride` elements apart, in boxes of `box` rows by 64.
int rows_map(CUtensorMap* map, int dtype, const void* p, long long rows, int inner, long long stride, int box) {
    const EncodeTiled encode = encoder();
    if (encode == nullptr) return -(int)cudaErrorNotSupported;
    const cuuint64_t sizes[2] = {(cuuint64_t)inner, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride * 2};
    const cuuint32_t boxes[2] = {kTileInner, (cuuint32_t)box}, ones[2] = {1, 1};
    return encode(map, map_type(dtype), 2, const_cast<void*>(p), sizes, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? A2A_OK
               : A2A_ERR_CONFIG;
}

// Weights [groups][features], or [groups][gate, up][features], rows of `inner` values `stride` apart, in boxes of `box` features by 64;
// with gate and up a box steps from one to the other first.
int weights_map(CUtensorMap* map, int dtype, const void* p, int groups, int features, bool paired, int inner, long long stride, int box) {
    const EncodeTiled encode = encoder();
    if (encode == nullptr) return -(int)cudaErrorNotSupported;
    const cuuint64_t row = (cuuint64_t)stride * 2, halves = paired ? 2 : 1;
    const cuuint64_t sizes[4] = {(cuuint64_t)inner, halves, (cuuint64_t)features, (cuuint64_t)groups};
    const cuuint64_t strides[3] = {paired ? row * features : row, row, row * features * halves};
    const cuuint32_t boxes[4] = {kTileInner, (cuuint32_t)halves, (cuuint32_t)box, 1}, ones[4] = {1, 1, 1, 1};
    return encode(map, map_type(dtype), 4, const_cast<void*>(p), sizes, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? A2A_OK
               : A2A_ERR_CONFIG;
}

constexpr int kDevices = 64;

// A word a device, on a page of mapped host memory that the process's first call asks for, and keeps: kernels record there that a wait ran out, and the
// host looks without a CUDA call. A first call may be a captured one, in which nothing is allocated unless the thread says that it may.
int32_t* error_word(int device) {
    static std::atomic<int32_t*> known{nullptr};
    if (device < 0 || device >= kDevices) return nullptr;
    int32_t* words = known.load(std::memory_order_acquire);
    if (words == nullptr) {
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) return nullptr;
        void* page = nullptr;
        int32_t* fresh = nullptr;
        if (cudaHostAlloc(&page, kDevices * sizeof(int32_t), cudaHostAllocPortable | cudaHostAllocMapped) == cudaSuccess) {
            fresh = static_cast<int32_t*>(page);
            memset(fresh, 0, kDevices * sizeof(int32_t));
            if (known.compare_exchange_strong(words, fresh, std::memory_order_acq_rel)) words = fresh;
            else cudaFreeHost(page);  // another thread was first
        } else {
            cudaGetLastError();
        }
        cudaThreadExchangeStreamCaptureMode(&mode);
    }
    return words == nullptr ? nullptr : words + device;
}

// What a call needs of the current device: its SMs, and its word for errors, which is 0 or the call's answer.
struct Ready {
    int sms;
    int32_t* error;
};
int get_ready(Ready* r) {
    static std::atomic<int> known[kDevices];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return -(int)e;
    if ((r->error = error_word(dev)) == nullptr) return -(int)cudaErrorMemoryAllocation;
    r->sms = known[dev].load(std::memory_order_relaxed);
    if (r->sms == 0) {
        if ((e = cudaDeviceGetAttribute(&r->sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return -(int)e;
        known[dev].store(r->sms, std::memory_order_relaxed);
    }
    return *reinterpret_cast<volatile int32_t*>(r->error);
}

// Lets the kernel have its shared memory on the current device.
template <TilesOp kOp, typename T, Together kTogether>
int opt_in() {
    static std::atomic<unsigned long long> opted{0};  // a bit a device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return -(int)e;
    if (dev < 64 && (opted.load(std::memory_order_acquire) >> dev & 1)) return A2A_OK;
    e = cudaFuncSetAttribute((const void*)&product_tiles_kernel<kOp, T, kTogether>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kTilesSharedBytes);
    if (e != cudaSuccess) return -(int)e;
    if (dev < 64) opted.fetch_or(1ull << dev, std::memory_order_release);
    return A2A_OK;
}

// How many clusters of `size` blocks run at once: they do not come to lie on every SM.
template <TilesOp kOp, typename T, Together kTogether>
int most_clusters(int size) {
    static std::atomic<int> known[kMaxSplit + 1];  // one more than the number; of the first device that asked, as all are alike
    int n = known[size].load(std::memory_order_relaxed);
    if (n == 0) {
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = size;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cudaLaunchConfig_t config{};
        config.gridDim = dim3(size);
        config.blockDim = dim3(kTilesThreads);
        config.dynamicSmemBytes = kTilesSharedBytes;
        config.attrs = &attr;
        config.numAttrs = 1;
        if (opt_in<kOp, T, kTogether>() != A2A_OK ||
            cudaOccupancyMaxActiveClusters(&n, reinterpret_cast<const void*>(&product_tiles_kernel<kOp, T, kTogether>), &config) != cudaSuccess) {
            cudaGetLastError();
            return 0;
        }
        known[size].store(++n, std::memory_order_relaxed);
    }
    return n - 1;
}

// A launch that may get ready while the one before it in the stream ends (its kernel waits for that one itself), in clusters of `cluster` blocks.
int launch(const void* fn, dim3 grid, int threads, size_t shared, int cluster, void* params, cudaStream_t st) {
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = shared;
    config.stream = st;
    config.attrs = attr;
    config.numAttrs = cluster > 1 ? 2 : 1;
    void* args[] = {params};
    const cudaError_t e = cudaLaunchKernelExC(&config, fn, args);
    return e == cudaSuccess ? A2A_OK : -(int)e;
}

template <TilesOp kOp, typename T, Together kTogether = kAlone>
int launch_tiles(const TilesParams& p, int grid, int cluster, cudaStream_t st) {
    const int rc = opt_in<kOp, T, kTogether>();
    if (rc != A2A_OK) return rc;
    return launch(reinterpret_cast<const void*>(&product_tiles_kernel<kOp, T, kTogether>), grid, kTilesThreads, kTilesSharedBytes, cluster, const_cast<TilesParams*>(&p), st);
}

// How a dense product is cut: features and columns of a tile, blocks that share a tile's inner length, or pairs of blocks.
struct DensePlan {
    int height, columns, split;
    bool pair;
};
// What the fullest SM needs least time for, of tiles of up to 256 columns and of heights that fill the SMs once or twice; a cluster's
// addition takes 1.5 us and 10 ns a column, the epilogue of the last tile 13 ns a column, and tiles that read the same rows at the same
// time 1.3 ns each for every block of 64 (fitted; blocks that begin at different places of the sum take no less). (With 256 columns wherever there are as many: 1024 rows of
// 2048 to 2048 27.6 us instead of 14.9, 200 of 4096 to 7168 30.8 instead of 22.7.)
template <TilesOp kOp, typename T>
DensePlan dense_plan(const a2a_linear_args& a, bool paired, int sms) {
    const int most = std::min(paired ? kTileRows / 2 : kTileRows, a.outputs), blocks = parts_of(a.inputs, kTileInner), least_down = parts_of(a.outputs, most);
    constexpr int widest = kOp == kDense32 ? kMaxColumns32 : kMaxColumns;
    DensePlan best{most, std::min(widest, round16(a.tokens)), 1, false};
    float least = 1e30f;
    static constexpr int kWidths[] = {256, 192, 160, 128, 96, 64, 48, 32, 16};
    for (const int width : kWidths) {
        if (width > widest) continue;
        const int across = parts_of(a.tokens, width);
        if (width > 16 && across == parts_of(a.tokens, width - 16) && width - 16 >= a.tokens) continue;  // wider than all there is
        const int columns = round16(parts_of(a.tokens, across));
        const float tail = columns * 13.0f;
        auto consider = [&](int down, int split) {
            int height = parts_of(a.outputs, down);
            if (columns > 16 && most % 8 == 0) height = (height + 7) & ~7;  // stores of sixteen bytes
            const int tiles = parts_of(a.outputs, height) * across;
            if (split > 1 && tiles > most_clusters<kOp, T, kCuts>(split)) return;
            const int busy = std::min(tiles * split, sms), rounds = split > 1 ? 1 : parts_of(tiles, sms);
            const float block = block_ns(paired ? 2 * height : height, columns, columns, busy / (6500.0f * across));
            const float t = rounds * parts_of(blocks, split) * std::max(block, 1.3f * std::min(parts_of(a.outputs, height), sms)) + tail +
                            (split > 1 ? 1500.0f + columns * 10.0f : 0.0f);
            if (t < least * 0.999f) least = t, best = DensePlan{height, columns, split, false};
        };
        consider(least_down, 1);
        for (int fill = 1; fill <= 2; ++fill) {
            const int down = fill * sms / across;
            if (down > least_down && parts_of(a.outputs, down) >= std::min(most, 8)) consider(down, 1);
        }
        for (int split = 2; split <= std::min(kMaxSplit, blocks); ++split) {
            const int room = most_clusters<kOp, T, kCuts>(split), down = room / across;
            if (down < least_down) break;
            consider(least_down, split);
            if (down > least_down && parts_of(a.outputs, down) >= std::min(most, 8)) consider(down, split);
        }
        if (width % 32 == 0) {
            const int wide = (parts_of(a.tokens, across) + 31) / 32 * 32, tiles = parts_of(a.outputs, 2 * most) * across, units = most_clusters<kOp, T, kPairs>(2);
            if (units < 1) continue;
            const float t = parts_of(tiles, units) * blocks * block_ns(paired ? 2 * most : most, wide, wide / 2, 2 * std::min(tiles, units) / (6500.0f * across)) + tail;
            if (t < least * 0.999f) least = t, best = DensePlan{most, wide, 1, true};
        }
    }
    return best;
}

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <TilesOp kOp, typename T>
int linear_of(const a2a_linear_args& a, const Ready& gpu, cudaStream_t st) {
    const bool paired = a.activation == A2A_ACT_SWIGLU;
    TilesParams p{};
    p.error = gpu.error;
    p.inner = a.inputs, p.features = a.outputs, p.paired = paired, p.groups = 1, p.tokens = a.tokens;
    p.activation = a.activation, p.bias_fp32 = a.bias_dtype == A2A_DTYPE_FP32;
    p.bias = a.bias, p.residual = a.residual, p.residual_stride = a.residual_stride, p.y = a.y, p.y_stride = a.y_stride;
    p.wide_stores = a.y_stride % 8 == 0 && aligned(a.y) && (a.residual == nullptr || (a.residual_stride % 8 == 0 && aligned(a.residual)));
    const DensePlan plan = dense_plan<kOp, T>(a, paired, gpu.sms);
    p.columns = plan.columns, p.full = plan.height, p.split = plan.split;
    int rc = weights_map(&p.weights, a.dtype, a.weight, 1, a.outputs, paired, a.inputs, a.weight_stride, plan.height);
    if (rc == A2A_OK) rc = rows_map(&p.rows, a.dtype, a.x, a.tokens, a.inputs, a.x_stride, plan.pair ? p.columns / 2 : p.columns);
    if (rc != A2A_OK) return rc;
    if (plan.pair) {
        const int tiles = parts_of(a.outputs, 2 * plan.height) * parts_of(a.tokens, plan.columns);
        return launch_tiles<kOp, T, kPairs>(p, 2 * std::min(tiles, most_clusters<kOp, T, kPairs>(2)), 2, st);
    }
    const int tiles = parts_of(a.outputs, plan.height) * parts_of(a.tokens, plan.columns);
    return plan.split > 1 ? launch_tiles<kOp, T, kCuts>(p, tiles * plan.split, plan.split, st) : launch_tiles<kOp, T>(p, std::min(tiles, gpu.sms), 1, st);
}

size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

// The workspace of a layer: the experts' inner values, and the rows of every pair.
struct LayerSpace {
    size_t parts, end;
};
LayerSpace layer_space(int tokens, int topk, int hidden_dim, int inner) {
    LayerSpace s{};
    const size_t pairs = (size_t)tokens * topk;
    s.parts = round256(pairs * inner * 2);
    s.end = s.parts + round256(pairs * hidden_dim * 4);
    return s;
}

bool sizes_fit(int experts, int hidden_dim, int inner) {
    return experts >= 1 && experts <= A2A_MAX_EXPERTS && hidden_dim >= 8 && hidden_dim % 8 == 0 && hidden_dim <= A2A_MAX_PRODUCT && inner >= 8 &&
           inner % 8 == 0 && inner <= A2A_MAX_PRODUCT;
}

// Sizes and weights of a launch over experts, in boxes of a whole tile and in pieces.
int expert_maps(TilesParams& p, int dtype, const void* weights, int experts, int features, bool paired, int inner) {
    p.inner = inner, p.features = features, p.paired = paired;
    p.full = std::min(paired ? kTileRows / 2 : kTileRows, features);
    const int rc = weights_map(&p.weights, dtype, weights, experts, features, paired, inner, inner, p.full);
    return rc == A2A_OK ? weights_map(&p.weights_piece, dtype, weights, experts, features, paired, inner, inner, kPieceRows / (paired ? 2 : 1)) : rc;
}
// Rows that lie in runs.
int run_maps(TilesParams& p, int dtype, const void* rows, long long count) {
    int rc = rows_map(&p.rows, dtype, rows, count, p.inner, p.inner, 64);
    if (rc == A2A_OK) rc = rows_map(&p.rows_some, dtype, rows, count, p.inner, p.inner, 32);
    return rc == A2A_OK ? rows_map(&p.rows_few, dtype, rows, count, p.inner, p.inner, 8) : rc;
}

template <typename T>
int layer_of(const a2a_layer_args& a, const Ready& gpu, cudaStream_t st) {
    uint8_t* const space = static_cast<uint8_t*>(a.workspace);
    const LayerSpace at = layer_space(a.tokens, a.topk, a.hidden_dim, a.inner);
    TilesParams p{};
    p.error = gpu.error;
    p.groups = a.experts, p.tokens = a.tokens, p.topk = a.topk, p.indices = a.topk_idx, p.weights_of = a.topk_weights;
    p.hidden = space, p.parts = reinterpret_cast<float*>(space + at.parts);
    p.columns = kMaxColumns;
    int rc = expert_maps(p, a.dtype, a.gate_up, a.experts, a.inner, true, a.hidden_dim);
    p.sorted = a.tokens > kSpreadTokens;
    if (rc == A2A_OK && !p.sorted) rc = rows_map(&p.rows, a.dtype, a.x, a.tokens, a.hidden_dim, a.hidden_dim, round16(a.tokens));
    if (rc == A2A_OK && p.sorted) {
        // where the second product will have its rows of pairs, which are wider
        rc = run_maps(p, a.dtype, p.parts, (long long)a.tokens * a.topk);
        SortParams sort{a.x, a.topk_idx, p.parts, a.tokens, a.topk, a.experts, a.hidden_dim * 2};
        if (rc == A2A_OK) rc = launch(reinterpret_cast<const void*>(&layer_rows_kernel), a.tokens * a.topk, kSortThreads, 0, 1, &sort, st);
    }
    if (rc == A2A_OK) rc = launch_tiles<kLayerUp, T>(p, gpu.sms, 1, st);
    if (rc != A2A_OK) return rc;
    rc = expert_maps(p, a.dtype, a.down, a.experts, a.hidden_dim, false, a.inner);
    if (rc == A2A_OK) rc = run_maps(p, a.dtype, p.hidden, (long long)a.tokens * a.topk);
    if (rc == A2A_OK) rc = launch_tiles<kLayerDown, T>(p, gpu.sms, 1, st);
    if (rc != A2A_OK) return rc;
    SumParams sum{p.parts, a.topk_idx, a.residual, a.y, a.topk, a.experts, a.hidden_dim};
    return launch(reinterpret_cast<const void*>(&layer_sum_kernel<T>), dim3(a.tokens, parts_of(a.hidden_dim, 4 * kSumThreads)), kSumThreads, 0, 1, &sum, st);
}

// Rows of inner values that a call on slabs may have: those of a slab are rounded up to whole steps.
long long inner_rows(int local_experts, int world, int capacity) { return (long long)local_experts * world * ((capacity + kManyStep - 1) & -kManyStep); }

template <typename T>
int experts_of(const a2a_experts_args& a, const Ready& gpu, cudaStream_t st) {
    const long long rows = (long long)a.local_experts * a.world * a.capacity;
    TilesParams p{};
    p.error = gpu.error;
    p.groups = a.local_experts, p.counts = a.counts, p.world = a.world, p.capacity = a.capacity, p.hidden = a.workspace;
    p.columns = kMaxColumns;
    int rc = expert_maps(p, a.dtype, a.gate_up, a.local_experts, a.inner, true, a.hidden_dim);
    if (rc == A2A_OK) rc = run_maps(p, a.dtype, a.rows, rows);
    if (rc == A2A_OK) rc = launch_tiles<kSlabUp, T, kPairs>(p, 2 * std::max(1, most_clusters<kSlabUp, T, kPairs>(2)), 2, st);
    if (rc != A2A_OK) return rc;
    p.y = a.out, p.wide_stores = aligned(a.out);
    rc = expert_maps(p, a.dtype, a.down, a.local_experts, a.hidden_dim, false, a.inner);
    if (rc == A2A_OK) rc = run_maps(p, a.dtype, a.workspace, inner_rows(a.local_experts, a.world, a.capacity));
    return rc == A2A_OK ? launch_tiles<kSlabDown, T, kPairs>(p, 2 * std::max(1, most_clusters<kSlabDown, T, kPairs>(2)), 2, st) : rc;
}

bool dtype16(int dtype) { return dtype == A2A_DTYPE_BF16 || dtype == A2A_DTYPE_FP16; }

}  // namespace

extern "C" int a2a_linear(const a2a_linear_args* args, void* stream) {
    if (args == nullptr) return A2A_ERR_CONFIG;
    const a2a_linear_args& a = *args;
    if (!dtype16(a.dtype) || (a.out_dtype != a.dtype && a.out_dtype != A2A_DTYPE_FP32)) return A2A_ERR_CONFIG;
    if (a.bias != nullptr && a.bias_dtype != a.dtype && a.bias_dtype != A2A_DTYPE_FP32) return A2A_ERR_CONFIG;
    if (a.activation < A2A_ACT_NONE || a.activation > A2A_ACT_SWIGLU) return A2A_ERR_CONFIG;
    if (a.tokens < 0 || a.tokens > A2A_MAX_ROWS || a.outputs < 1 || a.outputs > A2A_MAX_OUTPUTS || a.inputs < 8 || a.inputs % 8 != 0 || a.inputs > A2A_MAX_PRODUCT)
        return A2A_ERR_CONFIG;
    if (a.tokens == 0) return A2A_OK;
    if (a.x == nullptr || a.weight == nullptr || a.y == nullptr || !aligned(a.x) || !aligned(a.weight)) return A2A_ERR_CONFIG;
    if (a.x_stride < a.inputs || a.x_stride % 8 != 0 || a.weight_stride < a.inputs || a.weight_stride % 8 != 0) return A2A_ERR_CONFIG;
    if (a.y_stride < a.outputs || (a.residual != nullptr && a.residual_stride < 0)) return A2A_ERR_CONFIG;
    Ready gpu{};
    const int rc = get_ready(&gpu);
    if (rc != A2A_OK) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (a.out_dtype == A2A_DTYPE_FP32)
        return a.dtype == A2A_DTYPE_BF16 ? linear_of<kDense32, __nv_bfloat16>(a, gpu, st) : linear_of<kDense32, __half>(a, gpu, st);
    return a.dtype == A2A_DTYPE_BF16 ? linear_of<kDense, __nv_bfloat16>(a, gpu, st) : linear_of<kDense, __half>(a, gpu, st);
}

extern "C" size_t a2a_layer_workspace(int num_tokens, int experts_per_token, int hidden_dim, int inner) {
    if (num_tokens < 0 || experts_per_token < 1 || hidden_dim < 1 || inner < 1) return 0;
    return layer_space(num_tokens, experts_per_token, hidden_dim, inner).end;
}

extern "C" int a2a_layer(const a2a_layer_args* args, void* stream) {
    if (args == nullptr) return A2A_ERR_CONFIG;
    const a2a_layer_args& a = *args;
    if (!dtype16(a.dtype) || !sizes_fit(a.experts, a.hidden_dim, a.inner)) return A2A_ERR_CONFIG;
    if (a.tokens < 0 || a.tokens > A2A_MAX_LAYER_TOKENS || a.topk < 1 || a.topk > A2A_MAX_TOPK) return A2A_ERR_CONFIG;
    if (a.tokens == 0) return A2A_OK;
    if (a.x == nullptr || a.topk_idx == nullptr || a.topk_weights == nullptr || a.gate_up == nullptr || a.down == nullptr || a.y == nullptr ||
        a.workspace == nullptr)
        return A2A_ERR_CONFIG;
    if (!aligned(a.x) || !aligned(a.gate_up) || !aligned(a.down) || reinterpret_cast<uintptr_t>(a.workspace) % 256 != 0) return A2A_ERR_CONFIG;
    if (a.workspace_bytes < layer_space(a.tokens, a.topk, a.hidden_dim, a.inner).end) return A2A_ERR_CAPACITY;
    Ready gpu{};
    const int rc = get_ready(&gpu);
    if (rc != A2A_OK) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    return a.dtype == A2A_DTYPE_BF16 ? layer_of<__nv_bfloat16>(a, gpu, st) : layer_of<__half>(a, gpu, st);
}

extern "C" size_t a2a_experts_workspace(int local_experts, int world_size, int capacity, int inner) {
    if (local_experts < 1 || world_size < 1 || capacity < 1 || inner < 1) return 0;
    return round256((size_t)inner_rows(local_experts, world_size, capacity) * inner * 2);
}

extern "C" int a2a_experts(const a2a_experts_args* args, void* stream) {
    if (args == nullptr) return A2A_ERR_CONFIG;
    const a2a_experts_args& a = *args;
    if (!dtype16(a.dtype) || !sizes_fit(a.local_experts, a.hidden_dim, a.inner)) return A2A_ERR_CONFIG;
    if (a.world < 1 || a.world > A2A_MAX_WORLD || a.capacity < 1 || a.capacity > 65535) return A2A_ERR_CONFIG;
    if (a.rows == nullptr || a.counts == nullptr || a.gate_up == nullptr || a.down == nullptr || a.out == nullptr || a.workspace == nullptr)
        return A2A_ERR_CONFIG;
    if (!aligned(a.rows) || !aligned(a.gate_up) || !aligned(a.down) || reinterpret_cast<uintptr_t>(a.workspace) % 256 != 0) return A2A_ERR_CONFIG;
    if (a.workspace_bytes < a2a_experts_workspace(a.local_experts, a.world, a.capacity, a.inner)) return A2A_ERR_CAPACITY;
    Ready gpu{};
    const int rc = get_ready(&gpu);
    if (rc != A2A_OK) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    return a.dtype == A2A_DTYPE_BF16 ? experts_of<__nv_bfloat16>(a, gpu, st) : experts_of<__half>(a, gpu, st);
}

extern "C" int32_t* a2a_product_word(int device) { return error_word(device); }

extern "C" int a2a_product_status(int32_t* code) {
    if (code == nullptr) return A2A_ERR_CONFIG;
    Ready gpu{};
    const int rc = get_ready(&gpu);
    if (rc < 0) return rc;
    const cudaError_t e = cudaDeviceSynchronize();
    *code = __atomic_exchange_n(gpu.error, A2A_OK, __ATOMIC_ACQ_REL);
    return e == cudaSuccess ? A2A_OK : -(int)e;
}
