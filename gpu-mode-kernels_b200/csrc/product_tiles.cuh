// Products of weights with rows on the tensor cores (tcgen05): y[row] = W x[row], for one matrix and all rows (a dense product) or
// for a matrix per expert and the rows that chose it.
//
// The weights are the operand with 128 rows of a tile, the rows of x its columns: 16 to 256 of them, as many as there are. A decode
// batch leaves an expert a few rows; a tile of 128 rows of x would be filled to a few per cent, this one moves nothing but weights.
// Weights come through a ring of tiles in shared memory (tensor copies, 128-byte swizzle), 64 of the inner length at a time; the
// rows of an expert, which lie anywhere, four at a time by gathering copies into the same stage. Sums are fp32 in tensor memory,
// two buffers of 256 columns, so that one tile's epilogue runs beside the next one's products.
//
// Roles of the eight warps: 0 weights, 1 products, 2 rows, 3 the lists of rows, 4 to 7 the epilogue.
//
// SwiGLU: a tile is 64 features, their gate and up rows in turn (the tensor map's second dimension steps from gate to up), so that
// neighbouring lanes of the epilogue hold the two and exchange by shuffles.
#pragma once

#include "product_device.cuh"

namespace {

enum TilesOp { kDense, kLayerUp, kLayerDown, kSlabUp, kSlabDown };

constexpr int kTileRows = 128, kTileInner = 64, kMaxColumns = 256;
constexpr int kTilesThreads = 256;
constexpr int kRingBytes = 192 * 1024, kMaxStages = 12;
constexpr int kMaxGroups = A2A_MAX_EXPERTS;
constexpr int kTmemColumns = 512;

struct TilesParams {
    CUtensorMap weights;  // [groups][rows or features][1 or gate, up][inner], boxes of 128 rows by 64
    CUtensorMap rows;     // kDense: boxes of `columns` rows by 64; else of one row, for gathering
    int inner;            // length of a sum
    int features;         // of the output, per group
    int paired;           // SwiGLU
    int groups;           // matrices
    int columns;          // most columns a tile may have
    // kDense: rows of x, and the epilogue
    int tokens, activation, out_fp32, bias_fp32;
    const void* bias;
    const void* residual;  // also kLayerDown
    long long residual_stride;
    void* y;
    long long y_stride;
    // kLayer*
    const int* indices;
    const float* weights_of;
    int topk;
    void* hidden;   // [row][features] of *Up
    float* parts;   // [pair][features] of kLayerDown
    int* tickets;   // [token][tile of features] of kLayerDown, zeroed by kLayerUp
    int ticket_count;
    // kSlab*
    const int* counts;
    int world, capacity;
};

struct TilesShared {
    uint64_t full[kMaxStages], empty[kMaxStages];
    uint64_t sums_full[2], sums_empty[2];
    uint64_t list_full[2], list_empty[2];
    uint32_t tmem;
    int gave_up;
    int largest;    // rows of the largest group
    int last_count;
    int begin[kMaxGroups + 1];  // first tile of a group
    int count[kMaxGroups];      // its rows
    int list[2][kMaxColumns];
    float scale[2][kMaxColumns];
    int last[kMaxColumns];
};

constexpr size_t kTilesSharedBytes = 1024 + kRingBytes + sizeof(TilesShared);
static_assert(kTilesSharedBytes <= 227 * 1024, "a block's shared memory");

struct Tile {
    int group, m, first, columns;  // matrix, tile of its features, first row, rows
};

__device__ __forceinline__ int round16(int n) { return (n + 15) & ~15; }

template <TilesOp kOp, typename T>
__global__ void __launch_bounds__(kTilesThreads, 1) product_tiles_kernel(const __grid_constant__ TilesParams p) {
    constexpr bool kGrouped = kOp != kDense, kLayer = kOp == kLayerUp || kOp == kLayerDown;
    constexpr bool kFirst = kOp == kDense || kOp == kLayerUp || kOp == kSlabUp;  // nothing of the same call runs before it
    extern __shared__ uint8_t shared_raw[];
    uint8_t* const ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(shared_raw) + 1023) & ~(uintptr_t)1023);
    TilesShared& s = *reinterpret_cast<TilesShared*>(ring + kRingBytes);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < kMaxStages; ++i) {
            barrier_init(&s.full[i], 2);
            barrier_init(&s.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            barrier_init(&s.sums_full[i], 1);
            barrier_init(&s.sums_empty[i], 4);
            barrier_init(&s.list_full[i], 1);
            barrier_init(&s.list_empty[i], 2);
        }
        s.gave_up = s.largest = s.last_count = 0;
        barrier_init_done();
        prefetch_map(&p.weights);
        prefetch_map(&p.rows);
    }
    if (warp == 1) tmem_alloc(&s.tmem, kTmemColumns);
    // The second product of a call reads weights, indices and counts ahead of this: what wrote those was through before the
    // first product let this launch begin.
    if (kFirst) {
        cudaGridDependencySynchronize();
        cudaTriggerProgrammaticLaunchCompletion();
    }
    const int feature_tiles = (p.features + (p.paired ? kTileRows / 2 : kTileRows) - 1) / (p.paired ? kTileRows / 2 : kTileRows);
    if (kOp == kLayerUp)
        for (int i = blockIdx.x * kTilesThreads + tid; i < p.ticket_count; i += gridDim.x * kTilesThreads) p.tickets[i] = 0;

    // ---- how many rows every group has, and so the tiles ----
    int columns = p.columns;
    if (kGrouped) {
        for (int g = tid; g < p.groups; g += kTilesThreads) {
            int n = 0;
            if (!kLayer)
                for (int src = 0; src < p.world; ++src) n += min(max(p.counts[(size_t)src * 4 * p.groups + g], 0), p.capacity);
            s.count[g] = n;
        }
        __syncthreads();
        if (kLayer)
            for (int i = tid; i < p.tokens * p.topk; i += kTilesThreads) {
                const int e = p.indices[i];
                if (e >= 0 && e < p.groups) atomicAdd(&s.count[e], 1);
            }
        __syncthreads();
        int most = 0;
        for (int g = tid; g < p.groups; g += kTilesThreads) most = max(most, s.count[g]);
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) atomicMax(&s.largest, most);
        __syncthreads();
        columns = min(columns, max(16, round16(s.largest)));
        if (warp == 0) {
            int run = 0;
            for (int g0 = 0; g0 < p.groups; g0 += 32) {
                const int g = g0 + lane;
                const int own = g < p.groups ? (s.count[g] + columns - 1) / columns * feature_tiles : 0;
                int sum = own;
                for (int d = 1; d < 32; d <<= 1) {
                    const int left = __shfl_up_sync(0xffffffffu, sum, d);
                    if (lane >= d) sum += left;
                }
                if (g < p.groups) s.begin[g] = run + sum - own;
                run += __shfl_sync(0xffffffffu, sum, 31);
            }
            if (lane == 0) s.begin[p.groups] = run;
        }
    }
    tcgen05_before_sync();
    __syncthreads();
    tcgen05_after_sync();
    const uint32_t tmem = s.tmem;
    const int tiles = kGrouped ? s.begin[p.groups] : (p.tokens + columns - 1) / columns * feature_tiles;
    const int stage_bytes = kTileRows * 128 + columns * 128;
    const int stages = min(kMaxStages, kRingBytes / stage_bytes);
    const int steps = (p.inner + kTileInner - 1) / kTileInner;

    // Tiles that share weights come one after the other, so that blocks read them together.
    auto tile_of = [&](int t) {
        Tile x;
        int rows;
        if (kGrouped) {
            int lo = 0, hi = p.groups - 1;  // the last group that begins at or before t; groups without rows begin with the next
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (s.begin[mid] <= t) lo = mid;
                else hi = mid - 1;
            }
            x.group = lo;
            rows = s.count[lo];
            t -= s.begin[lo];
        } else {
            x.group = 0;
            rows = p.tokens;
        }
        const int across = (rows + columns - 1) / columns;
        x.m = t / across;
        x.first = (t - x.m * across) * columns;
        x.columns = min(columns, rows - x.first);
        return x;
    };

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 1;
            for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
                const Tile x = tile_of(t);
                const int f = x.m * (p.paired ? kTileRows / 2 : kTileRows);
                for (int i = 0; i < steps; ++i) {
                    if (!barrier_wait(&s.empty[stage], phase, &s.gave_up)) goto weights_done;
                    barrier_expect(&s.full[stage], kTileRows * 128);
                    copy_tile_4d(ring + stage * stage_bytes, &p.weights, i * kTileInner, 0, f, x.group, &s.full[stage]);
                    if (++stage == stages) stage = 0, phase ^= 1;
                }
            }
        weights_done:;
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int stage = 0, n = 0;
            uint32_t phase = 0;
            for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++n) {
                const Tile x = tile_of(t);
                const int buffer = n & 1;
                const uint32_t descriptor = instruction_descriptor(Element<T>::kFormat, round16(x.columns));
                if (!barrier_wait(&s.sums_empty[buffer], ((n >> 1) & 1) ^ 1, &s.gave_up)) goto products_done;
                tcgen05_after_sync();
                for (int i = 0; i < steps; ++i) {
                    if (!barrier_wait(&s.full[stage], phase, &s.gave_up)) goto products_done;
                    tcgen05_after_sync();
                    const uint64_t a = operand_descriptor(ring + stage * stage_bytes);
                    const uint64_t b = operand_descriptor(ring + stage * stage_bytes + kTileRows * 128);
#pragma unroll
                    for (int k = 0; k < kTileInner / 16; ++k)  // 16 of the inner length are 32 bytes of a row
                        tcgen05_mma(tmem + buffer * kMaxColumns, a + 2 * k, b + 2 * k, descriptor, i + k > 0);
                    tcgen05_commit(&s.empty[stage]);
                    if (++stage == stages) stage = 0, phase ^= 1;
                }
                tcgen05_commit(&s.sums_full[buffer]);
            }
        products_done:;
        }
    } else if (warp == 2) {
        if (!kFirst) cudaGridDependencySynchronize();
        int stage = 0, n = 0;
        uint32_t phase = 1;
        for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++n) {
            const Tile x = tile_of(t);
            if (!kGrouped) {
                if (lane == 0)
                    for (int i = 0; i < steps; ++i) {
                        if (!barrier_wait(&s.empty[stage], phase, &s.gave_up)) break;
                        barrier_expect(&s.full[stage], columns * 128);
                        copy_tile_2d(ring + stage * stage_bytes + kTileRows * 128, &p.rows, i * kTileInner, x.first, &s.full[stage]);
                        if (++stage == stages) stage = 0, phase ^= 1;
                    }
                if (s.gave_up) break;
                continue;
            }
            const int buffer = n & 1;
            if (!__all_sync(0xffffffffu, barrier_wait(&s.list_full[buffer], (n >> 1) & 1, &s.gave_up))) break;
            // Lane i's rows 4 i to 4 i + 3 and, of more than 128, the same further on. Behind the last row the first one stands
            // again: its sums are not read.
            int r[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int c = 128 * h + 4 * lane + j;
                    const int row = s.list[buffer][c < x.columns ? c : 0];
                    r[h][j] = kOp == kLayerUp ? row / p.topk : row;
                }
            __syncwarp();
            if (lane == 0) barrier_arrive(&s.list_empty[buffer]);
            const int fours = (x.columns + 3) >> 2;
            bool ok = true;
            for (int i = 0; i < steps; ++i) {
                ok = __all_sync(0xffffffffu, barrier_wait(&s.empty[stage], phase, &s.gave_up));
                if (!ok) break;
                if (lane == 0) barrier_expect(&s.full[stage], fours * 512);
                __syncwarp();
                uint8_t* const at = ring + stage * stage_bytes + kTileRows * 128;
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (32 * h + lane < fours)
                        copy_rows_4(at + (32 * h + lane) * 512, &p.rows, i * kTileInner, r[h][0], r[h][1], r[h][2], r[h][3], &s.full[stage]);
                if (++stage == stages) stage = 0, phase ^= 1;
            }
            if (!ok) break;
        }
    } else if (warp == 3) {
        if (kGrouped) {
            int n = 0;
            for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++n) {
                const Tile x = tile_of(t);
                const int buffer = n & 1;
                if (!__all_sync(0xffffffffu, barrier_wait(&s.list_empty[buffer], ((n >> 1) & 1) ^ 1, &s.gave_up))) break;
                if (kLayer) {
                    // pairs in ascending order: which tile of a group a pair belongs to is the same for every block
                    const int pairs = p.tokens * p.topk;
                    int seen = 0;
                    for (int i0 = 0; i0 < pairs && seen < x.first + x.columns; i0 += 128) {
                        int e[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int i = i0 + 32 * j + lane;
                            e[j] = i < pairs ? p.indices[i] : -1;
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const unsigned mine = __ballot_sync(0xffffffffu, e[j] == x.group);
                            const int at = seen + __popc(mine & ((1u << lane) - 1)) - x.first;
                            if (e[j] == x.group && at >= 0 && at < x.columns) {
                                const int pair = i0 + 32 * j + lane;
                                s.list[buffer][at] = pair;
                                if (kOp == kLayerDown) s.scale[buffer][at] = p.weights_of[pair];
                            }
                            seen += __popc(mine);
                        }
                    }
                } else {
                    for (int c = lane; c < x.columns; c += 32) {
                        int r = x.first + c, src = 0;
                        for (;;) {
                            const int have = min(max(p.counts[(size_t)src * 4 * p.groups + x.group], 0), p.capacity);
                            if (r < have || src == p.world - 1) break;
                            r -= have;
                            ++src;
                        }
                        s.list[buffer][c] = (x.group * p.world + src) * p.capacity + min(r, p.capacity - 1);
                    }
                }
                __syncwarp();
                if (lane == 0) barrier_arrive(&s.list_full[buffer]);
            }
        }
    } else {
        const int quarter = warp - 4, at = tid - 128;
        if (!kFirst) {
            cudaGridDependencySynchronize();
            cudaTriggerProgrammaticLaunchCompletion();
        }
        if (kOp == kLayerDown) {
            // tokens that no expert of the layer was chosen for: nobody below draws a ticket for them
            for (int token = blockIdx.x * 4 + quarter; token < p.tokens; token += gridDim.x * 4) {
                const int e = lane < p.topk ? p.indices[token * p.topk + lane] : -1;
                if (__any_sync(0xffffffffu, e >= 0 && e < p.groups)) continue;
                for (int f = lane; f < p.features; f += 32)
                    static_cast<T*>(p.y)[(size_t)token * p.features + f] =
                        p.residual != nullptr ? static_cast<const T*>(p.residual)[(size_t)token * p.features + f] : Element<T>::from_float(0.0f);
            }
        }
        int n = 0;
        for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++n) {
            const Tile x = tile_of(t);
            const int buffer = n & 1;
            bool here = !kGrouped || barrier_wait(&s.list_full[buffer], (n >> 1) & 1, &s.gave_up);
            here = here && barrier_wait(&s.sums_full[buffer], (n >> 1) & 1, &s.gave_up);
            if (!named_all(1, 128, here)) break;  // all four warps go on, or none
            tcgen05_after_sync();
            const uint32_t sums = tmem + buffer * kMaxColumns + ((uint32_t)(quarter * 32) << 16);
            // this lane's feature, and its row of the weights
            const int f = p.paired ? x.m * (kTileRows / 2) + quarter * 16 + (lane >> 1) : x.m * kTileRows + quarter * 32 + lane;
            const bool inside = f < p.features;
            float bias = 0.0f;
            if (kOp == kDense && p.bias != nullptr && inside)
                bias = load_any<T>(p.bias, p.paired ? (size_t)(lane & 1) * p.features + f : f, p.bias_fp32);
            for (int c0 = 0; c0 < x.columns; c0 += 16) {
                float v[16];
                tmem_load_16(sums + c0, v);
                if (p.paired) {
                    // lanes 2 i and 2 i + 1 hold gate and up of a feature: the first finishes the even columns, the second the odd ones
                    const bool up = lane & 1;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float even = v[2 * j] + bias, odd = v[2 * j + 1] + bias;
                        const float other = __shfl_xor_sync(0xffffffffu, up ? even : odd, 1);
                        const float gate = up ? other : even, lift = up ? odd : other;
                        v[j] = silu(gate) * lift;
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int c = c0 + 2 * j + (up ? 1 : 0);
                        if (!inside || c >= x.columns) continue;
                        if (kOp == kDense) {
                            const size_t token = x.first + c;
                            const float r = p.residual != nullptr ? load_any<T>(p.residual, token * p.residual_stride + f, p.out_fp32) : 0.0f;
                            store_any<T>(p.y, token * p.y_stride + f, v[j] + r, p.out_fp32);
                        } else {
                            // Rounded to the rows' type, since the next product takes 16-bit operands.
                            static_cast<T*>(p.hidden)[(size_t)s.list[buffer][c] * p.features + f] = Element<T>::from_float(v[j]);
                        }
                    }
                } else {
                    float r[16];
                    if (kOp == kDense && p.residual != nullptr) {
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            r[j] = inside && c0 + j < x.columns
                                       ? load_any<T>(p.residual, (size_t)(x.first + c0 + j) * p.residual_stride + f, p.out_fp32)
                                       : 0.0f;
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int c = c0 + j;
                        if (!inside || c >= x.columns) continue;
                        if (kOp == kDense) {
                            float out = activate(v[j] + bias, p.activation);
                            if (p.residual != nullptr) out += r[j];
                            store_any<T>(p.y, (size_t)(x.first + c) * p.y_stride + f, out, p.out_fp32);
                        } else if (kOp == kLayerDown) {
                            p.parts[(size_t)s.list[buffer][c] * p.features + f] = s.scale[buffer][c] * v[j];
                        } else {
                            static_cast<T*>(p.y)[(size_t)s.list[buffer][c] * p.features + f] = Element<T>::from_float(v[j]);
                        }
                    }
                }
            }
            tcgen05_before_sync();
            __syncwarp();
            if (lane == 0) barrier_arrive(&s.sums_empty[buffer]);
            if (kOp == kLayerDown) {
                // The tile that brings a token's last row adds its rows up, in the order of the token's choices whichever tile it is.
                __threadfence();
                named_sync(1, 128);
                for (int c = at; c < x.columns; c += 128) {
                    const int token = s.list[buffer][c] / p.topk;
                    int due = 0;
                    for (int k = 0; k < p.topk; ++k) {
                        const int e = p.indices[token * p.topk + k];
                        due += e >= 0 && e < p.groups;
                    }
                    if (atomicAdd(&p.tickets[token * feature_tiles + x.m], 1) == due - 1) s.last[atomicAdd(&s.last_count, 1)] = token;
                }
                __threadfence();
                named_sync(1, 128);
                const int ready = s.last_count;
                for (int i = quarter; i < ready; i += 4) {
                    const int token = s.last[i], g = x.m * kTileRows + 4 * lane;
                    if (g >= p.features) continue;  // features are a multiple of 8
                    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    for (int k = 0; k < p.topk; ++k) {
                        const int e = p.indices[token * p.topk + k];
                        if (e < 0 || e >= p.groups) continue;
                        const float4 part = __ldcg(reinterpret_cast<const float4*>(p.parts + ((size_t)token * p.topk + k) * p.features + g));
                        sum.x += part.x, sum.y += part.y, sum.z += part.z, sum.w += part.w;
                    }
                    const float out[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const size_t o = (size_t)token * p.features + g + j;
                        const float r = p.residual != nullptr ? Element<T>::to_float(static_cast<const T*>(p.residual)[o]) : 0.0f;
                        static_cast<T*>(p.y)[o] = Element<T>::from_float(out[j] + r);
                    }
                }
                named_sync(1, 128);
                if (at == 0) s.last_count = 0;
                // the next tile's first named_sync orders this before its counting
            }
            if (kGrouped) {
                if (kOp != kLayerDown) named_sync(1, 128);
                if (at == 0) barrier_arrive(&s.list_empty[buffer]);
            }
        }
    }
    __syncwarp();
    tcgen05_before_sync();
    __syncthreads();
    tcgen05_after_sync();
    if (s.gave_up) {
        // copies and products in flight end in less than this
        const long long begin = now_ns();
        while (now_ns() - begin < 1000000) __nanosleep(1000);
        if (tid == 0) atomicExch(&g_product_error, A2A_ERR_TIMEOUT);
        __syncthreads();
    }
    if (warp == 1) tmem_free(tmem, kTmemColumns);
}

}  // namespace
