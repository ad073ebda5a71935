// Products of weights with up to eight rows (kWide: sixteen): y[row] = W x[row], a dense product or a whole layer's experts for a few
// tokens. Nothing but reading the weights once costs anything here, so this is built around loads.
//
// Every SM gets the same number of the weights' rows, to one (7168 rows are 48.4 for each of 148 SMs; tiles of 16 would be 3.03, and so
// four on some). A block takes its rows in tiles of up to 16; its 16 warps share the tile's inner length, 64 at a time. A warp loads
// the weights straight into the registers of an m16n8k16 operand: which inner index stands at which place of the operand is free as
// long as the rows of x agree, so a thread takes eight neighbouring values of a row, 16 bytes, for two instructions. kDepth such
// steps are on their way at any time: 128 KB an SM. The rows of x come through L1, eight columns of the instruction, the
// columns of rows that are not there as zeros. The warps' sums meet in shared memory once a tile, while the next tile's loads are on their way.
//
// The first product of a layer takes gate and up rows of up to eight features as the two halves of a tile; the second one all chosen
// experts for its rows of the output, one after the other, so that a token's sum over its experts stays in the block: no second pass,
// no atomics, one rounding.
#pragma once

#include "product_device.cuh"

namespace {

enum RowsOp { kRowsDense, kRowsUp, kRowsDown };

constexpr int kRowsThreads = 512, kRowsWarps = kRowsThreads / 32;
constexpr int kDepth = 4;
constexpr int kRowsTokens = 8;                      // columns of one instruction
constexpr int kRowsPairs = kRowsTokens * A2A_MAX_TOPK;

struct RowsParams {
    const void* weights;
    long long weights_stride;  // between rows, elements
    const void* x;             // kRowsDense, kRowsUp: [tokens][inner]; kRowsDown: [pair][inner]
    long long x_stride;
    int inner, features, tokens;
    int activation, paired, out_fp32, bias_fp32;
    const void* bias;
    const void* residual;
    long long residual_stride;
    void* y;  // kRowsUp: [pair][features]
    long long y_stride;
    // kRowsUp, kRowsDown
    const int* indices;
    const float* weights_of;
    int topk, experts;
};

// What the blocks of a layer know of its pairs: the chosen experts in order of their first pair, and for each of them the tokens
// that chose it. A token that chose an expert twice counts once, with both weights.
struct Chosen {
    int first[A2A_MAX_EXPERTS];          // first pair of an expert
    int expert[kRowsPairs];              // chosen experts
    int row[kRowsPairs][kRowsTokens];    // row of the inner values of (chosen expert, token), or -1
    float weight[kRowsPairs][kRowsTokens];
    int scan[kRowsWarps];
};

struct NothingChosen {
    int expert[1], row[1][kRowsTokens];
    float weight[1][kRowsTokens];
};
template <bool kLayer>
struct ChosenOf {
    using type = Chosen;
};
template <>
struct ChosenOf<false> {
    using type = NothingChosen;
};

template <typename T>
__device__ __forceinline__ void multiply(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void multiply<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void multiply<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Weights are read once: they are not kept in L1, which is the rows'.
__device__ __forceinline__ uint4 load_weights(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// Fills `c` from the layer's pairs; all threads of the block. Returns the number of chosen experts.
__device__ __forceinline__ int find_chosen(Chosen& c, const int* indices, const float* weights_of, int tokens, int topk, int experts) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, pairs = tokens * topk;
    for (int i = tid; i < experts; i += kRowsThreads) c.first[i] = kRowsPairs;
    __syncthreads();
    int e = tid < pairs ? indices[tid] : -1;
    if (e >= experts) e = -1;
    if (e >= 0) atomicMin(&c.first[e], tid);
    __syncthreads();
    const bool leads = e >= 0 && c.first[e] == tid;
    const unsigned leaders = __ballot_sync(0xffffffffu, leads);
    if (lane == 0) c.scan[warp] = __popc(leaders);
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < kRowsPairs / 32; ++w) {
        if (w < warp) before += c.scan[w];
        all += c.scan[w];
    }
    __syncthreads();
    if (leads) {
        const int a = before + __popc(leaders & ((1u << lane) - 1));
        c.expert[a] = e;
        c.first[e] = a;  // from here on: the place of the expert among the chosen
    }
    for (int i = tid; i < all * kRowsTokens; i += kRowsThreads) {
        c.row[i / kRowsTokens][i % kRowsTokens] = -1;
        c.weight[i / kRowsTokens][i % kRowsTokens] = 0.0f;
    }
    __syncthreads();
    if (e >= 0) {
        const int token = tid / topk, k = tid - token * topk;
        bool again = false;
        float sum = 0.0f;
        for (int j = 0; j < topk; ++j) {
            const int other = indices[token * topk + j];
            if (other != e) continue;
            if (j < k) again = true;
            sum += weights_of[token * topk + j];
        }
        if (!again) {
            c.row[c.first[e]][token] = tid;
            c.weight[c.first[e]][token] = sum;
        }
    }
    __syncthreads();
    return all;
}

template <RowsOp kOp, typename T, int kWide>
__global__ void __launch_bounds__(kRowsThreads, 1) product_rows_kernel(const __grid_constant__ RowsParams p) {
    constexpr bool kLayer = kOp != kRowsDense;
    __shared__ float4 sums[2][kWide][kRowsWarps][32];
    __shared__ typename ChosenOf<kLayer>::type chosen;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, group = lane >> 2, quad = lane & 3;
    if (kOp != kRowsDown) {
        cudaGridDependencySynchronize();
        cudaTriggerProgrammaticLaunchCompletion();
    }
    // kRowsDown reads indices and weights ahead of the end of kRowsUp: what wrote those was through before kRowsUp let it begin.
    int experts = 1;
    if constexpr (kLayer) experts = find_chosen(chosen, p.indices, p.weights_of, p.tokens, p.topk, p.experts);
    const bool paired = kOp == kRowsUp || (kOp == kRowsDense && p.paired);
    const int height = paired ? 8 : 16;  // features of a tile
    const int chunks = (p.inner + 63) >> 6;
    // this block's features, of all experts for kRowsUp
    const long long total = kOp == kRowsUp ? (long long)experts * p.features : p.features;
    const int begin = (int)(total * blockIdx.x / gridDim.x), end = (int)(total * (blockIdx.x + 1) / gridDim.x);
    // steps of a warp in a tile: 64 of the inner length each, of kRowsDown's experts one after the other
    const long long all_chunks = kOp == kRowsDown ? (long long)experts * chunks : chunks;
    const int steps = max(1, (int)((all_chunks + kRowsWarps - 1) / kRowsWarps));
    const int step0 = kOp == kRowsDown ? min((int)all_chunks, warp * steps) : warp;
    const int own_steps = kOp == kRowsDown ? min(steps, (int)all_chunks - step0) : (chunks - warp + kRowsWarps - 1) / kRowsWarps;

    struct Place {
        int at, size;  // first feature of the tile (of all experts'), and how many
        int step;
    };
    // The tile that begins at feature `at`: the rest of the block's features, within one expert, in equal parts.
    auto height_at = [&](int at) {
        int left = end - at;
        if (kOp == kRowsUp) left = min(left, p.features - at % p.features);
        const int parts = (left + height - 1) / height;
        return parts > 0 ? (left + parts - 1) / parts : 0;
    };
    auto advance = [&](Place& q) {
        if (++q.step == steps) {
            q.step = 0;
            q.at += q.size;
            q.size = height_at(q.at);
        }
    };

    uint4 ring[kDepth][4];
    Place next{begin, height_at(begin), 0}, now = next;
    const T* weights = static_cast<const T*>(p.weights);
    // step `q` of this warp: which expert (kRowsDown: among the chosen) and where in the inner length
    auto locate = [&](const Place& q, int& a, int& inner0) {
        if (kOp == kRowsDown) {
            a = (step0 + q.step) / chunks;
            inner0 = (step0 + q.step - a * chunks) << 6;
        } else {
            a = kOp == kRowsUp ? q.at / p.features : 0;
            inner0 = (step0 + q.step * kRowsWarps) << 6;
        }
    };
    auto fetch = [&](uint4 (&to)[4]) {
        int a, inner0;
        const bool any = next.size > 0 && next.step < own_steps;
        locate(next, a, inner0);
        const uint4 zero = make_uint4(0, 0, 0, 0);
        to[0] = to[1] = to[2] = to[3] = zero;
        if (any) {
            const int feature = kOp == kRowsUp ? next.at - a * p.features : next.at;
            long long matrix = 0;  // the expert's first row
            if (kLayer) matrix = (long long)chosen.expert[a] * p.features * (kOp == kRowsUp ? 2 : 1);
            const bool low = group < next.size, high = paired ? low : group + 8 < next.size;
            const T* const r0 = weights + (matrix + feature + group) * p.weights_stride;
            const T* const r1 = r0 + (paired ? (long long)p.features : 8ll) * p.weights_stride;
            const int k0 = inner0 + 8 * quad, k1 = k0 + 32;
            if (low && k0 < p.inner) to[0] = load_weights(r0 + k0);
            if (high && k0 < p.inner) to[1] = load_weights(r1 + k0);
            if (low && k1 < p.inner) to[2] = load_weights(r0 + k1);
            if (high && k1 < p.inner) to[3] = load_weights(r1 + k1);
        }
        advance(next);
    };

#pragma unroll
    for (int d = 0; d < kDepth; ++d) fetch(ring[d]);
    if (kOp == kRowsDown) {
        cudaGridDependencySynchronize();
        cudaTriggerProgrammaticLaunchCompletion();
    }

    float acc[kWide][4], total_acc[4];
#pragma unroll
    for (int w = 0; w < kWide; ++w)
        for (int j = 0; j < 4; ++j) acc[w][j] = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) total_acc[j] = 0.0f;
    int buffer = 0, current = -1;

    while (now.size > 0) {
#pragma unroll
        for (int d = 0; d < kDepth; ++d) {
            if (now.size == 0) break;
            if (now.step < own_steps) {
                int a, inner0;
                locate(now, a, inner0);
                if (kOp == kRowsDown && a != current) {
                    if (current >= 0) {
                        // columns 2 quad and 2 quad + 1 of the expert that is through
                        const float w0 = chosen.weight[current][2 * quad], w1 = chosen.weight[current][2 * quad + 1];
                        const bool b0 = chosen.row[current][2 * quad] >= 0, b1 = chosen.row[current][2 * quad + 1] >= 0;
                        if (b0) total_acc[0] += w0 * acc[0][0], total_acc[2] += w0 * acc[0][2];
                        if (b1) total_acc[1] += w1 * acc[0][1], total_acc[3] += w1 * acc[0][3];
                        acc[0][0] = acc[0][1] = acc[0][2] = acc[0][3] = 0.0f;
                    }
                    current = a;
                }
                const int k0 = inner0 + 8 * quad, k1 = k0 + 32;
#pragma unroll
                for (int w = 0; w < kWide; ++w) {
                    const int column = 8 * w + group;
                    int row = column < p.tokens ? column : -1;
                    if (kLayer && row >= 0) {
                        row = chosen.row[a][row];
                        if (kOp == kRowsUp && row >= 0) row = column;
                    }
                    uint4 b0 = make_uint4(0, 0, 0, 0), b1 = b0;
                    if (row >= 0) {
                        const T* const xr = static_cast<const T*>(p.x) + row * p.x_stride;
                        if (k0 < p.inner) b0 = *reinterpret_cast<const uint4*>(xr + k0);
                        if (k1 < p.inner) b1 = *reinterpret_cast<const uint4*>(xr + k1);
                    }
                    multiply<T>(acc[w], ring[d][0].x, ring[d][1].x, ring[d][0].y, ring[d][1].y, b0.x, b0.y);
                    multiply<T>(acc[w], ring[d][0].z, ring[d][1].z, ring[d][0].w, ring[d][1].w, b0.z, b0.w);
                    multiply<T>(acc[w], ring[d][2].x, ring[d][3].x, ring[d][2].y, ring[d][3].y, b1.x, b1.y);
                    multiply<T>(acc[w], ring[d][2].z, ring[d][3].z, ring[d][2].w, ring[d][3].w, b1.z, b1.w);
                }
            }
            fetch(ring[d]);
            if (now.step == steps - 1) {
                // the tile is through: the warps' sums come together
                if (kOp == kRowsDown) {
                    if (current >= 0) {
                        const float w0 = chosen.weight[current][2 * quad], w1 = chosen.weight[current][2 * quad + 1];
                        const bool b0 = chosen.row[current][2 * quad] >= 0, b1 = chosen.row[current][2 * quad + 1] >= 0;
                        if (b0) total_acc[0] += w0 * acc[0][0], total_acc[2] += w0 * acc[0][2];
                        if (b1) total_acc[1] += w1 * acc[0][1], total_acc[3] += w1 * acc[0][3];
                    }
                    current = -1;
                    sums[buffer][0][warp][lane] = make_float4(total_acc[0], total_acc[1], total_acc[2], total_acc[3]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) total_acc[j] = 0.0f;
                } else {
#pragma unroll
                    for (int w = 0; w < kWide; ++w) sums[buffer][w][warp][lane] = make_float4(acc[w][0], acc[w][1], acc[w][2], acc[w][3]);
                }
#pragma unroll
                for (int w = 0; w < kWide; ++w)
                    for (int j = 0; j < 4; ++j) acc[w][j] = 0.0f;
                __syncthreads();
                // Thread i: feature i % height of the tile and column i / height. Row r of a tile, column c, is value
                // 2 (r / 8) + c % 2 of lane 4 (r % 8) + c / 2.
                const float* const flat = reinterpret_cast<const float*>(sums[buffer]);
                const int r = tid % height, column = tid / height;
                if (r < now.size && column < p.tokens) {
                    const float* const at = flat + (column >> 3) * kRowsWarps * 128 + (4 * (r & 7) + ((column & 7) >> 1)) * 4 + (column & 1) + (r & 8 ? 2 : 0);
                    float v = 0.0f, up = 0.0f;
#pragma unroll
                    for (int w = 0; w < kRowsWarps; ++w) {
                        v += at[w * 128];
                        if (paired) up += at[w * 128 + 2];
                    }
                    const int a = kOp == kRowsUp ? now.at / p.features : 0;
                    const int f = kOp == kRowsUp ? now.at - a * p.features + r : now.at + r;
                    if (kOp == kRowsUp) {
                        // Rounded to the rows' type, since the next product takes 16-bit operands.
                        const int row = chosen.row[a][column];
                        if (row >= 0) static_cast<T*>(p.y)[(size_t)row * p.features + f] = Element<T>::from_float(silu(v) * up);
                    } else {
                        if (kOp == kRowsDense) {
                            if (p.bias != nullptr) {
                                v += load_any<T>(p.bias, f, p.bias_fp32);
                                if (paired) up += load_any<T>(p.bias, (size_t)p.features + f, p.bias_fp32);
                            }
                            v = paired ? silu(v) * up : activate(v, p.activation);
                        }
                        if (p.residual != nullptr) v += load_any<T>(p.residual, column * p.residual_stride + f, p.out_fp32);
                        store_any<T>(p.y, column * p.y_stride + f, v, p.out_fp32);
                    }
                }
                buffer ^= 1;
            }
            advance(now);
        }
    }
}

}  // namespace
