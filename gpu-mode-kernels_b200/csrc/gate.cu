// The gate of a mixture-of-experts layer: the k experts of every token and their weights, from the router's logits.
//
//     s_e = softmax(l)_e or 1 / (1 + exp(-l_e));  chosen: the k largest of l (without a bias: both scores grow with l) or of s + b, ties to
//     the lowest index;  w_i = scale * s_i, or scale * s_i / sum of the chosen s
//
// A warp takes a token, a lane every 32nd expert, and everything stays in registers: one pass over the logits. The next
// expert is found k times by the warp's reduction of unsigned keys that order as the values do; only the lane that gave
// an expert away looks for its next best. Nothing but latency counts: T tokens read T * E logits, 2 MB for 2048 of 256.
// With a bias the scores that decide are 64-bit: 256 sigmoids of a batch lie near enough to one another that roundings to 32
// bits would swap two experts every few hundred tokens.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "a2a.h"

namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;

struct GateParams {
    const void* logits;
    long long stride;
    const float* bias;
    int* indices;
    float* weights;
    int tokens, experts, topk, sigmoid, renormalize;
    float scale;
};

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }

// Unsigned keys in the order of the values, a NaN above all, 0 below all: the place of an expert that is gone or was never there.
__device__ __forceinline__ uint32_t key_of(float v) {
    if (v != v) return 0xffffffffu;
    const uint32_t u = __float_as_uint(v + 0.0f);  // -0 becomes 0: the two are equal
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long key_of(double v) {
    if (v != v) return ~0ull;
    const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ unsigned long long warp_max(unsigned long long v) {
    const uint32_t high = warp_max((uint32_t)(v >> 32));
    const uint32_t low = warp_max((uint32_t)(v >> 32) == high ? (uint32_t)v : 0u);
    return (unsigned long long)high << 32 | low;
}
template <typename V>
__device__ __forceinline__ V warp_sum(V v) {
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
__device__ __forceinline__ float exponential(float v) { return expf(v); }
__device__ __forceinline__ double exponential(double v) { return exp(v); }

// V: float, or double where a bias decides; kOwn: experts of a lane.
template <typename T, typename V, int kOwn>
__global__ void __launch_bounds__(kThreads) gate_kernel(const GateParams p) {
    using Key = decltype(key_of(V()));
    cudaGridDependencySynchronize();
    cudaTriggerProgrammaticLaunchCompletion();
    const int token = blockIdx.x * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (token >= p.tokens) return;
    const T* const row = static_cast<const T*>(p.logits) + token * p.stride;
    // (unrolled by number: left to itself the compiler keeps 64-bit scores in local memory, 8.0 us for 2048 tokens of 256 instead of 7.3)
    V score[kOwn];
    Key key[kOwn];
    float bias[sizeof(V) == 8 ? kOwn : 1];
#pragma unroll kOwn
    for (int j = 0; j < kOwn; ++j) {
        const int e = 32 * j + lane;
        score[j] = e < p.experts ? (V)as_float(row[e]) : (V)-INFINITY;
        key[j] = 0;
        if (sizeof(V) == 4 && e < p.experts) key[j] = key_of(score[j]);
        if constexpr (sizeof(V) == 8) bias[j] = e < p.experts ? p.bias[e] : 0.0f;
    }
    // a logit of -inf is behind all others whatever its bias and theirs, of -inf too: a bit an expert
    uint32_t excluded = 0;
    if constexpr (sizeof(V) == 8) {
#pragma unroll kOwn
        for (int j = 0; j < kOwn; ++j) excluded |= (uint32_t)(score[j] == (V)-INFINITY) << j;
    }
    V total = 1;
    if (p.sigmoid) {
#pragma unroll kOwn
        for (int j = 0; j < kOwn; ++j) score[j] = (V)1 / ((V)1 + exponential(-score[j]));
    } else {
        V most = score[0];
        bool nan = score[0] != score[0];
#pragma unroll kOwn
        for (int j = 1; j < kOwn; ++j) {
            most = score[j] > most ? score[j] : most;
            nan = nan || score[j] != score[j];
        }
        for (int d = 16; d > 0; d >>= 1) {
            const V other = __shfl_xor_sync(0xffffffffu, most, d);
            most = other > most ? other : most;
        }
        if (__any_sync(0xffffffffu, nan)) most = (V)NAN;
        V sum = 0;
#pragma unroll kOwn
        for (int j = 0; j < kOwn; ++j) {
            // a row of nothing but -inf has no scores: zeros
            score[j] = most == (V)-INFINITY ? (V)0 : exponential(score[j] - most);
            sum += score[j];
        }
        total = warp_sum(sum);
    }
    const V share = p.sigmoid || total == 0 ? (V)1 : (V)1 / total;
#pragma unroll kOwn
    for (int j = 0; j < kOwn; ++j) {
        score[j] *= share;
        const int e = 32 * j + lane;
        if constexpr (sizeof(V) == 8)
            if (e < p.experts) key[j] = excluded >> j & 1 ? (Key)1 : key_of(score[j] + (V)bias[j]);
    }

    // this lane's best, the lowest index among equals
    auto best_of = [&](Key& best, int& at, V& value) {
        best = key[0], at = 0, value = score[0];
#pragma unroll kOwn
        for (int j = 1; j < kOwn; ++j)
            if (key[j] > best) best = key[j], at = j, value = score[j];
    };
    Key best;
    int at;
    V value, sum = 0, mine = 0;
    int chosen = 0;
    best_of(best, at, value);
    for (int k = 0; k < p.topk; ++k) {
        const Key top = warp_max(best);
        const uint32_t e = __reduce_min_sync(0xffffffffu, best == top ? (uint32_t)(32 * at + lane) : 0xffffffffu);
        const V got = __shfl_sync(0xffffffffu, value, e & 31);
        sum += got;
        if (lane == k) chosen = (int)e, mine = got;
        if (lane == (e & 31)) {
#pragma unroll kOwn
            for (int j = 0; j < kOwn; ++j)
                if (j == (int)(e >> 5)) key[j] = 0;
            best_of(best, at, value);
        }
    }
    // The ratio of scores does not hang on how small they are: where the chosen ones come to less than 2^-64 they are looked at again, in 64 bits and
    // relative to the largest logit among them (1 / (1 + exp(-l)) is 0 in 32 bits from -89 on; next to a larger sum what is lost there weighs
    // less than 2^-62).
    if (p.renormalize && sum < (V)(1.0 / 18446744073709551616.0)) {
        const double l = lane < p.topk ? (double)as_float(row[chosen]) : -INFINITY;
        double most = l;
        for (int d = 16; d > 0; d >>= 1) {
            const double other = __shfl_xor_sync(0xffffffffu, most, d);
            most = other > most ? other : most;
        }
        // (chosen from a row of nothing but -inf: zeros)
        double r = most == -INFINITY ? 0.0 : exp(l - most);
        if (p.sigmoid) r /= 1.0 + exp(l);
        const double all = warp_sum(r);
        if (lane < p.topk) {
            p.indices[(size_t)token * p.topk + lane] = chosen;
            p.weights[(size_t)token * p.topk + lane] = (float)(all == 0.0 ? 0.0 : r / all * (double)p.scale);
        }
        return;
    }
    if (lane < p.topk) {
        V w = mine;
        if (p.renormalize) w = w / sum;
        p.indices[(size_t)token * p.topk + lane] = chosen;
        p.weights[(size_t)token * p.topk + lane] = (float)(w * (V)p.scale);
    }
}

template <typename T, typename V>
const void* gate_fn(int experts) {
    if (experts <= 64) return (const void*)gate_kernel<T, V, 2>;
    if (experts <= 128) return (const void*)gate_kernel<T, V, 4>;
    if (experts <= 256) return (const void*)gate_kernel<T, V, 8>;
    if (experts <= 512) return (const void*)gate_kernel<T, V, 16>;
    return (const void*)gate_kernel<T, V, 32>;
}

}  // namespace

extern "C" int a2a_gate(const a2a_gate_args* args, void* stream) {
    if (args == nullptr) return A2A_ERR_CONFIG;
    const a2a_gate_args& a = *args;
    if (a.dtype != A2A_DTYPE_BF16 && a.dtype != A2A_DTYPE_FP16 && a.dtype != A2A_DTYPE_FP32) return A2A_ERR_CONFIG;
    if (a.tokens < 0 || a.tokens > A2A_MAX_ROWS || a.experts < 1 || a.experts > A2A_MAX_EXPERTS || a.topk < 1 || a.topk > A2A_MAX_TOPK || a.topk > a.experts) return A2A_ERR_CONFIG;
    if (a.score != A2A_SCORE_SOFTMAX && a.score != A2A_SCORE_SIGMOID) return A2A_ERR_CONFIG;
    if (a.tokens == 0) return A2A_OK;
    if (a.logits == nullptr || a.indices == nullptr || a.weights == nullptr || a.stride < 0) return A2A_ERR_CONFIG;
    GateParams p{a.logits, (long long)a.stride, a.bias, a.indices, a.weights, a.tokens, a.experts, a.topk, a.score == A2A_SCORE_SIGMOID, a.renormalize != 0, a.scale};
    const bool wide = a.bias != nullptr;
    const void* fn;
    if (a.dtype == A2A_DTYPE_BF16) fn = wide ? gate_fn<__nv_bfloat16, double>(a.experts) : gate_fn<__nv_bfloat16, float>(a.experts);
    else if (a.dtype == A2A_DTYPE_FP16) fn = wide ? gate_fn<__half, double>(a.experts) : gate_fn<__half, float>(a.experts);
    else fn = wide ? gate_fn<float, double>(a.experts) : gate_fn<float, float>(a.experts);
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t launch{};
    launch.gridDim = dim3((a.tokens - 1) / kWarps + 1);
    launch.blockDim = dim3(kThreads);
    launch.stream = reinterpret_cast<cudaStream_t>(stream);
    launch.attrs = &attr;
    launch.numAttrs = 1;
    void* params[] = {&p};
    const cudaError_t e = cudaLaunchKernelExC(&launch, fn, params);
    return e == cudaSuccess ? A2A_OK : -(int)e;
}
