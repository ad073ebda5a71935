// What the kernels of the products share: element types, the epilogue's arithmetic, barriers with bounded waits, the
// tensor copies and the tensor core's instructions as inline PTX.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include "a2a.h"

namespace {

// A wait inside a kernel ends after this long whatever happens: every barrier here is completed by the same block (or its
// cluster), so one that is not is a fault of this code, and it is to end in an error instead of a GPU that does not answer. Cycles: two
// seconds at 2 GHz, from when the launch before is through. (Not the global timer: reading it takes so long that a ring whose every wait did took 0.4 us a step, ten times
// what the step moved.)
constexpr long long kWaitCycles = 4000000000ll;

// ---- element types -----------------------------------------------------------------------------
template <typename T>
struct Element;
template <>
struct Element<__nv_bfloat16> {
    static constexpr unsigned kFormat = 1;  // of the tensor core's instruction descriptor
    static __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Element<__half> {
    static constexpr unsigned kFormat = 0;
    static __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
};

// A value of `T` or of fp32, by a flag that is the same for a whole launch.
template <typename T>
__device__ __forceinline__ float load_any(const void* p, size_t i, bool fp32) {
    return fp32 ? static_cast<const float*>(p)[i] : Element<T>::to_float(static_cast<const T*>(p)[i]);
}
template <typename T>
__device__ __forceinline__ void store_any(void* p, size_t i, float v, bool fp32) {
    if (fp32)
        static_cast<float*>(p)[i] = v;
    else
        static_cast<T*>(p)[i] = Element<T>::from_float(v);
}

// Eight values from a place on 16 bytes, added to `v`; and to one.
template <typename T>
__device__ __forceinline__ void add_eight(float (&v)[8], const void* p, size_t i, bool fp32) {
    if (fp32) {
        const float4* const at = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
        const float4 a = at[0], b = at[1];
        v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w, v[4] += b.x, v[5] += b.y, v[6] += b.z, v[7] += b.w;
    } else {
        const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const T*>(p) + i);
        const T* const e = reinterpret_cast<const T*>(&q);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += Element<T>::to_float(e[j]);
    }
}
template <typename T>
__device__ __forceinline__ void put_eight(void* p, size_t i, const float (&v)[8], bool fp32) {
    if (fp32) {
        float4* const at = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
        at[0] = make_float4(v[0], v[1], v[2], v[3]);
        at[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        alignas(16) T e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = Element<T>::from_float(v[j]);
        *reinterpret_cast<uint4*>(static_cast<T*>(p) + i) = *reinterpret_cast<const uint4*>(e);
    }
}
// Lanes that differ in the three bits from kStep on, and their eight values, change places: value i of the lane whose bits are j was value j of the
// one whose bits are i.
template <int kStep>
__device__ __forceinline__ void exchange_eight(float (&v)[8], int lane) {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        const bool high = lane & kStep << k;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i >> k & 1) continue;
            const int j = i | 1 << k;
            const float got = __shfl_xor_sync(0xffffffffu, high ? v[i] : v[j], kStep << k);
            v[i] = high ? got : v[i];
            v[j] = high ? v[j] : got;
        }
    }
}

// The same for values that are rounded to 16 bits anyway: the second and third exchange are of two values at a time.
template <int kStep, typename T>
__device__ __forceinline__ uint4 exchange_packed(float (&v)[8], int lane) {
    const bool high = lane & kStep;
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float got = __shfl_xor_sync(0xffffffffu, high ? v[i] : v[i + 1], kStep);
        alignas(4) T two[2] = {Element<T>::from_float(high ? got : v[i]), Element<T>::from_float(high ? v[i + 1] : got)};
        q[i / 2] = *reinterpret_cast<const uint32_t*>(two);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const bool up = lane & 2 * kStep << k;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i >> k & 1) continue;
            const int j = i | 1 << k;
            const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? q[i] : q[j], 2 * kStep << k);
            q[i] = up ? got : q[i];
            q[j] = up ? q[j] : got;
        }
    }
    return make_uint4(q[0], q[1], q[2], q[3]);
}

// ---- the epilogue's arithmetic: fp32, on the fp32 sums of a product -------------------------------
// (The quick division gives 0 where the divisor is above 2^126: below -87, where silu is less than 1e-35.)
__device__ __forceinline__ float silu(float v) { return __fdividef(v, 1.0f + expf(-v)); }

// Over all values at once: the choice inside a loop over them was two thirds of the epilogue (16384 rows of 1024 to 2048: 92 us where this took
// 62).
template <int kCount>
__device__ __forceinline__ void activate(float (&v)[kCount], int activation) {
    if (activation == A2A_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < kCount; ++j) v[j] = v[j] < 0.0f ? 0.0f : v[j];  // passes a NaN on, as torch's does
    } else if (activation == A2A_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < kCount; ++j) v[j] = 0.5f * v[j] * (1.0f + erff(v[j] * 0.70710678118654752f));
    } else if (activation == A2A_ACT_SILU) {
#pragma unroll
        for (int j = 0; j < kCount; ++j) v[j] = silu(v[j]);
    }
}

// ---- barriers in shared memory, by their 32-bit addresses ----------------------------------------------
__device__ __forceinline__ uint32_t shared_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void barrier_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared_addr(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_init_done() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void barrier_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool barrier_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}

// The same barrier of the first block of this block's cluster.
__device__ __forceinline__ uint32_t of_first_block(uint32_t bar) {
    uint32_t there;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(there) : "r"(bar));
    return there;
}
// Says that sums have been read, and no more: a release would wait for all stores that this thread has on their way, 1.9 us with an SM full of them. Nothing
// but tensor memory is handed over, and its order needs none: each thread's loads are through (tcgen05.wait::ld) before its
// tcgen05.fence::before_thread_sync, after which the warp meets and one lane arrives; the products' thread has tcgen05.fence::after_thread_sync between its
// wait and the next product. These two fences order tensor memory across any flag, a relaxed one too.
__device__ __forceinline__ void barrier_arrive_there(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Waits for the phase of `parity`; false where the block has given up, or does now because the time has run out.
__device__ __noinline__ bool barrier_wait_long(uint32_t bar, uint32_t parity, volatile int* gave_up) {
    long long begin = 0;
    for (;;) {
        for (int i = 0; i < 16; ++i)
            if (barrier_try(bar, parity)) return true;
        if (*gave_up) return false;
        if (begin == 0) {
            // A call's later launch may be here before the one in front of it is through, whose rows nothing here goes on without: that takes as
            // long as it takes.
            cudaGridDependencySynchronize();
            begin = clock64();
        }
        if (clock64() - begin > kWaitCycles) {
            *gave_up = 1;
            return false;
        }
    }
}
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity, volatile int* gave_up) {
    return barrier_try(bar, parity) || barrier_wait_long(bar, parity, gave_up);
}

// True in one lane of the warp, the same one each time. Tensor copies and products are issued under this and not under a test of the lane's
// number: it tells the compiler that a single thread runs, and their operands go to uniform registers without a loop over lanes.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(one));
    return one != 0;
}

// ---- tensor copies, global -> this block's shared memory -------------------------------------------
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
// kPair: of a pair of blocks, whose products one of them issues; its barrier is told of both blocks' copies.
template <bool kPair>
__device__ __forceinline__ void copy_tile_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if constexpr (kPair)
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                     ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y)
                     : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                     ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y)
                     : "memory");
}
template <bool kPair>
__device__ __forceinline__ void copy_tile_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
    if constexpr (kPair)
        asm volatile(
            "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
            ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
            ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
            : "memory");
}

// ---- tensor core (tcgen05) -------------------------------------------------------------------------
// kPair: by the same warp of both blocks of a pair, and products of 256 rows, 128 of each block, issued by the first.
template <bool kPair>
__device__ __forceinline__ void tmem_alloc(uint32_t* where, uint32_t columns) {
    if constexpr (kPair) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_addr(where)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_addr(where)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
}
template <bool kPair>
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t columns) {
    if constexpr (kPair)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns));
    else
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns));
}
__device__ __forceinline__ void tcgen05_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tcgen05_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Arrives at the barrier, of both blocks of a pair, when the products so far are through.
template <bool kPair>
__device__ __forceinline__ void tcgen05_commit(uint32_t bar) {
    if constexpr (kPair)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(bar), "h"((uint16_t)3)
                     : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
template <bool kPair>
__device__ __forceinline__ void tcgen05_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t descriptor, bool add) {
    if constexpr (kPair)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(descriptor), "r"((uint32_t)add)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(descriptor), "r"((uint32_t)add)
            : "memory");
}
// 16 columns of this warp's 32 lanes: a lane's values of columns c to c + 15.
__device__ __forceinline__ void tmem_load_16(uint32_t tmem, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(tmem));
    // the values go through the wait, so that nothing reads them ahead of it
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                   "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// The same as matrix fragments: v[8 h + 4 c + 2 r + j] is of lane 16 h + 8 r + (own lane) / 4 and column 8 c + 2 (own lane % 4) + j.
__device__ __forceinline__ void tmem_load_fragments(uint32_t tmem, float (&v)[16]) {
    uint32_t r[16];
#pragma unroll
    for (int h = 0; h < 2; ++h)
        asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(r[8 * h]), "=r"(r[8 * h + 1]), "=r"(r[8 * h + 2]), "=r"(r[8 * h + 3]), "=r"(r[8 * h + 4]), "=r"(r[8 * h + 5]),
                       "=r"(r[8 * h + 6]), "=r"(r[8 * h + 7])
                     : "r"(tmem + ((uint32_t)(16 * h) << 16)));
    // the values go through the wait, so that nothing reads them ahead of it
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                   "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
// Two values in 16 bits each, the first one lower.
template <typename T>
__device__ __forceinline__ uint32_t packed(float low, float high) {
    alignas(4) const T two[2] = {Element<T>::from_float(low), Element<T>::from_float(high)};
    return *reinterpret_cast<const uint32_t*>(two);
}
// Four matrices of 8 by 8 fragments of 16 bits, turned over on their way into shared memory; lane i has the place of row i % 8 of matrix i / 8.
__device__ __forceinline__ void store_turned(uint32_t to, const uint32_t (&q)[4]) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared::cta.b16 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(q[0]), "r"(q[1]), "r"(q[2]), "r"(q[3])
                 : "memory");
}

// 16 columns that need not be neighbours: of() gives each one's, the same in all lanes.
template <typename Of>
__device__ __forceinline__ void tmem_load_spread(uint32_t tmem, Of of, float (&v)[16]) {
    uint32_t r[16];
#pragma unroll
    for (int i = 0; i < 16; ++i)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r[i]) : "r"(tmem + (uint32_t)of(i)));
    // the values go through the wait, so that nothing reads them ahead of it
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                   "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// A K-major operand in shared memory, rows of 128 bytes in the 128-byte swizzle: groups of eight rows are 1024 bytes apart.
__device__ __forceinline__ uint64_t operand_descriptor(uint32_t at) {
    return (uint64_t)((at & 0x3ffff) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}
// fp32 sums of products of `format` (Element::kFormat), `rows` rows by `columns`, both operands K-major.
__device__ __forceinline__ uint32_t instruction_descriptor(unsigned format, int rows, int columns) {
    return 1u << 4 | format << 7 | format << 10 | (uint32_t)(columns >> 3) << 17 | (uint32_t)(rows >> 4) << 24;
}

// All threads of the cluster's blocks meet; what one wrote to its shared memory before, the others see after.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
// Where block `rank` of the cluster has what `p` is here.
template <typename V>
__device__ __forceinline__ V* cluster_address(V* p, int rank) {
    V* there;
    asm volatile("mapa.u64 %0, %1, %2;" : "=l"(there) : "l"(p), "r"(rank));
    return there;
}

// Whether all of `threads` threads, which meet here, say yes.
__device__ __forceinline__ bool named_all(int id, int threads, bool yes) {
    uint32_t all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 q, %3, 0;\n\t"
        "barrier.cta.red.and.pred p, %1, %2, q;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(all)
        : "r"(id), "r"(threads), "r"((uint32_t)yes)
        : "memory");
    return all != 0;
}
__device__ __forceinline__ void named_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

}  // namespace
