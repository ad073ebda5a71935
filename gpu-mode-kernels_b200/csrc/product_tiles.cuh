// Products of weights with rows on the tensor cores (tcgen05): y[row] = W x[row], for one matrix and all rows (a dense product) or
// for a matrix per expert and the rows that chose it.
//
// The weights are the operand with 128 rows, the rows of x its columns: 16 to 256 of them, as many as there are. A decode batch leaves
// an expert a few rows; a tile of 128 rows of x would be filled to a few per cent, this one moves nothing but weights.
// Weights come through a ring in shared memory (tensor copies, 128-byte swizzle), 64 of the inner length at a time, the rows of x with them.
// Sums are fp32 in tensor memory, two buffers of 256 columns, so that one tile's epilogue runs beside the next one's products.
//
// Few rows leave the weights' bytes as the only cost, and then the SMs should have the same number of them: a tile has as many
// features as makes the number of tiles fill the SMs (`height`), up to what 128 rows hold, and over experts the tiles of a last round that
// fills no SMs are cut smaller. Operand rows behind a tile's features are whatever lies there; their sums are not read. A dense product with too few features for all SMs is cut along the inner length too, over the blocks
// of a cluster, which add up their sums in the order of their ranks through distributed shared memory.
//
// Where rows of x come from: dense, and in the first product of a layer of up to kSpreadTokens, a box of all rows; of such a layer an expert's
// rows are picked from the sums of all tokens. Everything else lies in runs (a layer of more tokens gets its rows sorted by expert first,
// by a launch of its own). A copy's issue costs more than its bytes: a run of 64 rows or more is boxes of 64, the last of which
// begins 64 before the end and writes some rows a second time, the same bytes to the same place; one of 32 or more is boxes of 32
// in the same way; a shorter one boxes of 8. (Rows gathered four at a time by the copy engine: 100 cycles and more each, 43 rows of 173
// made a step of 64 take 1230 cycles where the weights' bytes take 700.)
//
// The second product of a layer leaves a row a pair, in fp32, and a launch of its own adds a token's rows up: tickets, by which the tile that
// brings a token's last row adds them, took 3 us a tile (64 tokens of 2048, top-6 of 64: 146 us a layer where this took 129).
//
// Roles of the twelve warps: 0 weights, 1 products, 2 rows, 3 the lists of rows, 4 to 11 the epilogue, two for each 32 lanes of the tensor
// memory: every other 16 columns each.
//
// Pairs of blocks (kPair): a product of 256 columns by 128 rows takes 48 KB of operands for 512 cycles, more than the L2 gives an SM (2048
// rows of 7168, SwiGLU to 2048: 100 us). Two blocks of a cluster therefore take 256 rows between them, each with its half of the weights' rows
// and of the columns in shared memory, 32 KB; the first block issues the products of both, and its `full` barriers expect and hear of both blocks'
// copies. (With arrivals of the other block's producers there, a release at cluster scope a stage: 129 us.)
//
// SwiGLU: a tile's operand rows are gate and up of its features in turn (the tensor map's second dimension steps from gate to up), so that
// neighbouring lanes of the epilogue hold the two and exchange by shuffles.
#pragma once

#include "product_device.cuh"
#include "product_shares.h"

namespace {

// kDense32: with a result of 32 bits
enum TilesOp { kDense, kDense32, kLayerUp, kLayerDown, kSlabUp, kSlabDown };
// Blocks have tiles of their own; are pairs, which share tiles; or clusters, whose blocks have a part of a tile's inner length each. (A kernel for each:
// the instructions of a short one come from far away, and those of the others between them cost a small product 0.3 us.)
enum Together { kAlone, kPairs, kCuts };

constexpr int kTileRows = 128, kTileInner = 64, kMaxColumns = 256;
constexpr int kRowBytes = kTileInner * 2;
constexpr int kTilesThreads = 384, kFinishers = 256;  // of which the epilogue's
constexpr int kRingBytes = 192 * 1024, kMaxStages = 12;
// A stage has about as many blocks of 64 as reach this: small tiles do not pay a barrier for each, and two blocks of a row's 128 bytes come
// one right after the other, which the memory likes (experts on slabs of 7 rows: 221 us with 32 KB, 194 with 48, 207 with 64).
constexpr int kStageBytes = 48 * 1024;
constexpr int kMaxGroups = A2A_MAX_EXPERTS;
constexpr int kTmemColumns = 512;
constexpr int kSpreadTokens = 64;  // 40 to 100 tokens take the same either way
constexpr int kPieceRows = 32;  // operand rows of a box of a tile that is less than full
constexpr int kMaxSplit = 8;
constexpr int kTilesAhead = 64;
// The tensor core cuts the sums it adds to: a sum of 7168 products came out 8e-6 off, of the 2-norm, where torch's 32-bit products are 1e-7 (few rows) to
// 9e-7 off (600). For a result of 32 bits a sum in tensor memory therefore is of at most 512 of the inner length (4.5e-7 off), and the epilogue's
// threads add the parts up in registers, which hold 128 columns. (896 at once, 8.6e-7 off, took 6.25 us for 16 rows of 7168 to 256 where this takes 6.45.)
constexpr int kSumBlocks = 8, kMaxColumns32 = 128;
constexpr int kManyStep = 32;  // columns of a source in the slabs come in so many where there are many
constexpr int kCached = 4096;  // pairs whose experts a block keeps in shared memory

struct TilesParams {
    CUtensorMap weights;        // [groups][features][1 or gate, up][inner], boxes of `full` features by 64
    CUtensorMap weights_piece;  // the same in boxes of kPieceRows operand rows; not kDense
    CUtensorMap rows;           // boxes of 64 of the inner length by: kDense `columns` rows, kLayerUp not sorted all tokens, else 64 rows
    CUtensorMap rows_some, rows_few;  // 32 and 8 rows; of runs
    int inner;                  // length of a sum
    int features;               // of the output, per group
    int paired;                 // SwiGLU
    int groups;                 // matrices
    int full;                   // most features a tile may have; kDense: what it has
    int columns;                // most columns a tile may have
    int split;                  // kDense: blocks of a cluster, which share a tile's inner length
    int tokens;
    // kDense: the epilogue
    int activation, bias_fp32;
    int wide_stores;  // rows of y, and of the residual, begin on 16 bytes; of kSlabDown too
    const void* bias;
    const void* residual;
    long long residual_stride;
    void* y;
    long long y_stride;
    // kLayer*
    const int* indices;
    const float* weights_of;
    int topk;
    int sorted;    // kLayerUp: `rows` are the pairs' rows by expert, and a launch of the same call has put them there
    void* hidden;  // kLayerUp: [pair, by expert][features]; kSlabUp: [column, by expert][features]
    float* parts;  // [pair][features] of kLayerDown
    // kSlab*
    const int* counts;
    int world, capacity;
    int* error;  // mapped host memory: where a wait that ran out is recorded
};

__host__ __device__ __forceinline__ int parts_of(int n, int size) { return quotient(n + size - 1, size); }

template <int kNumber>
struct Lanes {
    static constexpr int value = kNumber;
};

// How `tiles` tiles of `height` features go over `blocks` blocks: whole rounds, and those of the last round in `cut` parts of `part` features.
struct Rounds {
    int whole, cut, part;
};
// least: a power of two
__host__ __device__ __forceinline__ Rounds rounds_of(int tiles, int blocks, int height, int least) {
    constexpr int step = 8;
    Rounds r;
    r.whole = quotient(tiles, blocks);
    const int rest = tiles - r.whole * blocks;
    r.cut = rest > 0 ? max(1, min(quotient(blocks, rest), height / least)) : 1;
    r.part = height;
    if (r.cut > 1) {
        r.part = (parts_of(height, r.cut) + step - 1) & -step;
        r.cut = parts_of(height, r.part);
    }
    return r;
}


struct Tile {
    int group, f, height, first, columns;  // matrix, first feature, features, first column, columns
};

struct TilesShared {
    uint64_t full[kMaxStages], empty[kMaxStages];
    uint64_t sums_full[2], sums_empty[2];
    uint64_t list_full[2], list_empty[2];
    uint32_t tmem;
    int gave_up;
    int largest;  // columns of the largest group
    int height, tiles;
    Rounds rounds;
    int begin[kMaxGroups + 1];  // tiles of one feature tile before a group's
    int count[kMaxGroups];      // columns of a group
    int row[kMaxGroups];        // columns before a group's
    int list[2][kMaxColumns];   // columns of a tile: pair (kLayer*) or row of the slabs, -1 for none
    float scale[2][kMaxColumns];
    int2 box[2][kMaxColumns / 8];  // kSlab*: boxes of 64, of 32 and of 8 rows: first row and column
    int boxes[2][3];               // where each kind ends
    Tile tile[kTilesAhead];        // the block's first ones
    int box_rows[2];               // rows of all boxes, of both blocks of a pair
    union {
        short expert[kCached];                                 // kLayer*: expert of a pair, -1 for none
        alignas(16) uint16_t turned[kFinishers / 32][16][32];  // others: columns by features of a warp of the epilogue, on their way out
    };
};
// An operand of less than 128 rows at the end of the ring is read beyond it.
static_assert(sizeof(TilesShared) >= kTileRows * kRowBytes, "operands of 128 rows end within the shared memory");

constexpr size_t kTilesSharedBytes = 1024 + kRingBytes + sizeof(TilesShared);
static_assert(kTilesSharedBytes <= 227 * 1024, "a block's shared memory");

// The epilogue's 16 columns from 16 * half on, in steps of 32, with the registers that hold them (kParts: one for results of 16 bits).
template <int kParts, typename Do>
__device__ __forceinline__ void for_parts(int columns, int half, float (&total)[kParts][16], Do work) {
    if constexpr (kParts > 1) {
#pragma unroll
        for (int g = 0; g < kParts; ++g)
            if (16 * half + 32 * g < columns) work(16 * half + 32 * g, total[g]);
    } else {
        for (int c0 = 16 * half; c0 < columns; c0 += 32) work(c0, total[0]);
    }
}
template <int kParts>
__device__ __forceinline__ void add_part(uint32_t sums, bool needed, int columns, int half, float (&total)[kParts][16]) {
    if (!needed) return;
    for_parts(columns, half, total, [&](int c0, float (&sum)[16]) {
        float v[16];
        tmem_load_16(sums + c0, v);
#pragma unroll
        for (int j = 0; j < 16; ++j) sum[j] += v[j];
    });
}



__host__ __device__ __forceinline__ int round16(int n) { return (n + 15) & ~15; }
// What a block of 64 of a tile takes, in ns: the SM's share of the memory's rate for the weights (6.5 TB/s over 148), what the L2 gives an SM
// (90 bytes a ns; `held` of the columns are this block's to copy), or the products (256 columns by 64 in 512 cycles).
__host__ __device__ __forceinline__ float block_ns(int rows, int columns, int held, float memory_share) {
    const float memory = rows * kRowBytes * memory_share, cache = (rows + held) * kRowBytes * (1.0f / 90), products = columns * 1.05f;
    // below 110 ns the threads that issue copies and products do not keep up
    return fmaxf(fmaxf(fmaxf(memory, cache), products), 110.0f) + 10.0f;
}

template <TilesOp kOp, typename T, Together kTogether>
__global__ void __launch_bounds__(kTilesThreads, 1) product_tiles_kernel(const __grid_constant__ TilesParams p) {
    constexpr bool kPair = kTogether == kPairs, kCut = kTogether == kCuts;
    constexpr bool k32 = kOp == kDense32, kOne = kOp == kDense || k32, kGrouped = !kOne, kLayer = kOp == kLayerUp || kOp == kLayerDown, kSlab = kOp == kSlabUp || kOp == kSlabDown;
    constexpr bool kUp = kOp == kLayerUp || kOp == kSlabUp;
    const bool first = kOne || (kOp == kLayerUp && !p.sorted) || kOp == kSlabUp;  // nothing of the same call runs before it
    const bool runs = kGrouped && (!kUp || (kOp == kLayerUp && p.sorted));              // rows by expert
    extern __shared__ uint8_t shared_raw[];
    uint8_t* const ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(shared_raw) + 1023) & ~(uintptr_t)1023);
    TilesShared& s = *reinterpret_cast<TilesShared*>(ring + kRingBytes);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool paired = kUp || (kOne && p.paired);
    constexpr int kBlocks = kPair ? 2 : 1, kColumnStep = 16 * kBlocks;
    const int side = kPair ? (int)blockIdx.x & 1 : 0, units = (int)gridDim.x / kBlocks;  // block of the pair; blocks or pairs

    if (tid == 0) {
        for (int i = 0; i < kMaxStages; ++i) {
            barrier_init(&s.full[i], 2);
            barrier_init(&s.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            barrier_init(&s.sums_full[i], 1);
            barrier_init(&s.sums_empty[i], kFinishers / 32 * kBlocks);
            barrier_init(&s.list_full[i], 1);
            barrier_init(&s.list_empty[i], kOp == kSlabUp ? 2 : 1);  // the roles that read it
        }
        s.gave_up = s.largest = 0;
        barrier_init_done();
    }
    if (warp == 1) tmem_alloc<kPair>(&s.tmem, kTmemColumns);
    if (warp == 2 && lane < (!kGrouped ? 2 : kOp == kLayerUp && !p.sorted ? 3 : 4))
        prefetch_map(lane == 0 ? &p.weights : lane == 1 ? &p.rows : lane == 2 ? &p.weights_piece : &p.rows_few);
    if (kLayer)
#pragma unroll 1
        for (int g = tid; g < p.groups; g += kTilesThreads) s.count[g] = 0;
    // A call's later launches read weights, indices and counts ahead of this: what wrote those was through before the call's first launch let
    // the second one begin.
    if (first) {
        cudaGridDependencySynchronize();
        cudaTriggerProgrammaticLaunchCompletion();
    }

    // kSlab*: rows that source `src` has for group g, and the columns of a group, with those of every source rounded up to whole steps
    auto slab_rows = [&](int g, int src) { return min(max(p.counts[(size_t)src * 4 * p.groups + g], 0), p.capacity); };
    auto slab_columns = [&](int g, int step) {
        int n = 0;
#pragma unroll
        for (int src = 0; src < A2A_MAX_WORLD; ++src)
            if (src < p.world) n += (slab_rows(g, src) + step - 1) & -step;
        return n;
    };

    // ---- how many columns every group has, and so the tiles ----
    int columns = p.columns, height = p.full, slab_step = 8;
    if (kLayer) {
        const int pairs = p.tokens * p.topk;
        int next = tid < pairs ? p.indices[tid] : -1;  // on its way while the threads meet
        __syncthreads();
#pragma unroll 1
        for (int i = tid; i < pairs; i += kTilesThreads) {
            const int e = next < 0 || next >= p.groups ? -1 : next;
            if (i + kTilesThreads < pairs) next = p.indices[i + kTilesThreads];
            if (i < kCached) s.expert[i] = (short)e;
            if (e >= 0) atomicAdd(&s.count[e], 1);
        }
        __syncthreads();
    }
    if (kSlab) {
        int most = 0;
#pragma unroll 1
        for (int g = tid; g < p.groups; g += kTilesThreads) most = max(most, s.count[g] = slab_columns(g, 8));
        most = __reduce_max_sync(0xffffffffu, most);
        __syncthreads();  // `largest` is 0
        if (lane == 0) atomicMax(&s.largest, most);
        __syncthreads();
        if (s.largest > kMaxColumns) {
            // more than a tile of columns: columns without a row cost less than boxes of eight
            slab_step = kManyStep;
#pragma unroll 1
            for (int g = tid; g < p.groups; g += kTilesThreads) s.count[g] = slab_columns(g, slab_step);
            __syncthreads();
        }
    }
    auto widest = [&](int largest) { return min(p.columns, (max(largest, 1) + kColumnStep - 1) / kColumnStep * kColumnStep); };
    if (kGrouped) {
        if (warp == 0) {
            // a lane has neighbouring groups, whose sums the warp adds up once
            const int each = (p.groups + 31) >> 5, g0 = lane * each, g1 = min(g0 + each, p.groups);
            int largest = s.largest;
            if (kLayer) {
#pragma unroll 1
                for (int g = g0; g < g1; ++g) largest = max(largest, s.count[g]);
                largest = __reduce_max_sync(0xffffffffu, largest);
                if (lane == 0) s.largest = largest;
            }
            columns = widest(largest);
            int own = 0, own_rows = 0;
#pragma unroll 1
            for (int g = g0; g < g1; ++g) own += parts_of(s.count[g], columns), own_rows += s.count[g];
            int sum = own, sum_rows = own_rows;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int left = __shfl_up_sync(0xffffffffu, sum, d), left_rows = __shfl_up_sync(0xffffffffu, sum_rows, d);
                if (lane >= d) sum += left, sum_rows += left_rows;
            }
            const int run = __shfl_sync(0xffffffffu, sum, 31);
            sum -= own, sum_rows -= own_rows;
#pragma unroll 1
            for (int g = g0; g < g1; ++g) {
                s.begin[g] = sum, s.row[g] = sum_rows;
                sum += parts_of(s.count[g], columns), sum_rows += s.count[g];
            }
            // the height whose tiles take the fullest SM least: a whole box, or a lane a multiple of 8 from a piece on
            const int piece = kPieceRows / (kUp ? 2 : 1), h = lane == 31 ? p.full : 8 * (lane + 1);
            unsigned cost = 0xffffffffu;
            int tiles = 0;
            Rounds r{};
            if ((h >= piece && h < p.full) || lane == 31) {
                const int wide = kOp == kLayerUp && !p.sorted ? round16(p.tokens) : columns;
                tiles = run * parts_of(p.features, kBlocks * h);
                r = rounds_of(tiles, units, h, piece);
                // (pieces have to be issued: 30 ns)
                float ns = r.whole * (block_ns(h * (kUp ? 2 : 1), wide, wide / kBlocks, 1.0f / 44) + (h < p.full ? 30.0f : 0.0f));
                if (r.whole * units < tiles) ns += block_ns(r.part * (kUp ? 2 : 1), wide, wide / kBlocks, 1.0f / 44) + (r.part < p.full ? 30.0f : 0.0f);
                cost = (unsigned)fminf(ns * 8.0f, 1e9f);
            }
            const unsigned least = __reduce_min_sync(0xffffffffu, cost);
            const int best = 31 - __clz(__ballot_sync(0xffffffffu, cost == least));  // the highest of the best
            if (lane == best) s.begin[p.groups] = run, s.height = h, s.tiles = tiles, s.rounds = r;
        }
    }
    tcgen05_before_sync();
    __syncthreads();
    if (kPair) cluster_sync();  // the other block's barriers are there
    tcgen05_after_sync();
    if (kGrouped) height = s.height, columns = widest(s.largest);
    const uint32_t tmem = s.tmem;
    const uint32_t full0 = shared_addr(s.full), empty0 = shared_addr(s.empty), sums_full0 = shared_addr(s.sums_full), sums_empty0 = shared_addr(s.sums_empty),
                   list_full0 = shared_addr(s.list_full), list_empty0 = shared_addr(s.list_empty), ring0 = shared_addr(ring);
    const int feature_tiles = parts_of(p.features, kBlocks * height);
    const int full_tiles = kGrouped ? s.tiles : parts_of(p.tokens, columns) * feature_tiles;
    // over experts: the tiles that come in whole rounds, and the others in parts
    const int piece = kPieceRows / (paired ? 2 : 1);
    const Rounds rounds = kGrouped ? s.rounds : Rounds{0, 1, height};
    const int whole_tiles = kGrouped ? rounds.whole * units : 0;
    const int tiles = whole_tiles + (full_tiles - whole_tiles) * rounds.cut;
    // the operand's columns in a stage, of this block
    const int wide = kOp == kLayerUp && !p.sorted ? round16(p.tokens) : columns / kBlocks;
    const int highest = whole_tiles > 0 ? height : rounds.part;
    const int weight_bytes = ((paired ? 2 : 1) * max(highest, kGrouped ? piece : 0) * kRowBytes + 1023) & ~1023, block_bytes = weight_bytes + wide * kRowBytes;
    const int blocks_all = parts_of(p.inner, kTileInner);
    const int per_stage = stage_blocks(blocks_all, block_bytes, kStageBytes, k32 ? kSumBlocks : blocks_all);
    const int stages = min(kMaxStages, quotient(kRingBytes, block_bytes * per_stage));
    // this block's part of the inner length, and its tiles
    const int split = kCut ? p.split : 1, part = kCut ? (int)blockIdx.x % split : 0;
    const int block0 = blocks_all * part / split, blocks = blocks_all * (part + 1) / split - block0;
    const int tile0 = (int)blockIdx.x / (kBlocks * split), tile_step = units / split;

    // Tiles that share weights come one after the other, so that blocks read them together.
    auto tile_of = [&](int t) {
        Tile x;
        int count, cut = 0;
        x.height = height;
        if (t >= whole_tiles && rounds.cut > 1) {
            const int q = quotient(t - whole_tiles, rounds.cut);
            cut = (t - whole_tiles - q * rounds.cut) * rounds.part;
            t = whole_tiles + q;
            x.height = min(rounds.part, height - cut);
        }
        if (kGrouped) {
            const int q = quotient(t, feature_tiles);
            int lo = 0, hi = p.groups - 1;  // the last group that begins at or before q; groups without rows begin with the next
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (s.begin[mid] <= q) lo = mid;
                else hi = mid - 1;
            }
            x.group = lo;
            count = s.count[lo];
            t -= s.begin[lo] * feature_tiles;
        } else {
            x.group = 0;
            count = p.tokens;
        }
        const int across = parts_of(count, columns);
        const int m = quotient(t, across);
        x.f = kBlocks * (m * height + cut) + side * x.height;  // this block's
        x.first = (t - m * across) * columns;
        x.columns = min(columns, count - x.first);
        return x;
    };
    // Over experts the roles find their tiles in a table, the first ones at least: working one out takes 900 cycles, in which the ring empties.
    if (kGrouped) {
        if (tid < kTilesAhead && tile0 + tid * tile_step < tiles) s.tile[tid] = tile_of(tile0 + tid * tile_step);
        __syncthreads();
    }
    auto tile_at = [&](int n) { return kGrouped && n < kTilesAhead ? s.tile[n] : tile_of(tile0 + n * tile_step); };
    // columns of a tile's product, and of those the ones that block `of` copies, in eights
    auto product_columns = [&](const Tile& x) {
        if (kOne && kPair) return columns;
        return ((kOp == kLayerUp && !p.sorted ? p.tokens : x.columns) + kColumnStep - 1) / kColumnStep * kColumnStep;
    };
    auto columns_of = [&](const Tile& x, int of, int& from) { return copied_columns(x.columns, product_columns(x), kBlocks, of, &from); };
    // kLayer*: a pair's expert, -1 for none
    auto expert_of = [&](int pair) {
        if (pair < kCached) return (int)s.expert[pair];
        const int e = p.indices[pair];
        return e >= 0 && e < p.groups ? e : -1;
    };
    const bool spread = kOp == kLayerUp && !p.sorted;  // all tokens are a tile's columns
    const uint32_t stage_bytes = (uint32_t)per_stage * block_bytes;
    const int sum_of = sum_blocks(per_stage, kSumBlocks);  // kDense32
    if (warp == 0) {
        if (elect_one()) {
            int stage = 0;
            uint32_t phase = 1;
            for (int t = tile0, i = 0; t < tiles; t += tile_step, ++i) {
                const Tile x = tile_at(i);
                const int f = x.f, h1 = x.height;
                const bool whole = !kGrouped || h1 == p.full;  // a box of all features, or pieces
                const int bytes = whole ? (paired ? 2 : 1) * h1 * kRowBytes : parts_of(h1, piece) * kPieceRows * kRowBytes;
                int k = block0 * kTileInner;
                for (int left = blocks; left > 0; left -= per_stage) {
                    const uint32_t bar = kPair ? of_first_block(full0 + 8 * stage) : full0 + 8 * stage;
                    uint32_t at = ring0 + stage * stage_bytes;
                    if (!barrier_wait(empty0 + 8 * stage, phase, &s.gave_up)) goto weights_done;
                    int n = min(per_stage, left);
                    if (side == 0) barrier_expect(full0 + 8 * stage, n * bytes * kBlocks);
                    for (; n > 0; --n, k += kTileInner, at += block_bytes) {
                        if (whole) {
                            copy_tile_4d<kPair>(at, &p.weights, k, 0, f, x.group, bar);
                        } else {
                            for (int h0 = 0; h0 < h1; h0 += piece) {
                                const int h = max(0, min(h0, h1 - piece));  // the last one overlaps: the same bytes to the same place
                                copy_tile_4d<kPair>(at + h * (paired ? 2 : 1) * kRowBytes, &p.weights_piece, k, 0, f + h, x.group, bar);
                            }
                        }
                    }
                    if (++stage == stages) stage = 0, phase ^= 1;
                }
            }
        weights_done:;
        }
    } else if (warp == 1) {
        if (side == 0 && elect_one()) {
            int stage = 0, n = 0;
            uint32_t phase = 0;
            const uint64_t ring_descriptor = operand_descriptor(ring0);
            for (int t = tile0, i = 0; t < tiles; t += tile_step, ++i) {
                const Tile x = tile_at(i);
                const uint32_t descriptor = instruction_descriptor(Element<T>::kFormat, kTileRows * kBlocks, product_columns(x));
                for (int chunk = blocks; chunk > 0; ++n) {
                    // a sum in tensor memory: the whole inner length, or for a result of 32 bits a part of it
                    const int buffer = n & 1;
                    const uint32_t sums = tmem + buffer * kMaxColumns;
                    if (!barrier_wait(sums_empty0 + 8 * buffer, ((n >> 1) & 1) ^ 1, &s.gave_up)) goto products_done;
                    tcgen05_after_sync();
                    bool add = false;
                    const int end = k32 ? max(0, chunk - sum_of) : 0;
                    for (int left = chunk; left > end; left -= per_stage) {
                        uint64_t w = ring_descriptor + (stage * stage_bytes >> 4);
                        if (!barrier_wait(full0 + 8 * stage, phase, &s.gave_up)) goto products_done;
                        for (int b = min(per_stage, left); b > 0; --b, w += block_bytes >> 4) {
                            const uint64_t r = w + (weight_bytes >> 4);
                            // 16 of the inner length are 32 bytes of a row
                            tcgen05_mma<kPair>(sums, w, r, descriptor, add);
                            tcgen05_mma<kPair>(sums, w + 2, r + 2, descriptor, true);
                            tcgen05_mma<kPair>(sums, w + 4, r + 4, descriptor, true);
                            tcgen05_mma<kPair>(sums, w + 6, r + 6, descriptor, true);
                            add = true;
                        }
                        tcgen05_commit<kPair>(empty0 + 8 * stage);
                        if (++stage == stages) stage = 0, phase ^= 1;
                    }
                    tcgen05_commit<kPair>(sums_full0 + 8 * buffer);
                    chunk = end;
                }
            }
        products_done:;
        }
    } else if (warp == 2) {
        if (!first) cudaGridDependencySynchronize();
        if (elect_one()) {
            int stage = 0, n = 0;
            uint32_t phase = 1;
            for (int t = tile0, i = 0; t < tiles; t += tile_step, ++n, ++i) {
                const Tile x = tile_at(i);
                // the tile's copies of a block of 64: one box, or the boxes of a run, or of the runs of the slabs
                int bytes = wide * kRowBytes * kBlocks, wide_boxes = 0, some_boxes = 0, boxes = 0, run = 0, from = 0;  // bytes: of both blocks
                if (kOne) columns_of(x, side, from);
                if (runs) {
                    bytes = 0;
                    for (int of = 0; of < kBlocks; ++of) bytes += boxed_rows(columns_of(x, of, from)) * kRowBytes;
                    run = columns_of(x, side, from);
                } else if (kOp == kSlabUp) {
                    if (!barrier_wait(list_full0 + 8 * (n & 1), (n >> 1) & 1, &s.gave_up)) goto rows_done;
                    wide_boxes = s.boxes[n & 1][0], some_boxes = s.boxes[n & 1][1], boxes = s.boxes[n & 1][2];
                    bytes = s.box_rows[n & 1] * kRowBytes;
                }
                int k = block0 * kTileInner;
                for (int left = blocks; left > 0; left -= per_stage) {
                    const uint32_t bar = kPair ? of_first_block(full0 + 8 * stage) : full0 + 8 * stage;
                    uint32_t at = ring0 + stage * stage_bytes + weight_bytes;
                    if (!barrier_wait(empty0 + 8 * stage, phase, &s.gave_up)) goto rows_done;
                    int have = min(per_stage, left);
                    if (side == 0) barrier_expect(full0 + 8 * stage, have * bytes);
                    for (; have > 0; --have, k += kTileInner, at += block_bytes) {
                        if (kOne || spread) {
                            copy_tile_2d<kPair>(at, &p.rows, k, kOne ? x.first + from : 0, bar);
                        } else if (runs) {
                            const int row = s.row[x.group] + x.first + from;
                            if (run >= 64) {
                                for (int c = 0; c < run; c += 64) copy_tile_2d<kPair>(at + min(c, run - 64) * kRowBytes, &p.rows, k, row + min(c, run - 64), bar);
                            } else if (run >= 32) {
                                for (int c = 0; c < run; c += 32) copy_tile_2d<kPair>(at + min(c, run - 32) * kRowBytes, &p.rows_some, k, row + min(c, run - 32), bar);
                            } else {
                                for (int c = 0; c < run; c += 8) copy_tile_2d<kPair>(at + c * kRowBytes, &p.rows_few, k, row + c, bar);
                            }
                        } else {
                            const int2* const list = s.box[n & 1];
                            int j = 0;
                            for (; j < wide_boxes; ++j) copy_tile_2d<kPair>(at + list[j].y * kRowBytes, &p.rows, k, list[j].x, bar);
                            for (; j < some_boxes; ++j) copy_tile_2d<kPair>(at + list[j].y * kRowBytes, &p.rows_some, k, list[j].x, bar);
                            for (; j < boxes; ++j) copy_tile_2d<kPair>(at + list[j].y * kRowBytes, &p.rows_few, k, list[j].x, bar);
                        }
                    }
                    if (++stage == stages) stage = 0, phase ^= 1;
                }
                if (kOp == kSlabUp) barrier_arrive(list_empty0 + 8 * (n & 1));
            }
        rows_done:;
        }
    } else if (warp == 3) {
        if (kGrouped) {
            int n = 0;
            for (int t = tile0, i = 0; t < tiles; t += tile_step, ++n, ++i) {
                const Tile x = tile_at(i);
                const int buffer = n & 1;
                if (!__all_sync(0xffffffffu, barrier_wait(list_empty0 + 8 * buffer, ((n >> 1) & 1) ^ 1, &s.gave_up))) break;
                if (kLayer) {
                    // pairs in ascending order: which tile of a group a pair belongs to is the same for every block
                    const int pairs = p.tokens * p.topk;
                    int seen = 0;
                    for (int i0 = 0; i0 < pairs && seen < x.first + x.columns; i0 += 128) {
                        int e[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int i = i0 + 32 * j + lane;
                            e[j] = i < pairs ? expert_of(i) : -1;
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const unsigned mine = __ballot_sync(0xffffffffu, e[j] == x.group);
                            const int at = seen + __popc(mine & ((1u << lane) - 1)) - x.first;
                            if (e[j] == x.group && at >= 0 && at < x.columns) {
                                const int pair = i0 + 32 * j + lane;
                                s.list[buffer][at] = pair;
                            }
                            seen += __popc(mine);
                        }
                    }
                    if (kOp == kLayerDown) {
                        __syncwarp();
                        for (int c = lane; c < x.columns; c += 32) s.scale[buffer][c] = p.weights_of[s.list[buffer][c]];
                    }
                } else {
                    // The row of the slabs that stands at a column, and whether it is a valid one. The sources' counts are read once for all
                    // columns (one after the other for each column they took longer than a tile's products).
                    int have[A2A_MAX_WORLD];
#pragma unroll
                    for (int src = 0; src < A2A_MAX_WORLD; ++src) have[src] = src < p.world ? slab_rows(x.group, src) : 0;
                    auto row_at = [&](int c, bool& valid) {
                        int r = x.first + c, src = 0, rows = 0;
#pragma unroll
                        for (int i = 0, begin = 0; i < A2A_MAX_WORLD; ++i) {
                            if (i < p.world && x.first + c >= begin) src = i, r = x.first + c - begin, rows = have[i];
                            begin += (have[i] + slab_step - 1) & -slab_step;
                        }
                        valid = r < rows;
                        return (x.group * p.world + src) * p.capacity + r;
                    };
                    bool valid;
                    for (int c = lane; c < x.columns; c += 32) {
                        const int row = row_at(c, valid);
                        s.list[buffer][c] = valid ? row : -1;
                    }
                    // Lane i looks at columns 8 i to 8 i + 7: where their run begins and ends, and whether a box begins there. (The columns that a second
                    // block copies for nothing are of rows of any kind, or behind the last one, which come as zeros.)
                    int box_rows = 0;
                    for (int of = 0; of < kBlocks; ++of) {
                        int from;
                        const int eights = columns_of(x, of, from) >> 3, row = lane < eights ? row_at(from + 8 * lane, valid) : -1;
                        const int before = __shfl_up_sync(0xffffffffu, row, 1);
                        const unsigned breaks = __ballot_sync(0xffffffffu, lane == 0 || lane >= eights || row != before + 8);
                        const int run0 = 31 - __clz(breaks & (0xffffffffu >> (31 - lane)));
                        const unsigned later = lane == 31 ? 0 : breaks >> (lane + 1);
                        const int run1 = later ? lane + __ffs(later) : 32;
                        const int run = run1 - run0, place = lane - run0, size = run >= 8 ? 8 : run >= 4 ? 4 : 1;
                        const bool begins = lane < eights && ((place % size == 0 && place + size <= run) || place == run - size);
                        int boxes = 0;
#pragma unroll
                        for (int kind = 0; kind < 3; ++kind) {
                            const int rows = kind == 0 ? 8 : kind == 1 ? 4 : 1;
                            const bool mine = begins && size == rows;
                            const unsigned all = __ballot_sync(0xffffffffu, mine);
                            if (of == side && mine) s.box[buffer][boxes + __popc(all & ((1u << lane) - 1))] = make_int2(row, 8 * lane);
                            boxes += __popc(all);
                            box_rows += 8 * rows * __popc(all);
                            if (of == side && lane == 0) s.boxes[buffer][kind] = boxes;
                        }
                    }
                    if (lane == 0) s.box_rows[buffer] = box_rows;
                }
                __syncwarp();
                if (lane == 0) barrier_arrive(list_full0 + 8 * buffer);
            }
        }
    } else {
        const int quarter = warp & 3, half = (warp - 4) >> 2, at = tid - 128;
        if (!first) {
            cudaGridDependencySynchronize();
            cudaTriggerProgrammaticLaunchCompletion();
        }
        int n = 0;
        bool met = !kCut;
        auto sums_read = [&](int buffer) {
            tcgen05_before_sync();
            __syncwarp();
            if (lane == 0) kPair ? barrier_arrive_there(of_first_block(sums_empty0 + 8 * buffer)) : barrier_arrive(sums_empty0 + 8 * buffer);
        };
        for (int t = tile0, i = 0; t < tiles; t += tile_step, ++n, ++i) {
            const Tile x = tile_at(i);
            const bool needed = (paired ? quarter * 16 : quarter * 32) < x.height;  // by warp
            // kDense32: the tile's sum, of those of its parts
            float total[k32 ? kMaxColumns32 / 32 : 1][16];
            if constexpr (k32) {
#pragma unroll
                for (int g = 0; g < kMaxColumns32 / 32; ++g)
#pragma unroll
                    for (int j = 0; j < 16; ++j) total[g][j] = 0.0f;
                bool all = true;
                for (int chunk = blocks; chunk > sum_of && all; chunk -= sum_of, ++n) {
                    all = named_all(1, kFinishers, barrier_wait(sums_full0 + 8 * (n & 1), (n >> 1) & 1, &s.gave_up));
                    if (!all) break;
                    tcgen05_after_sync();
                    add_part(tmem + (n & 1) * kMaxColumns + ((uint32_t)(quarter * 32) << 16), needed, x.columns, half, total);
                    sums_read(n & 1);
                }
                if (!all) break;
            }
            const int buffer = n & 1;
            bool here = !kGrouped || barrier_wait(list_full0 + 8 * buffer, (n >> 1) & 1, &s.gave_up);
            here = here && barrier_wait(sums_full0 + 8 * buffer, (n >> 1) & 1, &s.gave_up);
            if (!named_all(1, kFinishers, here)) break;  // all warps go on, or none
            tcgen05_after_sync();
            const uint32_t sums = tmem + buffer * kMaxColumns + ((uint32_t)(quarter * 32) << 16);
            if constexpr (k32) {
                add_part(sums, needed, x.columns, half, total);
                sums_read(buffer);
            }
            // this lane's feature
            const int own = quarter * 32 + lane, within = paired ? own >> 1 : own, f = x.f + within;
            const bool inside = within < x.height && f < p.features, up = paired && (lane & 1);
            float bias = 0.0f;
            if (kOne && p.bias != nullptr && inside)
                bias = load_any<T>(p.bias, (size_t)(up ? p.features : 0) + f, p.bias_fp32);
            // Finishes columns c0 to c0 + kCount - 1 (an even number). With SwiGLU lanes 2 i and 2 i + 1 hold gate and up of a feature: the
            // first finishes the even columns, the second the odd ones. Values first, then the stores, so that the columns overlap.
            auto finish = [&](int c0, auto& v) {
                constexpr int kCount = sizeof(v) / sizeof(float);
                if (paired) {
                    float out[kCount / 2], add[kCount / 2];
#pragma unroll
                    for (int j = 0; j < kCount / 2; ++j) {
                        const int c = c0 + 2 * j + up;
                        add[j] = 0.0f;
                        if (p.residual != nullptr && inside && c < x.columns)
                            add[j] = load_any<T>(p.residual, (size_t)(x.first + c) * p.residual_stride + f, k32);
                    }
#pragma unroll
                    for (int j = 0; j < kCount / 2; ++j) {
                        const float even = v[2 * j] + bias, odd = v[2 * j + 1] + bias;
                        const float other = __shfl_xor_sync(0xffffffffu, up ? even : odd, 1);
                        out[j] = silu(up ? other : even) * (up ? odd : other) + add[j];
                    }
                    if (!inside) return;
#pragma unroll
                    for (int j = 0; j < kCount / 2; ++j) {
                        const int c = c0 + 2 * j + up;
                        if (c >= x.columns) continue;
                        store_any<T>(p.y, (size_t)(x.first + c) * p.y_stride + f, out[j], k32);
                    }
                    return;
                }
                if (!inside) return;
                if (kOne) {
                    float add[kCount], out[kCount];
#pragma unroll
                    for (int j = 0; j < kCount; ++j) {
                        add[j] = 0.0f;
                        if (p.residual != nullptr && c0 + j < x.columns)
                            add[j] = load_any<T>(p.residual, (size_t)(x.first + c0 + j) * p.residual_stride + f, k32);
                        out[j] = v[j] + bias;
                    }
                    activate(out, p.activation);
#pragma unroll
                    for (int j = 0; j < kCount; ++j)
                        if (c0 + j < x.columns) store_any<T>(p.y, (size_t)(x.first + c0 + j) * p.y_stride + f, out[j] + add[j], k32);
                } else {
#pragma unroll
                    for (int j = 0; j < kCount; ++j) {
                        const int c = c0 + j;
                        if (c >= x.columns) break;
                        const int row = s.list[buffer][c];
                        if (kOp == kLayerDown) p.parts[(size_t)row * p.features + f] = s.scale[buffer][c] * v[j];
                        else if (row >= 0) static_cast<T*>(p.y)[(size_t)row * p.features + f] = Element<T>::from_float(v[j]);
                    }
                }
            };
            // The same for whole 16 columns and features in eights, with 16-byte stores: three exchanges between lanes turn a lane's 8 columns of a
            // feature into 8 features of a column. (A store of two bytes for each value took 132 us for experts on slabs of 7000 rows of
            // 2048 where this took 117.)
            // (inner values: always)
            const bool wide_stores = kUp || (kOp != kLayerDown && p.wide_stores && (x.f & 7) == 0 && (x.height & 7) == 0);
            // where features f0 to f0 + 7 of column c go, and how many of them there are; none: 0
            auto place_of = [&](int c, int within8, int& f0, void*& to, size_t& o) {
                f0 = x.f + within8;
                if (within8 >= x.height || f0 >= p.features || c >= x.columns) return 0;
                if (kOne) {
                    o = (size_t)(x.first + c) * p.y_stride + f0;
                    to = p.y;
                    return min(8, p.features - f0);
                }
                if (kUp) {
                    o = (size_t)(s.row[x.group] + x.first + c) * p.features + f0;
                    to = p.hidden;
                    return 8;
                }
                const int row = s.list[buffer][c];
                o = (size_t)row * p.features + f0;
                to = p.y;
                return row >= 0 ? 8 : 0;
            };
            // A column's features `q` to their places.
            auto store_packed = [&](const uint4& q, int c, int within8) {
                int f0;
                void* to;
                size_t o;
                const int n = place_of(c, within8, f0, to, o);
                if (n == 8) {
                    *reinterpret_cast<uint4*>(static_cast<T*>(to) + o) = q;
                } else if (n > 0) {  // the last ones
                    const uint32_t word[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (j < n) reinterpret_cast<uint16_t*>(to)[o + j] = (uint16_t)(word[j / 2] >> 16 * (j & 1));
                }
            };
            // Without SwiGLU, residual and 32-bit results the exchange is the shared memory's: fragments of the sums go there turned over, and come back
            // as 8 features of a column. (16384 rows of 1024 to 2048: 51 us, with shuffles 60; 8192 of 512 to 4096 35 and 55.)
            const bool turns = kOp != kLayerDown && !k32 && !kUp && wide_stores && !paired && (!kOne || p.residual == nullptr);
            float biases[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (kOne && turns && p.bias != nullptr)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int at_row = quarter * 32 + 8 * j + (lane >> 2);
                    if (at_row < x.height && x.f + at_row < p.features) biases[j] = load_any<T>(p.bias, (size_t)x.f + at_row, p.bias_fp32);
                }
            auto finish_turned = [&](int c0, float (&v)[16]) {
                if (kOne) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] += biases[2 * (i >> 3) + (i >> 1 & 1)];
                    activate(v, p.activation);
                }
                const uint32_t mine = shared_addr(s.turned[warp - 4]);
                // (16 bytes of neighbouring rows lie apart, so that the eight of a matrix come from all banks)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t q[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) q[j] = packed<T>(v[8 * (j >> 1) + 4 * c + 2 * (j & 1)], v[8 * (j >> 1) + 4 * c + 2 * (j & 1) + 1]);
                    store_turned(mine + (8 * c + (lane & 7)) * 64 + (((lane >> 3) ^ (lane >> 1 & 3)) << 4), q);
                }
                __syncwarp();
                uint4 q[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int c = 8 * h + (lane >> 2);
                    q[h] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(s.turned[warp - 4]) + c * 64 + (((lane & 3) ^ (c >> 1 & 3)) << 4));
                }
                __syncwarp();
#pragma unroll
                for (int h = 0; h < 2; ++h) store_packed(q[h], c0 + 8 * h + (lane >> 2), quarter * 32 + 8 * (lane & 3));
            };
            // kStep: what the columns of the eight values differ by in lanes. Inner values are rounded to the rows' type, since the next product
            // takes 16-bit operands.
            auto store_eight = [&](float (&v)[8], auto step, int c, int within8) {
                constexpr int kStep = decltype(step)::value;
                int f0;
                void* to;
                size_t o;
                if (!kOne || (p.residual == nullptr && !k32)) {
                    store_packed(exchange_packed<kStep, T>(v, lane), c, within8);
                    return;
                }
                exchange_eight<kStep>(v, lane);
                const int n = place_of(c, within8, f0, to, o);
                const size_t from = (size_t)(x.first + c) * p.residual_stride + f0;
                if (n == 8) {
                    if (p.residual != nullptr) add_eight<T>(v, p.residual, from, k32);
                    put_eight<T>(to, o, v, k32);
                } else if (n > 0) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if (j >= n) break;
                        const float add = p.residual != nullptr ? load_any<T>(p.residual, from + j, k32) : 0.0f;
                        store_any<T>(to, o + j, v[j] + add, k32);
                    }
                }
            };
            auto finish_wide = [&](int c0, float (&v)[16]) {
                if (paired) {
                    float out[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float even = v[2 * j] + bias, odd = v[2 * j + 1] + bias;
                        const float other = __shfl_xor_sync(0xffffffffu, up ? even : odd, 1);
                        out[j] = silu(up ? other : even) * (up ? odd : other);
                    }
                    store_eight(out, Lanes<2>(), c0 + (lane & 15), quarter * 16 + 8 * (lane >> 4));
                }
#pragma unroll
                for (int h = 0; h < 2 && !paired; ++h) {
                    float out[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) out[j] = kOne ? v[8 * h + j] + bias : v[8 * h + j];
                    if (kOne) activate(out, p.activation);
                    store_eight(out, Lanes<1>(), c0 + 8 * h + (lane & 7), quarter * 32 + 8 * (lane >> 3));
                }
            };
            if (kCut) {
                // The cluster's blocks leave their sums in the ring, which nothing uses any more, and each finishes its share of the
                // columns, two at a time.
                float* const left = reinterpret_cast<float*>(ring);
                for_parts(x.columns, half, total, [&](int c0, float (&part_sums)[16]) {
                    float v[16];
                    if (!needed) return;
                    if constexpr (!k32) tmem_load_16(sums + c0, v);
#pragma unroll
                    for (int j = 0; j < 16; ++j) left[(c0 + j) * kTileRows + own] = k32 ? part_sums[j] : v[j];
                });
                cluster_sync();
                met = true;
                for (int c = 2 * (part + split * half); c < x.columns && needed; c += 4 * split) {
                    float v[2] = {0.0f, 0.0f};
                    for (int r = 0; r < split; ++r) {
                        const float* const theirs = cluster_address(left, r);
                        v[0] += theirs[c * kTileRows + own];
                        v[1] += theirs[(c + 1) * kTileRows + own];
                    }
                    finish(c, v);
                }
            } else if (k32) {
                for_parts(x.columns, half, total, [&](int c0, float (&v)[16]) {
                    if (!needed) return;
                    if (wide_stores) finish_wide(c0, v);
                    else finish(c0, v);
                });
            } else if (needed) {
                for (int c0 = 16 * half; c0 < x.columns; c0 += 32) {
                    float v[16];
                    if (spread) tmem_load_spread(sums, [&](int j) { return s.list[buffer][min(c0 + j, x.columns - 1)] / p.topk; }, v);
                    else if (turns) tmem_load_fragments(sums + c0, v);
                    else tmem_load_16(sums + c0, v);
                    if (c0 + 32 >= x.columns) sums_read(buffer);
                    if (turns) finish_turned(c0, v);
                    else if (wide_stores) finish_wide(c0, v);
                    else if constexpr (!kUp) finish(c0, v);
                }
            }
            if (!k32 && (!needed || 16 * half >= x.columns)) sums_read(buffer);  // this warp had none to read
            if (kGrouped) {
                named_sync(1, kFinishers);
                if (at == 0) barrier_arrive(list_empty0 + 8 * buffer);
            }
        }
        if (!met) cluster_sync();  // it gave up; the cluster's other blocks are waiting
    }
    __syncwarp();
    // What the epilogue's threads meet at, the others meet here: nobody leaves while its sums are read.
    if (kCut) {
        if (warp < 4) cluster_sync();
        cluster_sync();
    }
    tcgen05_before_sync();
    __syncthreads();
    if (kPair) cluster_sync();  // the other block's products and arrivals have come here
    tcgen05_after_sync();
    if (s.gave_up) {
        // copies and products in flight end in less than this
        const long long begin = clock64();
        while (clock64() - begin < 2000000) __nanosleep(1000);
        if (tid == 0) {
            *reinterpret_cast<volatile int*>(p.error) = A2A_ERR_TIMEOUT;
            __threadfence_system();
        }
        __syncthreads();
    }
    if (warp == 1) tmem_free<kPair>(tmem, kTmemColumns);
}

// The rows of a layer's pairs by expert, and within an expert in the order of the pairs: a block a pair, which counts the pairs before its own
// and copies the token's row. (A warp a pair: 18 us for 2048 of 4096, instead of 9.)
constexpr int kSortThreads = 128;
struct SortParams {
    const void* x;
    const int* indices;
    void* rows;
    int tokens, topk, experts, row_bytes;
};
__global__ void __launch_bounds__(kSortThreads) layer_rows_kernel(const SortParams p) {
    __shared__ int counted[kSortThreads / 32];
    cudaGridDependencySynchronize();
    cudaTriggerProgrammaticLaunchCompletion();
    const int pairs = p.tokens * p.topk, pair = blockIdx.x, tid = threadIdx.x;
    const int own = p.indices[pair];
    if (own < 0 || own >= p.experts) return;
    int before = 0;
#pragma unroll 8
    for (int i = tid; i < pairs; i += kSortThreads) {
        const int e = p.indices[i];
        before += e >= 0 && (e < own || (e == own && i < pair));
    }
    before = __reduce_add_sync(0xffffffffu, before);
    if ((tid & 31) == 0) counted[tid >> 5] = before;
    __syncthreads();
    before = 0;
    for (int w = 0; w < kSortThreads / 32; ++w) before += counted[w];
    const uint4* const from = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.x) + (size_t)(pair / p.topk) * p.row_bytes);
    uint4* const to = reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.rows) + (size_t)before * p.row_bytes);
#pragma unroll 4
    for (int i = tid; i < p.row_bytes / 16; i += kSortThreads) to[i] = from[i];
}

// y[t] = residual[t] + the rows of the token's pairs, in the order of its choices; a thread four features.
constexpr int kSumThreads = 256;
struct SumParams {
    const float* parts;
    const int* indices;
    const void* residual;
    void* y;
    int topk, experts, features;
};
template <typename T>
__global__ void __launch_bounds__(kSumThreads) layer_sum_kernel(const SumParams p) {
    const int token = blockIdx.x, f = 4 * (blockIdx.y * kSumThreads + threadIdx.x);
    // indices and residual were there before the call
    unsigned chosen = 0;
    for (int k = 0; k < p.topk; ++k) {
        const int e = p.indices[token * p.topk + k];
        chosen |= (unsigned)(e >= 0 && e < p.experts) << k;
    }
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f}, add[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const bool inside = f < p.features;  // a multiple of 8
    const size_t o = (size_t)token * p.features + f;
    if (inside && p.residual != nullptr)
#pragma unroll
        for (int j = 0; j < 4; ++j) add[j] = Element<T>::to_float(static_cast<const T*>(p.residual)[o + j]);
    cudaGridDependencySynchronize();
    cudaTriggerProgrammaticLaunchCompletion();
    if (!inside) return;
    const float* const parts = p.parts + (size_t)token * p.topk * p.features + f;
#pragma unroll 8
    for (int k = 0; k < p.topk; ++k) {
        if (!(chosen >> k & 1)) continue;
        const float4 v = __ldcg(reinterpret_cast<const float4*>(parts + (size_t)k * p.features));
        sum[0] += v.x, sum[1] += v.y, sum[2] += v.z, sum[3] += v.w;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) static_cast<T*>(p.y)[o + j] = Element<T>::from_float(sum[j] + add[j]);
}

}  // namespace
