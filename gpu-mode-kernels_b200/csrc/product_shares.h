// What a block copies of a tile's rows, and how much of a sum stays together, in plain functions: the kernel's roles, which have to agree on the bytes that a
// barrier expects, take it from here, and so do tests on the host (tests/test_product_pairs.py has a model of the roles).
#pragma once

#ifdef __CUDACC__
#define PRODUCT_SHARES __host__ __device__ __forceinline__
#else
#define PRODUCT_SHARES inline
#endif

// Columns that block `of` of `blocks` copies, from `from` on, in eights: of a tile of `columns`, whose product has `product` of them (a multiple of 16 a
// block). A pair's second block copies eight even where the tile has none for it. The first block's barrier then waits for these bytes, and so the
// products wait for the role that copies them: a role whose bytes nobody waited for stayed behind the ring, whose barriers are waited for by the
// parity of their phase, and once it was two phases behind its wait did not end. (What it copies there are columns that nothing reads.)
PRODUCT_SHARES int copied_columns(int columns, int product, int blocks, int of, int* from) {
    const int share = product / blocks;
    *from = of * share;
    int n = columns - of * share;
    n = n < share ? n : share;
    n = (n + 7) & ~7;
    return n > 8 ? n : 8;
}

// a / b for a >= 0, b > 0. A block works out a dozen of them, one after the other, before its first copy is on its way: an integer division is
// 100 cycles and more, this half of that. (The quotient of a + 1/2 is at least 1/(2 b) away from a whole number, and __fdividef
// is off by 2^-22 of it.)
PRODUCT_SHARES int quotient(int a, int b) {
#ifdef __CUDA_ARCH__
    if (a < 1 << 20) return (int)__fdividef((float)a + 0.5f, (float)b);
#endif
    return a / b;
}

// Blocks of 64 of the inner length in a stage of the ring, of `blocks` of `block_bytes` each: about as many as reach `stage_bytes`, at most `most`.
PRODUCT_SHARES int stage_blocks(int blocks, int block_bytes, int stage_bytes, int most) {
    int n = quotient(stage_bytes + block_bytes / 2, block_bytes);
    n = n > 1 ? n : 1;
    n = n < most ? n : most;
    return n < blocks ? n : blocks;
}
// Blocks that a sum in tensor memory is of where it may be of `most`: whole stages.
PRODUCT_SHARES int sum_blocks(int per_stage, int most) { return quotient(most, per_stage) * per_stage; }

// Rows of a box where a run has `n` rows, a multiple of eight, and of all its boxes, the last of which begins early.
PRODUCT_SHARES int box_of_run(int n) { return n >= 64 ? 64 : n >= 32 ? 32 : 8; }
PRODUCT_SHARES int boxed_rows(int n) {
    const int box = box_of_run(n);
    return (n + box - 1) / box * box;
}
