// What a block copies of a tile's rows, in plain functions: the kernel's roles, which have to agree on the bytes that a barrier expects, take it from
// here, and so does the model of these roles that runs on the host (tests/test_product_pairs.py).
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

// Rows of a box where a run has `n` rows, a multiple of eight, and of all its boxes, the last of which begins early.
PRODUCT_SHARES int box_of_run(int n) { return n >= 64 ? 64 : n >= 32 ? 32 : 8; }
PRODUCT_SHARES int boxed_rows(int n) {
    const int box = box_of_run(n);
    return (n + box - 1) / box * box;
}
