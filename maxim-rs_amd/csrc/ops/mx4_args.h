// Argument blocks of the 4-bit operators' kernels.
//
// 4-bit matrices: lines of `tiles` times 128 bytes, a tile 256 elements, and
// scales in groups of 64 lines, 512 bytes a group and tile, in the order that a
// wave's lanes feed its matrix instructions: [k / 32 % 4][line % 16][line / 16 %
// 4][k / 128 % 2].
#pragma once

#include <stdint.h>

#include "ops_args.h"

// x [rows][cols] at rs and cs elements to or from codes and scales.
struct Mx4CodeArgs {
    const void *x;
    void *y;
    uint8_t *codes, *scales;
    int64_t rows, cols, rs, cs;
    int32_t tiles, pad;
};

// The epilogue's and the splits' fields are a product's (a, b, lda and ldb are
// not read); k counts tiles, and split s has tiles [s kchunk, (s + 1) kchunk).
struct Mx4GemmArgs {
    OpsGemmArgs g;
    const uint8_t *a, *b;    // codes; a: few rows take x itself, lda elements apart
    const uint8_t *sa, *sb;  // scales
    int64_t cols;            // features of x, few rows
};
