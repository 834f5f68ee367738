// Argument block of the gradient norm's and clipping's kernels.
#pragma once

#include <stdint.h>

// Up to so many tensors a launch: the block of arguments stays below 4 KiB.
enum { MXN_TENSORS = 128, MXN_CHUNK = 16384 };

// Tensors as runs of MXN_CHUNK bytes: tensor i's are first[i] to first[i + 1],
// its elements n[i], of the type in n's top byte.
struct GradsArgs {
    const void *src[MXN_TENSORS];
    void *dst[MXN_TENSORS];
    uint64_t n[MXN_TENSORS];
    uint32_t first[MXN_TENSORS + 1];
    int32_t count;
    double *part;        // a block's sum of squares each
    float *norm;         // clipping: read; few chunks: written
    float max_norm;
    int32_t clip;        // few chunks: not the norm alone
};

struct GradsJoinArgs {
    const double *part;
    float *norm;
    int32_t nparts, pad;
};
