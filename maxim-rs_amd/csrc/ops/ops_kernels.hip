// The gfx950 code object of the training and serving operators
// (include/maxim_ops.h), apart from the executor's: a program that only runs
// plans never loads it.
#include "ops_rows.h"
#include "ops_gemm.h"
#include "ops_gemm_big.h"
#include "ops_skinny.h"
