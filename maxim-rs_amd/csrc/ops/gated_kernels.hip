// The gfx950 code object of the gated Dense (include/maxim_block_ops.h).
#define OPS_GATED
#include "ops_gated.h"
