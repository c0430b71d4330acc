// The backward kernels of the norms around a residual block for f16 operands (a file per type: they compile side by side).
#define FNET_BLOCK_NORM_BWD_KERNEL
#include "fnet_block_norm_bwd.h"

FNET_BLOCK_NORM_BWD_INSTANCES(f16_t)
