// The kernels of the norms around a residual block for f32 operands (a file per type: they compile side by side).
#define FNET_BLOCK_NORM_KERNELS
#include "fnet_block_norm_bwd.h"
#include "fnet_block_norm_fwd.h"

FNET_BLOCK_NORM_INSTANCES(float)
