"""Element type codes of the C ABI (include/fluidnet_hip.h FNET_F32 / FNET_BF16 / FNET_F16) by torch dtype."""
import torch

from .runtime import BF16, F16, F32

ELEM = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}
