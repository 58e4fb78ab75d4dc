"""What the calls on rows of heads share (rope, kvcache): the rows' types, the GPU and the stream of a launch."""
import contextlib

import torch

from . import _native as nat

_ROW = {torch.bfloat16: nat.RH3_DTYPE_BF16, torch.float16: nat.RH3_DTYPE_F16, torch.float32: nat.RH3_DTYPE_F32}
_HERE = contextlib.nullcontext()


# The small calls (a token of one sequence is 12 us of GPU work in two launches) are bound by what the host does: shapes, strides
# and devices are asked for once a call, devices as numbers, and the workspace's size once for each set of sizes.
def _on(index):
    """The tensors' GPU as the current one for a launch, where it is another."""
    return _HERE if index == torch._C._cuda_getDevice() else torch.cuda.device(index)


_stream = torch._C._cuda_getCurrentRawStream
