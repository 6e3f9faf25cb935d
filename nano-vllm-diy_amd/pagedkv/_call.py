"""Calls of the C-ABI for operators whose work is a few microseconds: no device guard where the tensors'
device is the current one, and the current stream's handle without a stream object."""
from __future__ import annotations

import torch

from ._lib import check

# (not a public function: without it, through the stream object)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def call(fn, what: str, device: torch.device, *args) -> None:
    """fn(*args, current stream of device) with device current; raises what it refuses."""
    index = device.index
    if index is None:
        raise ValueError(f"{what}: tensors must be on a GPU, not on {device}")
    if index == torch.cuda.current_device():
        code = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            code = fn(*args, _raw_stream(index))
    if code:
        check(code, what)


def scratch(nbytes: int, device: torch.device) -> torch.Tensor:
    """One buffer per call: stream-ordered by the allocator outside capture, from the capture's own
    pool under it, so neither two streams nor two graphs share one."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device)
