"""The current stream of a device, and a library call on a device that may not be the current one, at the cost a decode
step can bear."""

from __future__ import annotations

import torch

from lean_vllm_b200._native import check


def raw_stream(device: int) -> int:
    """The current stream of CUDA device `device`, as a cudaStream_t (torch.cuda.current_stream builds an object for
    it, 1 us more)."""
    return torch._C._cuda_getCurrentRawStream(device)


def call(device: int, function, *args) -> None:
    """Calls a library function that launches on the current device, with `device` as that; raises for an error."""
    if torch.cuda.current_device() == device:
        check(function(*args))
    else:
        with torch.cuda.device(device):
            check(function(*args))
