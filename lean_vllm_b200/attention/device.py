"""The current stream of a device, and a library call on a device that may not be the current one, at the cost a decode
step can bear."""

from __future__ import annotations

import ctypes

import torch

from lean_vllm_b200._native import check, lib


def raw_stream(device: int) -> int:
    """The current stream of CUDA device `device`, as a cudaStream_t (torch.cuda.current_stream builds an object for
    it, 1 us more)."""
    return torch._C._cuda_getCurrentRawStream(device)


def stream_of(handle: int, device: torch.device) -> torch.cuda.Stream:
    """The stream object of a cudaStream_t; 0 is the default stream (torch.cuda.ExternalStream(0) would be another)."""
    return torch.cuda.ExternalStream(handle, device) if handle else torch.cuda.default_stream(device)


def output_like(query: torch.Tensor, stream: int | None) -> torch.Tensor:
    """An uninitialised contiguous tensor of the queries' shape that a launch on `stream` (a cudaStream_t; None: the current
    stream) may write at once. It is that stream's memory: what is still queued on the current stream for memory freed
    there cannot reach it. The current stream, where the caller goes on, is made known to the allocator."""
    if stream is None or not query.is_cuda:
        return torch.empty_like(query, memory_format=torch.contiguous_format)  # half the cost of torch.empty
    with torch.cuda.stream(stream_of(stream, query.device)):
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
    out.record_stream(torch.cuda.current_stream(query.device))
    return out


def no_gradient(*tensors: torch.Tensor | None) -> None:
    """Refuses tensors whose gradient would be lost: these calls are for serving and have no backward pass."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError("no gradient passes through this call: make it under torch.no_grad() or inference_mode(), or "
                         "detach its inputs")


def call(device: int, function, *args) -> None:
    """Calls a library function that launches on the current device, with `device` as that; raises for an error."""
    if torch.cuda.current_device() == device:
        check(function(*args))
    else:
        with torch.cuda.device(device):
            check(function(*args))


def _bind():
    """The C++ marshalling of the plain calls (csrc/calls.cpp), bound to the library; None where it is not built, or was
    built against another torch (which may keep it from loading, or not): the Python wrappers then do the same, slower."""
    try:
        from lean_vllm_b200 import _calls
    except ImportError:
        return None
    if getattr(_calls, "torch_version", None) != torch.__version__:
        return None
    handle = lib()
    _calls.bind(ctypes.cast(handle.kvx_attention, ctypes.c_void_p).value,
                ctypes.cast(handle.kvx_rotate_store, ctypes.c_void_p).value)
    return _calls


_bound: list = []


def calls():
    """The bound module, or None."""
    if not _bound:
        _bound.append(_bind())
    return _bound[0]
