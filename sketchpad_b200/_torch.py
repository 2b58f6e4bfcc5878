"""torch plumbing for the ctypes calls: dtype codes, stream handles, pointer extraction."""
from __future__ import annotations

import ctypes

import torch

from . import _lib

_DT = {torch.float32: _lib.SP_F32, torch.float16: _lib.SP_F16, torch.bfloat16: _lib.SP_BF16}


def dtype_code(t: torch.dtype) -> int:
    try:
        return _DT[t]
    except KeyError:
        raise TypeError(f"unsupported dtype {t}; expected float32, float16 or bfloat16") from None


def require_cuda(*tensors: torch.Tensor) -> torch.device:
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("sketchpad_b200 ops take CUDA tensors (there is no CPU path)")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"tensors on different devices: {dev} and {t.device}")
    return dev


def stream_ptr(device: torch.device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


try:
    _raw_stream = torch._C._cuda_getCurrentRawStream
except AttributeError:  # a torch built without CUDA: the operators raise before they get here
    def _raw_stream(index: int) -> int:
        return torch.cuda.current_stream(index).cuda_stream

try:
    _current_device = torch._C._cuda_getDevice
except AttributeError:
    def _current_device() -> int:
        return torch.cuda.current_device()


def raw_stream(index: int) -> int:
    """The handle of the device's current stream as an int (stream_ptr builds a Stream object
    first, 2.3 us of a small operator's call)."""
    return _raw_stream(index)


def cuda_index(x: torch.Tensor, *others) -> int:
    """The device index that x and the others (None: absent) share, which has to be the current
    one (kernels are launched there); ValueError as require_cuda."""
    i = x.get_device()
    if i < 0:
        raise ValueError("sketchpad_b200 ops take CUDA tensors (there is no CPU path)")
    if i != _current_device():
        raise ValueError(f"the tensors are on cuda:{i} and the current device is "
                         f"cuda:{_current_device()} (torch.cuda.set_device)")
    for t in others:
        if t is not None and t.get_device() != i:
            require_cuda(x, *others)
    return i


class Workspaces:
    """Zero-initialised device workspaces, one per (device, stream): the kernels that use them
    leave their counters zero again, so calls in one stream's order share one, which grows with
    them.  A call that is being captured never gets the stream's: the graph would outlive it, and
    replays would meet the stream's other calls in it.  It gets one of the graph's own memory,
    zeroed by a node of the graph (a workspace that the caller keeps saves that node)."""

    def __init__(self):
        self._kept = {}

    def get(self, index: int, stream: int, nbytes: int):
        """(tensor to hold on to until the launch, pointer, bytes) of at least nbytes."""
        capturing = torch.cuda.is_current_stream_capturing()
        w = None if capturing else self._kept.get((index, stream))
        if w is None or w[2] < nbytes:
            n = (nbytes + 3) // 4
            t = torch.zeros(n, dtype=torch.int32, device=torch.device("cuda", index))
            w = (t, t.data_ptr(), n * 4)
            if not capturing:
                self._kept[index, stream] = w
        return w


def given_workspace(t: torch.Tensor):
    """What Workspaces.get returns, of a workspace that the caller gives."""
    if not t.is_contiguous():
        raise ValueError("workspace must be contiguous")
    return t, t.data_ptr(), t.numel() * t.element_size()


def ptr(t) -> ctypes.c_void_p:
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


def strides4(t: torch.Tensor):
    return _lib.i64_array(t.stride())
