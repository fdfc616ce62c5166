"""Launch path of the batched operators: torch's current stream of a device, the native call, and the caching allocator's
stream bookkeeping (_native.record) with as little host time as the calls themselves allow.

A decode step makes several of these calls per layer, so their host time is the step's time when the batch is small: the
stream comes as a raw handle, the device is switched only when it is not the current one, and Stream objects are kept
per handle for record_stream.
"""

from __future__ import annotations

import torch

from . import _native
from ._module import get_module

_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_capturing = torch._C._cuda_isCurrentStreamCapturing
_functions = {}
_streams = {}
_ready = set()


def ready(device):
    """The device's index, its module loaded (outside capture the first time)."""
    index = device.index
    if index not in _ready:
        if device.type != "cuda":
            raise ValueError("Expected CUDA tensors")
        get_module(device)
        _ready.add(index)
    return index


def _resolve(name):
    fn = _functions[name] = getattr(_native.lib(), name)
    return fn


def _stream_object(index, raw):
    stream = _streams[index, raw] = torch.cuda.current_stream(index)
    return stream


def launch(name, index, args, tensors):
    """lib().<name>(*args, stream) on device `index`'s current stream; `tensors` are recorded on it outside capture."""
    fn = _functions.get(name) or _resolve(name)
    raw = _raw_stream(index)
    if _current_device() == index:
        rc = fn(*args, raw)
        capturing = _capturing()
    else:
        with torch.cuda.device(index):
            rc = fn(*args, raw)
            capturing = _capturing()
    if rc:
        _native.check(rc, name)
    if not capturing:
        stream = _streams.get((index, raw)) or _stream_object(index, raw)
        for t in tensors:
            t.record_stream(stream)
