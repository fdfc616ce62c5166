"""Launch path of the batched operators.

A decode step makes several of these calls per layer, so their host time is the step's time when the batch is small. Plain
calls go through the CPython module built from csrc/torch_binding.cpp (`fast`, loaded with the first device), which checks,
allocates and launches in a few microseconds; whatever it answers None to comes back to the Python wrappers, which raise or
launch through ctypes (`launch`): torch's current stream, the device switched only when it is not the current one, and the
caching allocator told which stream used the tensors (_native.record). Where the binding was not built (no headers of torch
or Python), every call goes that way, 10 to 16 us of host time slower.
"""

from __future__ import annotations

import ctypes as ct
import importlib.machinery
import importlib.util
import threading
import warnings

import torch

from . import _native
from ._module import get_module

_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_capturing = torch._C._cuda_isCurrentStreamCapturing
_functions = {}
_streams = {}
_ready = set()
_lock = threading.Lock()
# The entry points in the order that the binding takes them.
_ENTRIES = ("klab_kv_build_step", "klab_kv_store", "klab_kv_read", "klab_kv_attention", "klab_kv_attention_new",
            "klab_kv_attention_scratch", "klab_adapter_linear", "klab_adapter_scratch")
BINDING = _native.LIB_DIR / "klab_torch.so"
fast = None  # the binding, once a device is ready


def load_binding():
    """The binding module with _native's entry points (no device needed)."""
    if not BINDING.exists():
        raise RuntimeError(f"{BINDING} is missing: build it with `python -m klab_b200.build`")
    loader = importlib.machinery.ExtensionFileLoader("klab_torch", str(BINDING))
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader("klab_torch", loader))
    loader.exec_module(module)
    lib = _native.lib()
    module.bind(*(ct.cast(getattr(lib, name), ct.c_void_p).value for name in _ENTRIES))
    return module


def ready(device):
    """The device's index, its module loaded (outside capture the first time)."""
    index = device.index
    if index not in _ready:
        if device.type != "cuda":
            raise ValueError("Expected CUDA tensors")
        get_module(device)
        global fast
        with _lock:
            if fast is None and BINDING.exists():
                fast = load_binding()
            if fast is None:
                if not _ready:
                    warnings.warn(f"{BINDING.name} is not built: batched operators launch through ctypes", RuntimeWarning,
                                  stacklevel=3)
            elif index < 64:
                fast.mark_ready(index)
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
