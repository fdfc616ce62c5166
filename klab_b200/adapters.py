"""Low-rank adapters of many requests beside a shared projection.

adapter_linear(x, w, a, b, scales, ids) is the projection x W^T of this package (BF16, INT8 or FP4 weights) with, for each
token row, the low-rank product of its own adapter added before the one rounding:

    y[m] = x[m] W^T + scales[i] * (x[m] a[i]^T) b[i]^T,   i = ids[m]; ids[m] = -1: x[m] W^T alone.

Adapters of different ranks share a stack by padding with zero rows of a (and columns of b). No counterpart in the
reference, whose projections serve one set of weights.
"""

from __future__ import annotations

from functools import lru_cache

import torch

from . import _launch, _native
from ._launch import launch, ready
from .compressed_bf16 import PackedBF16
from .fp4 import FP4F16Weights
from .int8_weights import Int8Weights

MAX_RANK = 256


# Formats whose projection runs inside the adapters' own kernel (16-byte aligned rows); the others call the projection.
_STREAMED = (_native.W_BF16, _native.W_I8_ROW, _native.W_FP4_G32H)


@lru_cache(maxsize=256)
def _scratch_bytes(index, *shape):
    with torch.cuda.device(index):
        need = _native.lib().klab_adapter_scratch(*shape)
    if need < 0:
        _native.check(int(need), "klab_adapter_scratch")
    return int(need)


def _workspace(index, device, wfmt, m, n, k):
    """The projection's split-K workspace. A captured call gets its own: two graphs captured on one stream may be replayed
    on two, and must not share tickets."""
    need = int(_native.lib().klab_gemv_workspace_bytes(wfmt, m, n, k))
    if torch.cuda.is_current_stream_capturing():
        return (torch.zeros(need, device=device, dtype=torch.uint8), need) if need else (None, 0)
    buffer = _native.WORKSPACES.get(index, torch.cuda.current_stream(device), need)
    return (buffer, buffer.numel()) if buffer is not None else (None, 0)


def _weights(w, k):
    """(format, weights, side tensor, N) of the shared projection."""
    if isinstance(w, Int8Weights):
        codes, scales = w.codes, w.scales
        if codes.dtype != torch.int8 or codes.ndim != 2 or codes.shape[1] != k or scales.dtype != torch.float32:
            raise ValueError("Expected INT8 codes [N,K] and FP32 scales")
        n = codes.shape[0]
        if scales.shape == (n,):
            return _native.W_I8_ROW, codes, scales, n
        if k % 64 or scales.shape != (n, k // 64):
            raise ValueError("INT8 scales must be [N] or [N,K/64]")
        return _native.W_I8_G64, codes, scales, n
    if isinstance(w, FP4F16Weights):
        n = w.packed.shape[0]
        if k % 32 or w.packed.dtype != torch.uint8 or w.packed.shape != (n, k // 2) or w.scales.dtype != torch.float16 \
                or w.scales.shape != (n, k // 32):
            raise ValueError("Expected packed uint8 [N,K/2] and FP16 scales [N,K/32]")
        return _native.W_FP4_G32H, w.packed, w.scales, n
    if isinstance(w, PackedBF16):
        if w.k != k or k % 64:
            raise ValueError("Expected x=[M,K] matching the weights, K a multiple of 64")
        return _native.W_CBF16, w.payload, w.metadata, w.n
    if not isinstance(w, torch.Tensor) or w.dtype != torch.bfloat16 or w.ndim != 2 or w.shape[1] != k:
        raise ValueError("w must be BF16 [N,K], Int8Weights, FP4F16Weights or PackedBF16 with x's K")
    return _native.W_BF16, w, None, w.shape[0]


def adapter_linear(x, w, a, b, scales, ids, *, out=None, output_dtype=torch.bfloat16):
    """x BF16 [M, K]; w BF16 [N, K], Int8Weights, FP4F16Weights or PackedBF16; a BF16 [adapters, rank, K], b BF16
    [adapters, N, rank] (rank a multiple of 8, at most 256), scales FP32 [adapters], ids int32 [M]. Returns [M, N] in
    output_dtype (BF16 or FP32). K must be a multiple of 8. An index outside -1 .. adapters - 1 counts as -1 and sets the
    device status to 6."""
    if _launch.fast is not None and output_dtype in (torch.bfloat16, torch.float32):
        fp32 = output_dtype is torch.float32
        if type(w) is torch.Tensor:
            done = _launch.fast.adapter_linear(_native.W_BF16, x, w, None, a, b, scales, ids, out, fp32)
        elif type(w) is Int8Weights:
            done = _launch.fast.adapter_linear(_native.W_I8_ROW, x, w.codes, w.scales, a, b, scales, ids, out, fp32)
        elif type(w) is FP4F16Weights:
            done = _launch.fast.adapter_linear(_native.W_FP4_G32H, x, w.packed, w.scales, a, b, scales, ids, out, fp32)
        else:
            done = None
        if done is not None:
            return done if type(done) is not int else _native.check(done, "klab_adapter_linear")
    if x.ndim != 2 or x.dtype != torch.bfloat16:
        raise ValueError("Expected BF16 x [M,K]")
    m, k = x.shape
    wfmt, weights, side, n = _weights(w, k)
    if a.dtype != torch.bfloat16 or b.dtype != torch.bfloat16 or a.ndim != 3 or b.ndim != 3 or a.shape[2] != k \
            or b.shape != (a.shape[0], n, a.shape[1]):
        raise ValueError("Expected BF16 a=[adapters, rank, K] and b=[adapters, N, rank]")
    count, rank, _ = a.shape
    if scales.dtype != torch.float32 or scales.shape != (count,) or ids.dtype != torch.int32 or ids.shape != (m,):
        raise ValueError("Expected FP32 scales [adapters] and int32 ids [M]")
    if min(m, n, k, count, rank) <= 0 or rank % 8 or rank > MAX_RANK or k % 8 or m > 65535:
        raise ValueError("Expected positive sizes, M <= 65535, K a multiple of 8, rank a multiple of 8 up to 256")
    if max(m * k, n * k, m * n) >= 2 ** 31:
        raise ValueError("Require 32-bit indices")
    if output_dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("output_dtype must be torch.bfloat16 or torch.float32")
    device = x.device
    read = [t for t in (x, weights, side, a, b, scales, ids) if t is not None]
    for t in read:
        if t.device != device or not t.is_contiguous() or t.requires_grad:
            raise ValueError("Inference-only contiguous tensors on one device required")
    if x.data_ptr() % 16 or a.data_ptr() % 16 or b.data_ptr() % 16 or weights.data_ptr() % (32 if side is not None and wfmt == _native.W_CBF16 else 4):
        raise ValueError("x, a and b must be 16-byte aligned, the weights 4-byte (packed ones 32-byte)")
    if out is not None:
        if out.dtype != output_dtype or out.device != device or out.shape != (m, n) or not out.is_contiguous() \
                or out.requires_grad:
            raise ValueError("out must be contiguous [M,N] of the requested dtype")
        o0, o1 = out.data_ptr(), out.data_ptr() + out.numel() * out.element_size()
        if any(o0 < t.data_ptr() + t.numel() * t.element_size() and t.data_ptr() < o1 for t in read):
            raise ValueError("out must not overlap the inputs")
    if device.type != "cuda":
        raise ValueError("Expected CUDA tensors")
    index = ready(device)
    if out is None:
        out = torch.empty((m, n), device=device, dtype=output_dtype)
    need = _scratch_bytes(index, wfmt, m, n, k, rank)
    scratch = torch.empty(need, device=device, dtype=torch.uint8)
    workspace, ws_bytes = None, 0
    if wfmt not in _STREAMED or weights.data_ptr() % 16 or weights.stride(0) * weights.element_size() % 16:
        workspace, ws_bytes = _workspace(index, device, wfmt, m, n, k)
    launch("klab_adapter_linear", index,
           (wfmt, x.data_ptr(), weights.data_ptr(), None if side is None else side.data_ptr(), a.data_ptr(), b.data_ptr(),
            scales.data_ptr(), ids.data_ptr(), out.data_ptr(),
            _native.DT_F32 if output_dtype is torch.float32 else _native.DT_BF16, m, n, k, rank, count, scratch.data_ptr(),
            need, None if workspace is None else workspace.data_ptr(), ws_bytes), (*read, out))
    return out
