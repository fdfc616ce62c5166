"""A batch of requests over 4-bit K/V pages: page tables, rows into pages and back, and attention over them.

Where decode_attn serves one sequence from a contiguous BF16 cache (the reference's form,
research/l2-prefetch/src/decode_attn.py:20-107), these serve many requests of uneven lengths from shared pages that
hold 4.5 bits a value. One step of a batch:

    step = build_step(new_tokens, lengths, table, free_pages, free_count, page_size=16, max_tokens=m)
    ...                                        # projections of the step's token rows
    store(k, v, pages, step.slots)
    out = attention(q, pages, table, step.lengths, step.starts, max_new=1)

Everything that changes from step to step stays on the GPU (lengths, table, free pages, slots), so a captured CUDA graph
serves any lengths: launch shapes depend on tensor shapes alone. Values that the device reads and that are out of range
(a page, a length) never leave a buffer's bounds: the work is skipped and _native.device_status() says so.

pages is uint8 [num_pages, kv_heads, page_bytes(page_size, head_dim)]: 16-token blocks of signed 4-bit codes with one FP16
scale per 32 dims of a token and head (include/klab_b200.h gives the format, csrc/kv_pages.cuh the order of the bytes).
"""

from __future__ import annotations

import math
from functools import lru_cache
from typing import NamedTuple

import torch

from . import _launch, _native
from ._launch import launch, ready

HEAD_DIMS = (64, 128, 256)
GROUP = 32            # dims that share a scale
MAX_NEW = 16          # new tokens of a request in one attention call
MAX_REQUESTS = 8192
MAX_GROUP = 64        # query heads of a kv head
STEP_OK, STEP_LENGTH, STEP_TABLE, STEP_PAGES, STEP_TOKENS = range(5)
_DT = {torch.bfloat16: _native.DT_BF16, torch.float16: _native.DT_F16}
_ODT = {**_DT, torch.float32: _native.DT_F32}


class BatchStep(NamedTuple):
    """What build_step gives out (all int32 on the GPU)."""

    slots: torch.Tensor       # [max_tokens] where each new token goes; -1 behind the last
    positions: torch.Tensor   # [max_tokens] its position in its request; 0 behind the last
    rows: torch.Tensor        # [max_tokens] its request; -1 behind the last
    starts: torch.Tensor      # [requests + 1] first new token of each request
    lengths: torch.Tensor     # [requests] tokens of each request after the step
    free_count: torch.Tensor  # [1] free pages after the step
    result: torch.Tensor      # [1] STEP_OK, or why nothing was given out


def page_bytes(page_size: int, head_dim: int) -> int:
    """Bytes of one page of one kv head: codes of K and V, and their scales."""
    _check_page_size(page_size)
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}")
    return page_size * head_dim * 9 // 8


def empty_pages(num_pages: int, kv_heads: int, page_size: int, head_dim: int, device="cuda") -> torch.Tensor:
    """Pages of any content (what no token was stored into is never read as a value)."""
    if min(num_pages, kv_heads) <= 0 or num_pages * page_size >= 2 ** 31:
        raise ValueError("num_pages and kv_heads must be positive, num_pages * page_size below 2^31")
    return torch.empty((num_pages, kv_heads, page_bytes(page_size, head_dim)), device=device, dtype=torch.uint8)


def _check_page_size(page_size):
    if isinstance(page_size, bool) or not isinstance(page_size, int) or not 16 <= page_size <= 1024 \
            or page_size & (page_size - 1):
        raise ValueError("page_size must be a power of two from 16 to 1024")


def _check_ints(device, **tensors):
    for name, t in tensors.items():
        if t.dtype is not torch.int32 or not t.is_contiguous() or t.device != device:
            raise ValueError(f"{name} must be a contiguous int32 tensor on {device}")


def _check_device(device, *tensors):
    for t in tensors:
        if t.requires_grad:
            raise ValueError("Inference only: no requires_grad")
    if device.type != "cuda":
        raise ValueError("Expected CUDA tensors")


def _span(t):
    """First and last byte + 1 that a tensor with positive strides reaches."""
    p = t.data_ptr()
    if t.is_contiguous():
        return p, p + t.numel() * t.element_size()
    return p, p + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()


def _disjoint(written, *read):
    """`written` shares no byte with the others."""
    w0, w1 = _span(written)
    for t in read:
        if t is not written:
            r0, r1 = _span(t)
            if r0 < w1 and w0 < r1:
                raise ValueError("Tensors that are written must not overlap the others")


@lru_cache(maxsize=256, typed=True)
def _check_sizes(page_size, lengths, table, free_pages, free_count):
    """The shapes of a batch's state; cached, since a server's never change."""
    _check_page_size(page_size)
    if len(lengths) != 1 or len(table) != 2 or table[0] != lengths[0] or len(free_pages) != 1 \
            or math.prod(free_count) != 1 or min(table) <= 0 or free_pages[0] <= 0:
        raise ValueError("Expected lengths=[requests], table=[requests, width], free_pages=[num_pages], free_count=[1]")
    if lengths[0] > MAX_REQUESTS or free_pages[0] * page_size >= 2 ** 31 or table[1] * page_size >= 2 ** 31:
        raise ValueError(f"At most {MAX_REQUESTS} requests, and fewer than 2^31 slots and positions")
    return table[0], table[1], free_pages[0]


def _check_state(lengths, table, free_pages, free_count, page_size):
    """(requests, width, num_pages) of a batch's state."""
    _check_ints(lengths.device, lengths=lengths, table=table, free_pages=free_pages, free_count=free_count)
    try:
        return _check_sizes(page_size, lengths.shape, table.shape, free_pages.shape, free_count.shape)
    except TypeError:
        raise ValueError("page_size must be a power of two from 16 to 1024") from None


def build_step(new_tokens, lengths, table, free_pages, free_count, *, page_size, max_tokens, inplace=False) -> BatchStep:
    """Pages and places for new_tokens[i] tokens behind the lengths[i] that request i has cached.

    lengths [requests], table [requests, width] (pages of each request in order), free_pages [num_pages] (a stack: the
    first free_count entries are free; its size is the number of pages) and free_count [1] are int32 on the GPU. New pages
    come from the top of the stack, requests in order, and are written into table; the other results are a new BatchStep,
    whose lengths and free_count are the state after the step (with inplace=True they are `lengths` and `free_count`
    themselves, for a captured step). max_tokens bounds the step's tokens. All or nothing: where result is not STEP_OK,
    no page was given out and there are no tokens.
    """
    if _launch.fast is not None:
        step = _launch.fast.build_step(new_tokens, lengths, table, free_pages, free_count, page_size, max_tokens, inplace)
        if step is not None:
            return BatchStep(*step) if type(step) is tuple else _native.check(step, "klab_kv_build_step")
    requests, width, num_pages = _check_state(lengths, table, free_pages, free_count, page_size)
    device = lengths.device
    _check_ints(device, new_tokens=new_tokens)
    if new_tokens.shape != lengths.shape:
        raise ValueError("new_tokens must have one entry per request")
    if not 0 < max_tokens < 2 ** 31:
        raise ValueError("max_tokens must be positive and below 2^31")
    _disjoint(table, new_tokens, lengths, free_pages, free_count)
    if inplace:
        _disjoint(lengths, new_tokens, free_pages, free_count)
        _disjoint(free_count, new_tokens, free_pages)
    _check_device(device)
    index = ready(device)
    sizes = (max_tokens, max_tokens, max_tokens, requests + 1, 1)
    if inplace:
        slots, positions, rows, starts, result = torch.empty(sum(sizes), device=device, dtype=torch.int32).split(sizes)
        lengths_out, count_out = lengths, free_count
    else:
        sizes += (requests, 1)
        slots, positions, rows, starts, result, lengths_out, count_out = torch.empty(
            sum(sizes), device=device, dtype=torch.int32).split(sizes)
    launch("klab_kv_build_step", index,
           (new_tokens.data_ptr(), lengths.data_ptr(), table.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(),
            requests, width, num_pages, page_size, max_tokens, slots.data_ptr(), positions.data_ptr(),
            rows.data_ptr(), starts.data_ptr(), lengths_out.data_ptr(), count_out.data_ptr(), result.data_ptr()),
           (new_tokens, lengths, free_pages, free_count, table))
    return BatchStep(slots, positions, rows, starts, lengths_out, count_out, result)


def release(ended, lengths, table, free_pages, free_count, *, page_size) -> None:
    """Requests with ended[i] (bool) give their pages back: pushed on the free stack, their table entries -1 and their
    lengths 0, all in place. Nothing changes (device status 4) when one of their table entries is no page."""
    requests, width, num_pages = _check_state(lengths, table, free_pages, free_count, page_size)
    device = lengths.device
    if ended.dtype != torch.bool or ended.device != device or ended.shape != lengths.shape or not ended.is_contiguous():
        raise ValueError("ended must be a contiguous bool tensor with one entry per request")
    state = (ended, lengths, table, free_pages, free_count)
    for t in state[1:]:
        _disjoint(t, *state)
    _check_device(device)
    launch("klab_kv_release", ready(device),
           (ended.data_ptr(), lengths.data_ptr(), table.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(),
            requests, width, num_pages, page_size), state)


@lru_cache(maxsize=256, typed=True)
def _page_layout(shape, head_dim):
    """(num_pages, kv_heads, page_size) of pages of this shape for heads of head_dim."""
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}")
    if len(shape) != 3:
        raise ValueError("pages must be [num_pages, kv_heads, page_bytes]")
    num_pages, kv_heads, size = shape
    page_size = size * 8 // (9 * head_dim)
    if min(num_pages, kv_heads) <= 0 or page_size * head_dim * 9 != size * 8:
        raise ValueError("pages do not hold whole tokens of this head_dim (see page_bytes)")
    _check_page_size(page_size)
    if num_pages * page_size >= 2 ** 31:
        raise ValueError("Fewer than 2^31 slots are supported")
    return num_pages, kv_heads, page_size


def _check_pages(pages, head_dim):
    layout = _page_layout(pages.shape, head_dim)
    if pages.dtype is not torch.uint8 or not pages.is_contiguous() or pages.data_ptr() % 16:
        raise ValueError("pages must be a contiguous, 16-byte aligned uint8 tensor [num_pages, kv_heads, page_bytes]")
    return layout


def store(k, v, pages, slots) -> None:
    """Rows k, v [tokens, kv_heads, head_dim] (BF16 or FP16; any token and head strides that are multiples of 4 elements,
    such as slices of a fused projection's output) into pages at slots [tokens] (int32). A slot of -1 is skipped; two
    tokens of one call must not name the same slot."""
    if _launch.fast is not None:
        done = _launch.fast.store(k, v, pages, slots)
        if done is not None:
            return None if done is True else _native.check(done, "klab_kv_store")
    shape, dtype = k.shape, k.dtype
    if len(shape) != 3 or v.shape != shape or dtype not in _DT or v.dtype is not dtype:
        raise ValueError("Expected k and v [tokens, kv_heads, head_dim] in BF16 or FP16")
    tokens, heads, dim = shape
    num_pages, kv_heads, page_size = _check_pages(pages, dim)
    if heads != kv_heads or tokens <= 0:
        raise ValueError("k and v must have the pages' kv_heads and at least one token")
    if tokens * heads * dim >= 2 ** 31:
        raise ValueError("Too many values for one call")
    device = pages.device
    if slots.dtype is not torch.int32 or slots.shape != (tokens,) or not slots.is_contiguous() or slots.device != device:
        raise ValueError(f"slots must be a contiguous int32 tensor with one entry per token on {device}")
    ks, kh, kd = k.stride()
    vs, vh, vd = v.stride()
    if tokens == 1 or heads == 1:  # a stride that is never taken may be anything
        ks, vs = (ks, vs) if tokens > 1 else (0, 0)
        kh, vh = (kh, vh) if heads > 1 else (0, 0)
    kp, vp, pp = k.data_ptr(), v.data_ptr(), pages.data_ptr()
    if kd != 1 or vd != 1 or (ks | vs | kh | vh) & 3 or (kp | vp) & 7 or k.device != device or v.device != device:
        raise ValueError("k and v need contiguous dims, strides of multiples of 4 and 8-byte alignment on the pages' device")
    _disjoint(pages, k, v, slots)
    _check_device(device, k, v)
    launch("klab_kv_store", ready(device),
           (kp, vp, _DT[dtype], ks, vs, kh, vh, pp, slots.data_ptr(), tokens, num_pages, page_size, kv_heads, dim),
           (k, v, pages, slots))


def read(pages, slots, head_dim, dtype=torch.bfloat16):
    """(k, v) [tokens, kv_heads, head_dim] as held at slots [tokens]: (code - 8) * scale, rounded once to dtype (float32:
    exact). Zeros for a slot of -1."""
    if _launch.fast is not None:
        rows = _launch.fast.read(pages, slots, head_dim, _ODT.get(dtype))
        if rows is not None:
            return rows if type(rows) is tuple else _native.check(rows, "klab_kv_read")
    num_pages, kv_heads, page_size = _check_pages(pages, head_dim)
    device = pages.device
    if dtype not in _ODT or slots.ndim != 1 or slots.numel() <= 0:
        raise ValueError("Expected slots=[tokens] and a dtype of float32, bfloat16 or float16")
    if slots.dtype is not torch.int32 or not slots.is_contiguous() or slots.device != device:
        raise ValueError(f"slots must be a contiguous int32 tensor on {device}")
    tokens = slots.numel()
    if tokens * kv_heads * head_dim >= 2 ** 31:
        raise ValueError("Too many values for one call")
    _check_device(device)
    index = ready(device)
    k = torch.empty(tokens, kv_heads, head_dim, device=device, dtype=dtype)
    v = torch.empty_like(k)
    launch("klab_kv_read", index,
           (pages.data_ptr(), slots.data_ptr(), k.data_ptr(), v.data_ptr(), _ODT[dtype], tokens, num_pages, page_size,
            kv_heads, head_dim), (pages, slots))
    return k, v


@lru_cache(maxsize=256)
def _scratch_bytes(index, *shape):
    """klab_kv_attention_scratch of these shapes on device `index` (the grid depends on its SM count)."""
    with torch.cuda.device(index):
        need = _native.lib().klab_kv_attention_scratch(*shape)
    if need < 0:
        _native.check(int(need), "klab_kv_attention_scratch")
    return int(need)


def attention(q, pages, table, lengths, starts, *, max_new=1, scale=None, out=None):
    """softmax(scale * q K^T) V of each request's new tokens over its pages.

    q [tokens, heads, head_dim] (BF16 or FP16, any token stride that is a multiple of 8 elements): request i's rows are
    starts[i] .. starts[i+1], at most max_new (<= 16) of them, the last of its lengths[i] tokens; token j of n sees positions
    below lengths[i] - n + j + 1, and a row that sees none gives zeros. scale defaults to 1 / sqrt(head_dim). Rows of q
    that belong to no request (a padded batch's) leave their rows of a given `out` as they were; in a new result they are
    zeros.
    """
    if _launch.fast is not None:
        done = _launch.fast.attention(q, pages, table, lengths, starts, max_new, scale, out)
        if done is not None:
            return done if type(done) is not int else _native.check(done, "klab_kv_attention")
    shape, dtype = q.shape, q.dtype
    if len(shape) != 3 or dtype not in _DT:
        raise ValueError("Expected q [tokens, heads, head_dim] in BF16 or FP16")
    tokens, heads, dim = shape
    num_pages, kv_heads, page_size = _check_pages(pages, dim)
    device = pages.device
    token_stride, head_stride, dim_stride = q.stride()
    qp = q.data_ptr()
    if tokens <= 0 or dim_stride != 1 or (heads > 1 and head_stride != dim) or (tokens > 1 and token_stride % 8) or qp % 16 \
            or q.device != device:
        raise ValueError("q needs contiguous heads, a token stride of a multiple of 8 and 16-byte alignment on the pages' device")
    if heads % kv_heads or heads // kv_heads > MAX_GROUP:
        raise ValueError(f"heads must be a multiple of kv_heads, at most {MAX_GROUP} each")
    for t in (table, lengths, starts):
        if t.dtype is not torch.int32 or not t.is_contiguous() or t.device != device:
            raise ValueError(f"table, lengths and starts must be contiguous int32 tensors on {device}")
    if table.ndim != 2 or lengths.shape != table.shape[:1] or starts.numel() != table.shape[0] + 1:
        raise ValueError("Expected table=[requests, width], lengths=[requests], starts=[requests + 1]")
    requests, width = table.shape
    if min(requests, width) <= 0 or requests > MAX_REQUESTS or width * page_size >= 2 ** 31:
        raise ValueError(f"From 1 to {MAX_REQUESTS} requests and fewer than 2^31 positions")
    if max_new is True or not 1 <= max_new <= MAX_NEW:
        raise ValueError(f"max_new must be from 1 to {MAX_NEW}")
    if scale is None:
        scale = dim ** -0.5
    elif not 0.0 < scale < math.inf:
        raise ValueError("scale must be positive and finite")
    _check_device(device, q)
    if out is not None:
        if out.dtype is not dtype or out.device != device or out.shape != shape or not out.is_contiguous() \
                or out.data_ptr() % 16 or out.requires_grad:
            raise ValueError("out must be contiguous, 16-byte aligned, of q's shape, dtype and device")
        _disjoint(out, q, pages, table, lengths, starts)
        name, tensors = "klab_kv_attention", (q, pages, table, lengths, starts, out)
    else:
        out = torch.empty(tokens, heads, dim, device=device, dtype=dtype)
        name, tensors = "klab_kv_attention_new", (q, pages, table, lengths, starts)
    index = ready(device)
    # Scratch of this call alone: a captured graph keeps its own, and nothing has to be zero in it.
    need = _scratch_bytes(index, requests, width, page_size, heads, kv_heads, dim, max_new)
    scratch = torch.empty(need, device=device, dtype=torch.uint8)
    launch(name, index,
           (qp, token_stride if tokens > 1 else 0, _DT[dtype], pages.data_ptr(), table.data_ptr(), lengths.data_ptr(),
            starts.data_ptr(), out.data_ptr(), scratch.data_ptr(), need, tokens, requests, width, num_pages, page_size, heads,
            kv_heads, dim, max_new, scale), tensors)
    return out
