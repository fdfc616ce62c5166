"""64-bit restatement of the batched 4-bit page cache (klab_b200.kv_pages): quantisation, the order of the bytes,
page tables, and attention with the sums that error bounds are built from."""

from __future__ import annotations

import numpy as np

GROUP, BLOCK = 32, 16


def quantize(x):
    """x [..., dim] float64 -> (codes 1..15 [..., dim], scales float64 [..., dim / 32])."""
    g = np.where(np.isnan(x), 0.0, x).reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    with np.errstate(over="ignore"):
        scale = np.minimum(np.abs(g).max(-1, initial=0.0) / 7, 65504.0).astype(np.float16).astype(np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        code = np.where(scale[..., None] > 0, np.clip(np.rint(g / scale[..., None]), -7, 7), 0.0) + 8
    return code.astype(np.int64).reshape(x.shape), scale


def values(codes, scales):
    g = (codes.reshape(*scales.shape, GROUP) - 8) * scales[..., None]
    return g.reshape(codes.shape)


def pack_block(k_codes, k_scales, v_codes, v_scales):
    """The bytes of one block of 16 tokens: codes [16, dim], scales [16, dim / 32] (float16 values)."""
    dim = k_codes.shape[1]
    ng = dim // GROUP
    q = min(ng, 4)
    out = np.zeros(18 * dim, np.uint8)
    words = out[:16 * dim].view("<u4")
    scale = out[16 * dim:].view("<f2")
    for r in range(BLOCK):
        for d in range(dim):
            group, w = d // 32, d % 32
            quad, inner = group // q, group % q
            t = w // 8
            words[quad * 64 * q + (r * 4 + t) * q + inner] |= np.uint32(int(k_codes[r, d]) << 4 * (w % 8))
            g = w // 4
            at = 2 * dim + quad * 64 * q + ((r // 8 * 8 + g) * 4 + r % 8 // 2) * q + inner
            words[at] |= np.uint32(int(v_codes[r, d]) << (4 * (w % 4) + 16 * (r % 2)))
        for group in range(ng):
            scale[r * ng + group] = k_scales[r, group]
            scale[16 * ng + ((r // 8 * 4 + r % 8 // 2) * ng + group) * 2 + r % 2] = v_scales[r, group]
    return out


def build_step(new, lengths, table, free, count, page, most):
    """The step by loops: (dict of outputs, table after)."""
    new, lengths, table = (np.array(x, np.int64) for x in (new, lengths, table))
    n = len(new)
    bad = 0
    for i in range(n):
        if new[i] < 0 or lengths[i] < 0:
            bad = max(bad, 1)
        elif -(-(lengths[i] + new[i]) // page) > table.shape[1]:
            bad = max(bad, 2)
    fresh = 0 if bad else int(sum(-(-(lengths[i] + new[i]) // page) - -(-lengths[i] // page) for i in range(n)))
    if not bad and new.sum() > most:
        bad = 4
    elif not bad and (not 0 <= count <= len(free) or fresh > count):
        bad = 3
    out = {"slots": np.full(most, -1), "positions": np.zeros(most, np.int64), "rows": np.full(most, -1),
           "starts": np.zeros(n + 1, np.int64), "lengths": lengths.copy(), "free_count": np.array([count]),
           "result": np.array([bad])}
    if bad:
        return out, table
    x = 0
    for i in range(n):
        out["starts"][i] = x
        for position in range(lengths[i], lengths[i] + new[i]):
            if position % page == 0:
                count -= 1
                table[i, position // page] = free[count]
            out["slots"][x] = table[i, position // page] * page + position % page
            out["positions"][x], out["rows"][x] = position, i
            x += 1
        out["lengths"][i] += new[i]
    out["starts"][n], out["free_count"][0] = x, count
    return out, table


def attention(q, k, v, new, scale):
    """One request: q [new, heads, dim], k, v [length, kv_heads, dim], float64. Returns (out, sum of softmax |v|)."""
    length, kvh, dim = k.shape
    heads = q.shape[1]
    out, size = np.zeros(q.shape), np.zeros(q.shape)
    for j in range(new):
        seen = max(0, length - new + j + 1)
        if not seen:
            continue
        s = np.einsum("hgd,phd->hgp", q[j].reshape(kvh, heads // kvh, dim), k[:seen]) * scale
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        out[j] = np.einsum("hgp,phd->hgd", p, v[:seen]).reshape(heads, dim)
        size[j] = np.einsum("hgp,phd->hgd", p, np.abs(v[:seen])).reshape(heads, dim)
    return out, size


def adapter_delta(x, a, b, c, ids):
    """c_a * (x A_a^T) B_a^T per row, float64; and the same with absolute values (for error bounds)."""
    out, size = np.zeros((len(x), b.shape[1])), np.zeros((len(x), b.shape[1]))
    for m, i in enumerate(ids):
        if i >= 0:
            out[m] = c[i] * (b[i] @ (a[i] @ x[m]))
            size[m] = abs(c[i]) * (np.abs(b[i]) @ (np.abs(a[i]) @ np.abs(x[m])))
    return out, size
