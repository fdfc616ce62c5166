"""Cases of the operators of a batched decode step: pages of requests (kv_pages.build_step), rows into 4-bit pages and
back (kv_pages.store, kv_pages.read), attention over those pages (kv_pages.attention) and low-rank adapters of many
requests beside a shared projection (adapters.adapter_linear).

A page is uint8 [kv_heads, bytes] of blocks of 16 tokens; a block holds, for NG = head_dim / 32 groups in quads of at
most Q = 4 and with r = token mod 16,
  K codes   16-bit pieces of 4 dims: 32-bit word [quad][r][t][group in quad] = dims 32 G + 8 t .. + 7, low nibble first
  V codes   16-bit pieces of 4 dims: 32-bit word [quad][r div 8][g][(r mod 8) div 2][group in quad] = dims
            32 G + 4 g .. + 3 of token r (r even: low half) and of its neighbour (high half)
  K scales  fp16 [r][G]
  V scales  fp16 [r div 8][(r mod 8) div 2][G][r mod 2]
and a value is (code - 8) * scale.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------- cases

def listed():
    return [
        # Eight requests that each add one token: what every decode step asks first. Launch latency.
        {"name": "tables_decode_8", "op": "tables", "requests": 8, "longest": 4096, "prompts": 0, "page": 16, "short": False},
        # A full scheduler: 1024 rows, a tenth of them with prompts of up to 2048 tokens.
        {"name": "tables_prompts_1024", "op": "tables", "requests": 1024, "longest": 8192, "prompts": 2048, "page": 64,
         "short": False},
        # The rows of one decode step of 16 requests, slices of one fused QKV result, written and read back.
        {"name": "store_decode_16", "op": "store", "tokens": 16, "pad": 2, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "dtype": "bf16", "back": "fp32"},
        # A prompt of 16384 tokens put into pages and read back for a 16-bit attention.
        {"name": "store_prompt_16k", "op": "store", "tokens": 16384, "pad": 0, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "dtype": "bf16", "back": "bf16"},
        # One request with a short cache and heads of 64, as the single-sequence attention serves it.
        {"name": "attend_1x300", "op": "attend", "requests": 1, "longest": 300, "new": 1, "heads": 32, "kv_heads": 8, "dim": 64,
         "page": 16, "dtype": "bf16"},
        # Sixteen requests of uneven lengths, one token each: an ordinary decode step.
        {"name": "attend_16x4k", "op": "attend", "requests": 16, "longest": 4096, "new": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "dtype": "bf16"},
        # Eight requests that check up to five drafted tokens each; seven query heads a kv head, FP16.
        {"name": "attend_drafts_8x2k", "op": "attend", "requests": 8, "longest": 2047, "new": 5, "heads": 28, "kv_heads": 4,
         "dim": 128, "page": 32, "dtype": "fp16"},
        # One very long document: the split over the cache's length.
        {"name": "attend_1x131072", "op": "attend", "requests": 1, "longest": 131072, "new": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "dtype": "bf16"},
        # A full machine: 64 requests of up to 8192 tokens.
        {"name": "attend_64x8k", "op": "attend", "requests": 64, "longest": 8192, "new": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "dtype": "bf16"},
        # One request's token through the query projection with its adapter.
        {"name": "adapter_bf16_m1", "op": "adapter", "weights": "bf16", "tokens": 1, "n": 4096, "k": 4096, "rank": 16,
         "adapters": 8},
        # Eight requests, INT8 weights of the gate projection, adapters of rank 16.
        {"name": "adapter_int8_m8", "op": "adapter", "weights": "int8", "tokens": 8, "n": 14336, "k": 4096, "rank": 16,
         "adapters": 32},
        # Sixteen requests, BF16 weights of the down projection, adapters of rank 64.
        {"name": "adapter_bf16_m16", "op": "adapter", "weights": "bf16", "tokens": 16, "n": 4096, "k": 14336, "rank": 64,
         "adapters": 32},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("tables", "store", "attend", "attend", "attend", "adapter", "adapter"))
    if op == "tables":
        return {"op": op, "requests": _spread(rng, 1, 1024), "longest": _spread(rng, 1, 8192),
                "prompts": rng.choice((0, _spread(rng, 2, 2048))), "page": rng.choice((16, 32, 64)), "short": rng.random() < 0.1}
    if op == "store":
        kv = rng.choice((1, 2, 4, 5, 8))
        return {"op": op, "tokens": _spread(rng, 1, 16384), "pad": rng.randrange(4), "heads": kv * rng.randint(1, 8),
                "kv_heads": kv, "dim": rng.choice((64, 128, 256)) if kv <= 4 else rng.choice((64, 128)),
                "page": rng.choice((16, 32, 64)), "dtype": rng.choice(("bf16", "fp16")), "back": rng.choice(("fp32", "bf16"))}
    if op == "attend":
        kv = rng.choice((1, 2, 4, 5, 8))
        requests = _spread(rng, 1, 64)
        return {"op": op, "requests": requests, "longest": _spread(rng, 1, 131072 // max(1, requests // 4)),
                "new": rng.choice((1, 1, 1, 2, 3, 4, 8)), "heads": kv * rng.choice((1, 2, 3, 4, 6, 7, 8, 16)), "kv_heads": kv,
                "dim": rng.choice((64, 128, 128, 256)) if kv <= 4 else rng.choice((64, 128)), "page": rng.choice((16, 32, 64)),
                "dtype": rng.choice(("bf16", "bf16", "fp16"))}
    return {"op": op, "weights": rng.choice(("bf16", "int8", "fp4")), "tokens": _spread(rng, 1, 16),
            "n": rng.choice((1000, 1024, 2048, 4096, 8192, 14336)), "k": 64 * rng.choice((16, 29, 32, 64, 77, 128)),
            "rank": rng.choice((8, 16, 24, 32, 64)), "adapters": _spread(rng, 1, 64)}


# ---------------------------------------------------------------- inputs

def _lengths(case):
    """Cached and new tokens of each request, from the case alone (the seed orders them)."""
    pick = np.random.RandomState(case["requests"] * 131 + case["longest"])
    n = case["requests"]
    total = np.exp(pick.uniform(math.log(max(1, case["longest"] / 16)), math.log(case["longest"]), n)).astype(np.int64)
    total = np.maximum(1, total)
    total[0] = case["longest"]
    if case["op"] == "attend":
        new = np.minimum(total, pick.randint(1, case["new"] + 1, n))
        new[0] = min(case["longest"], case["new"])
        return total - new, new
    cached = total - 1
    new = np.ones(n, np.int64)
    if case["prompts"]:
        begin = pick.rand(n) < 0.1
        begin[0] = True
        new = np.where(begin, pick.randint(1, case["prompts"] + 1, n), new)
        cached = np.where(begin, 0, cached)
    else:
        new[pick.rand(n) < 0.05] = 0  # a request that waits
    return cached, new


def _dev(a, dtype=torch.int32):
    return torch.as_tensor(np.ascontiguousarray(a)).to(device=DEVICE, dtype=dtype)


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _normal(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dtype)


def _places(slots, kv_heads, dim, page):
    """Where a token's K pieces, V pieces [T, heads, dim / 4], K scales and V scales [T, heads, dim / 32] stand, in 16-bit
    units from the start of the pages."""
    ng = dim // 32
    q = min(ng, 4)
    block = 16 * dim * 9 // 16  # 16-bit units of a block
    slots = slots.long()
    number = slots // page * kv_heads
    head = torch.arange(kv_heads, device=slots.device)
    base = ((number[:, None] + head) * (page // 16) + (slots % page // 16)[:, None]) * block
    r = (slots % 16)[:, None, None]
    piece = torch.arange(dim // 4, device=slots.device)
    group, g = piece // 8, piece % 8
    quad, inner = group // q, group % q
    kp = quad * (128 * q) + r * (8 * q) + g // 2 * (2 * q) + inner * 2 + g % 2
    vp = 4 * dim + quad * (128 * q) + r // 8 * (64 * q) + g * (8 * q) + r % 8 // 2 * (2 * q) + inner * 2 + r % 2
    group = torch.arange(ng, device=slots.device)
    ks = 8 * dim + r * ng + group
    vs = 8 * dim + 16 * ng + (r // 8 * 4 + r % 8 // 2) * (2 * ng) + group * 2 + r % 2
    base = base[:, :, None]
    return base + kp, base + vp, base + ks, base + vs


def _codes(x):
    """4-bit pieces [T, heads, dim / 4] and scales [T, heads, dim / 32] of rows [T, heads, dim]."""
    t, h, d = x.shape
    x = x.float().reshape(t, h, d // 32, 32)
    x = torch.where(torch.isnan(x), torch.zeros_like(x), x)
    scale = (x.abs().amax(-1) / torch.tensor(7.0, device=x.device)).clamp_max(65504.0).to(torch.float16)
    s = scale.float().unsqueeze(-1)
    code = torch.where(s > 0, torch.round(x / s).clamp(-7, 7), torch.zeros_like(x)).to(torch.int32) + 8
    code = code.reshape(t, h, d // 4, 4)
    piece = code[..., 0] | code[..., 1] << 4 | code[..., 2] << 8 | code[..., 3] << 12
    return piece.to(torch.int16), scale


def _values(pages, slots, dim, page):
    """K and V rows [T, heads, dim] that the pages hold at these slots, in 32 bits."""
    heads = pages.shape[1]
    words = pages.view(torch.int16).reshape(-1)
    kp, vp, ks, vs = _places(slots, heads, dim, page)
    shift = torch.tensor([0, 4, 8, 12], device=pages.device, dtype=torch.int32)

    def rows(at, scale_at):
        code = (words[at].to(torch.int32).unsqueeze(-1) >> shift & 15) - 8
        scale = words[scale_at].view(torch.float16).float()
        return (code.float().reshape(*scale.shape, 32) * scale.unsqueeze(-1)).reshape(at.shape[0], heads, dim)

    return rows(kp, ks), rows(vp, vs)


def _put(pages, k, v, slots, page):
    """Rows into the pages, but for those whose slot is -1."""
    kp, vp, ks, vs = _places(slots.clamp_min(0), k.shape[1], k.shape[2], page)
    words = pages.view(torch.int16).reshape(-1)
    there = (slots >= 0)[:, None, None]
    for x, at, scale_at in ((k, kp, ks), (v, vp, vs)):
        piece, scale = _codes(x)
        words[at[there.expand_as(at)]] = piece[there.expand_as(piece)]
        words[scale_at[there.expand_as(scale_at)]] = scale.view(torch.int16)[there.expand_as(scale)]


def _paged(total, page, order, extra=0):
    """A table for these total lengths over pages in a shuffled order: (table, pages in use, all pages)."""
    held = -(-total // page)
    width = int(held.max()) + extra
    number = int(held.sum())
    ids = order.permutation(number + 1 + extra * len(total))
    table = np.full((len(total), max(1, width)), -1, np.int64)
    table[np.arange(table.shape[1])[None, :] < held[:, None]] = ids[:number]
    return table, ids[number:], len(ids)


def prepare(case, seed):
    order = np.random.RandomState(seed % (1 << 31))
    gen = _generator(seed)
    if case["op"] == "tables":
        cached, new = _lengths(case)
        at = order.permutation(len(cached))
        cached, new = cached[at], new[at]
        page = case["page"]
        held, need = -(-cached // page), -(-(cached + new) // page)
        extra = int((need - held).sum())
        ids = order.permutation(int(held.sum()) + extra + 7)
        table = np.full((len(cached), int(need.max()) + 4), -1, np.int64)
        table[np.arange(table.shape[1])[None, :] < held[:, None]] = ids[:int(held.sum())]
        free = np.full(len(ids), -1, np.int64)
        free[:extra + 7] = ids[int(held.sum()):]
        count = max(0, extra - 1) if case["short"] else extra + 7
        return {"case": case, "new": _dev(new), "lengths": _dev(cached), "table": _dev(table), "free": _dev(free),
                "count": _dev([count]), "most": int(new.sum()) + 5}
    if case["op"] == "store":
        t, pad, heads, kv, d, page = (case[x] for x in ("tokens", "pad", "heads", "kv_heads", "dim", "page"))
        number = -(-t // page) + 2
        slots = np.full(t + pad, -1, np.int64)
        table = order.permutation(number)
        token = np.arange(t) + order.randint(0, page)
        slots[:t] = table[token // page] * page + token % page
        qkv = _normal(gen, t + pad, (heads + 2 * kv) * d, dtype=DTYPES[case["dtype"]])
        pages = torch.zeros((number, kv, page * d * 9 // 8), device=DEVICE, dtype=torch.uint8)
        return {"case": case, "qkv": qkv, "slots": _dev(slots), "pages": pages}
    if case["op"] == "attend":
        cached, new = _lengths(case)
        at = order.permutation(len(cached))
        cached, new = cached[at], new[at]
        page, kv, d = case["page"], case["kv_heads"], case["dim"]
        total = cached + new
        table, _, number = _paged(total, page, order)
        # What no token has written yet stays as the allocator left it: any bytes.
        pages = torch.randint(0, 256, (number, kv, page * d * 9 // 8), generator=gen, device=DEVICE, dtype=torch.uint8)
        token = np.arange(int(total.sum())) - np.repeat(np.cumsum(total) - total, total)
        row = np.repeat(np.arange(len(total)), total)
        slots = _dev(table[row, token // page] * page + token % page, torch.int64)
        # Keys with a few strong channels and a mean of their own, values around zero.
        strength = torch.exp(0.5 * torch.randn((kv, d), generator=gen, device=DEVICE))
        mean = torch.randn((kv, d), generator=gen, device=DEVICE)
        part = max(1, (1 << 26) // (kv * d))
        for s in torch.split(slots, part):
            k = ((torch.randn((len(s), kv, d), generator=gen, device=DEVICE) + mean) * strength).to(DTYPES[case["dtype"]])
            _put(pages, k, _normal(gen, len(s), kv, d, dtype=DTYPES[case["dtype"]]), s, page)
        tokens = int(new.sum())
        qkv = _normal(gen, tokens, (case["heads"] + 2 * kv) * d, dtype=DTYPES[case["dtype"]])
        return {"case": case, "q": qkv[:, :case["heads"] * d].view(tokens, case["heads"], d), "pages": pages,
                "table": _dev(table), "lengths": _dev(total), "starts": _dev(np.concatenate([[0], np.cumsum(new)]))}
    m, n, k, r, count = (case[x] for x in ("tokens", "n", "k", "rank", "adapters"))
    ids = order.randint(0, count, m)
    if m > 2:
        ids[order.randint(0, m)] = -1  # a request without an adapter
    state = {"case": case, "x": _normal(gen, m, k), "a": _normal(gen, count, r, k) * 0.02, "b": _normal(gen, count, n, r) * 0.02,
             "c": torch.rand(count, generator=gen, device=DEVICE) + 0.5, "ids": _dev(ids)}
    if case["weights"] == "bf16":
        state["w"] = _normal(gen, n, k) * 0.02
    elif case["weights"] == "int8":
        state["w"] = (torch.randn((n, k), generator=gen, device=DEVICE) * 40).round().clamp(-127, 127).to(torch.int8)
        state["s"] = torch.rand(n, generator=gen, device=DEVICE) * 4e-4 + 4e-4
    else:
        state["w"] = torch.randint(0, 256, (n, k // 2), generator=gen, device=DEVICE, dtype=torch.uint8)
        state["s"] = (torch.rand((n, k // 32), generator=gen, device=DEVICE) * 5e-3 + 5e-3).to(torch.float16)
    return state


# ---------------------------------------------------------------- plain forms

def _plain_tables(s):
    page, most = s["case"]["page"], s["most"]
    new, lengths, table, free, count = (s[x].long() for x in ("new", "lengths", "table", "free", "count"))
    held, need = (lengths + page - 1) // page, (lengths + new + page - 1) // page
    fresh = need - held
    good = ((new >= 0) & (lengths >= 0)).all() & (fresh.sum() <= count[0]) & (need <= table.shape[1]).all() & (new.sum() <= most)
    before = torch.cumsum(fresh, 0) - fresh
    p = torch.arange(table.shape[1], device=table.device)
    given = (p >= held[:, None]) & (p < need[:, None]) & good
    which = count[0] - 1 - (before[:, None] + p - held[:, None])
    table = torch.where(given, free[which.clamp(0, len(free) - 1)], table)
    starts = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0)]) * good
    token = torch.arange(most, device=table.device)
    row = torch.searchsorted(starts[1:], token, right=True)
    there = row < len(new)
    at = row.clamp_max(len(new) - 1)
    position = torch.where(there, lengths[at] + token - starts[at], torch.zeros_like(token))
    slot = table[at, (position // page).clamp_max(table.shape[1] - 1)] * page + position % page
    minus = torch.full_like(token, -1)
    return {k: v.to(torch.int32) for k, v in {
        "slots": torch.where(there, slot, minus), "positions": position, "rows": torch.where(there, row, minus), "starts": starts,
        "lengths": torch.where(good, lengths + new, lengths), "free_count": torch.where(good, count - fresh.sum(), count),
        "table": table}.items()}


def _qkv(s):
    heads, kv, d = (s["case"][x] for x in ("heads", "kv_heads", "dim"))
    t = s["qkv"].shape[0]
    return s["qkv"][:, heads * d:(heads + kv) * d].view(t, kv, d), s["qkv"][:, (heads + kv) * d:].view(t, kv, d)


def _plain_store(s):
    k, v = _qkv(s)
    page, back = s["case"]["page"], DTYPES[s["case"]["back"]]
    _put(s["pages"], k, v, s["slots"], page)
    k, v = _values(s["pages"], s["slots"].clamp_min(0), k.shape[2], page)
    there = (s["slots"] >= 0)[:, None, None]
    return {"k": (k * there).to(back), "v": (v * there).to(back)}


def _plain_attend(s):
    case, q = s["case"], s["q"]
    page, kv, d, most = case["page"], case["kv_heads"], case["dim"], case["new"]
    table, lengths, starts = s["table"].long(), s["lengths"].long(), s["starts"].long()
    requests, width = table.shape
    slots = (table.clamp_min(0)[:, :, None] * page + torch.arange(page, device=q.device)).reshape(-1)
    k, v = (x.view(requests, width * page, kv, d) for x in _values(s["pages"], slots, d, page))
    new = starts[1:] - starts[:-1]
    j = torch.arange(most, device=q.device)
    rows = q.float()[(starts[:-1, None] + j).clamp_max(q.shape[0] - 1)].view(requests, most, kv, -1, d)
    score = torch.einsum("rnhgd,rphd->rhgnp", rows, k) / math.sqrt(d)
    p = torch.arange(width * page, device=q.device)
    seen = p < (lengths - new)[:, None, None] + j[:, None] + 1
    seen = (seen & (p < lengths[:, None, None]))[:, None, None]
    score = torch.where(seen, score, torch.full_like(score, -math.inf))
    top = score.amax(-1, keepdim=True)
    weight = torch.where(seen, torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top)), torch.zeros_like(score))
    v = torch.where((p < lengths[:, None])[:, :, None, None], v, torch.zeros_like(v))
    out = torch.einsum("rhgnp,rphd->rnhgd", weight / weight.sum(-1, keepdim=True).clamp_min(1e-38), v)
    token = torch.arange(q.shape[0], device=q.device)
    row = torch.searchsorted(starts[1:], token, right=True)
    return out.reshape(requests, most, -1, d)[row, token - starts[row]].to(q.dtype)


def _weights(s):
    if s["case"]["weights"] == "bf16":
        return s["w"].float()
    if s["case"]["weights"] == "int8":
        return s["w"].float() * s["s"][:, None]
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=s["w"].device)
    codes = torch.stack((s["w"] & 15, s["w"] >> 4), -1).reshape(s["w"].shape[0], -1, 32)
    return (table[codes.long()] * s["s"].float()[:, :, None]).reshape(s["w"].shape[0], -1)


def _plain_adapter(s):
    x, ids = s["x"].float(), s["ids"].long()
    at = ids.clamp_min(0)
    small = torch.bmm(s["a"][at].float(), x[:, :, None])
    more = torch.bmm(s["b"][at].float(), small)[:, :, 0] * s["c"][at][:, None]
    return (x @ _weights(s).T + torch.where((ids >= 0)[:, None], more, torch.zeros_like(more))).to(torch.bfloat16)


# ---------------------------------------------------------------- the framework's calls

def _own_tables(s):
    from klab_b200 import kv_pages

    step = kv_pages.build_step(s["new"], s["lengths"], s["table"], s["free"], s["count"], page_size=s["case"]["page"],
                               max_tokens=s["most"])
    return {"slots": step.slots, "positions": step.positions, "rows": step.rows, "starts": step.starts, "lengths": step.lengths,
            "free_count": step.free_count, "table": s["table"]}


def _own_store(s):
    from klab_b200 import kv_pages

    k, v = _qkv(s)
    kv_pages.store(k, v, s["pages"], s["slots"])
    k, v = kv_pages.read(s["pages"], s["slots"], k.shape[2], dtype=DTYPES[s["case"]["back"]])
    return {"k": k, "v": v}


def _own_attend(s):
    from klab_b200 import kv_pages

    return kv_pages.attention(s["q"], s["pages"], s["table"], s["lengths"], s["starts"], max_new=s["case"]["new"])


def _own_adapter(s):
    from klab_b200 import adapters, fp4, int8_weights

    kind = s["case"]["weights"]
    w = s["w"] if kind == "bf16" else int8_weights.Int8Weights(s["w"], s["s"]) if kind == "int8" else fp4.FP4F16Weights(s["w"], s["s"])
    return adapters.adapter_linear(s["x"], w, s["a"], s["b"], s["c"], s["ids"])


def run(state):
    op = state["case"]["op"]
    if own:
        return {"tables": _own_tables, "store": _own_store, "attend": _own_attend, "adapter": _own_adapter}[op](state)
    return {"tables": _plain_tables, "store": _plain_store, "attend": _plain_attend, "adapter": _plain_adapter}[op](state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["op"] == "tables":
        cached, new = _lengths(case)
        fresh = -(-(cached + new) // case["page"]) + -cached // case["page"]
        return {"bytes": 4 * (4 * len(cached) + 1) + 12 * int(new.sum()) + 8 * int(np.maximum(0, fresh).sum()) + 8, "flops": 0}
    if case["op"] == "store":
        values = 2 * case["tokens"] * case["kv_heads"] * case["dim"]
        packed = values * 9 // 16
        return {"bytes": 2 * values + packed + packed + (4 if case["back"] == "fp32" else 2) * values + 8 * case["tokens"], "flops": 0}
    if case["op"] == "attend":
        cached, new = _lengths(case)
        d, total = case["dim"], cached + new
        seen = int((new * cached + new * (new + 1) // 2).sum())
        return {"bytes": int(total.sum()) * case["kv_heads"] * d * 9 // 8 + 4 * int(new.sum()) * case["heads"] * d
                + 4 * int((-(-total // case["page"])).sum()) + 8 * len(total), "flops": 4 * seen * case["heads"] * d}
    m, n, k, r = (case[x] for x in ("tokens", "n", "k", "rank"))
    stored = {"bf16": 2 * n * k, "int8": n * k + 4 * n, "fp4": n * k // 2 + n * k // 16}[case["weights"]]
    used = case["adapters"] * (1 - (1 - 1 / case["adapters"]) ** m)  # distinct adapters that m draws meet
    return {"bytes": int(stored + 2 * m * (k + n) + used * 2 * r * (n + k) + 4 * m), "flops": 2 * m * n * k + 2 * m * r * (n + k)}


# ---------------------------------------------------------------- in 64 bits

def _block_values(pages, dim):
    """Every value of the pages as float64 (k, v) [page, head, token of the page, dim], block by block."""
    number, heads, size = pages.shape
    ng, blocks = dim // 32, size // (18 * dim)
    q = min(ng, 4)
    raw = pages.reshape(number, heads, blocks, 18 * dim)
    kc, vc, ks, vs = torch.split(raw, [8 * dim, 8 * dim, 32 * ng, 32 * ng], dim=-1)

    def nibbles(x):
        return torch.stack((x & 15, x >> 4), -1).flatten(-2).double() - 8

    def halves(x):
        return x.contiguous().view(torch.float16).double()

    lead = (number, heads, blocks)
    k = nibbles(kc).reshape(*lead, ng // q, 16, 4, q, 8).permute(0, 1, 2, 4, 3, 6, 5, 7).reshape(*lead, 16, ng, 32)
    k = k * halves(ks).reshape(*lead, 16, ng, 1)
    # [quad][r div 8][g][pair][group][r mod 2][dim of 4] -> [r][group][g][dim]
    v = nibbles(vc).reshape(*lead, ng // q, 2, 8, 4, q, 2, 4).permute(0, 1, 2, 4, 6, 8, 3, 7, 5, 9).reshape(*lead, 16, ng, 32)
    v = v * halves(vs).reshape(*lead, 2, 4, ng, 2).permute(0, 1, 2, 3, 4, 6, 5).reshape(*lead, 16, ng, 1)
    return (x.reshape(number, heads, blocks * 16, dim) for x in (k, v))


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "tables":
        return None  # whole numbers: the plain form has them
    if case["op"] == "store":
        heads, kv, d = case["heads"], case["kv_heads"], case["dim"]
        rows = s["qkv"].double().reshape(len(s["qkv"]), -1, 32)
        scale = (rows.abs().amax(-1, keepdim=True) / 7).clamp(max=65504).to(torch.float16).double()
        held = torch.where(scale > 0, torch.round(rows / scale.clamp_min(1e-30)).clamp(-7, 7) * scale, 0.0)
        held = held.reshape(len(rows), heads + 2 * kv, d) * (s["slots"] >= 0)[:, None, None]
        return {"k": held[:, heads:heads + kv], "v": held[:, heads + kv:]}
    if case["op"] == "attend":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        lengths, starts, group = s["lengths"].tolist(), s["starts"].tolist(), case["heads"] // case["kv_heads"]
        for i, length in enumerate(lengths):
            ids = s["table"][i, :-(-length // case["page"])].long()
            k, v = (x.transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"])[:length] for x in _block_values(s["pages"][ids], case["dim"]))
            for j in range(starts[i + 1] - starts[i]):
                seen = length - (starts[i + 1] - starts[i]) + j + 1
                q = s["q"][starts[i] + j].double().view(case["kv_heads"], group, case["dim"])
                p = torch.softmax(q @ k[:seen].permute(1, 2, 0) * case["dim"] ** -0.5, -1)
                out[starts[i] + j] = (p @ v[:seen].transpose(0, 1)).reshape(-1, case["dim"])
        return out
    x = s["x"].double()
    if case["weights"] == "fp4":
        sign = 1 - 2 * (torch.stack((s["w"] >> 3 & 1, s["w"] >> 7), -1).double())
        low = torch.stack((s["w"] & 7, s["w"] >> 4 & 7), -1).double()
        size = torch.where(low < 2, low / 2, (1 + low % 2 / 2) * 2 ** (torch.div(low, 2, rounding_mode="floor") - 1))
        w = (sign * size).reshape(len(s["w"]), -1, 32) * s["s"].double()[:, :, None]
        w = w.reshape(len(s["w"]), -1)
    else:
        w = s["w"].double() if case["weights"] == "bf16" else s["w"].double() * s["s"].double()[:, None]
    y = x @ w.T
    for m, a in enumerate(s["ids"].tolist()):
        if a >= 0:
            y[m] += s["c"][a].double() * (s["b"][a].double() @ (s["a"][a].double() @ x[m]))
    return y
