"""Batched 4-bit pages on the GPU against the 64-bit oracle: page tables, rows into pages and back, attention, and a run
of them together under one captured graph."""

import numpy as np
import pytest
import torch

from oracle import kv_pages as ok

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(autouse=True)
def native():
    from klab_b200 import _native

    _native.lib()
    assert _native.device_status(clear=True) == 0
    yield _native
    assert _native.device_status(clear=True) == 0


def i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).cuda()


def f64(t):
    return t.double().cpu().numpy()


# ---------------------------------------------------------------- tables

def table_state(rng, lengths, page, spare, slack=2, extra=0):
    """(table, free stack, free count) for these lengths; pages in a shuffled order."""
    held = -(-np.asarray(lengths) // page)
    ids = rng.permutation(int(held.sum()) + spare)
    table = np.full((len(lengths), int(held.max(initial=0)) + slack), -1)
    at = 0
    for i, n in enumerate(held):
        table[i, :n] = ids[at:at + n]
        at += n
    free = np.full(len(ids) + extra, -1)
    free[:spare] = ids[at:]
    return table, free, spare


STEPS = [([0], [1], 16, 4, 5), ([15, 16, 17, 0], [1, 1, 1, 1], 16, 9, 4), ([5, 0, 31, 64], [0, 0, 0, 0], 32, 0, 3),
         ([0] * 3, [100, 1, 0], 16, 12, 120), ([1000, 3, 77], [1, 5000, 1], 64, 90, 5100),
         (list(range(0, 2000, 7)), [3] * 286, 16, 286, 858), ([1] * 1500, [1] * 1500, 16, 10, 1501),
         ([63] * 8192, [1, 2] * 4096, 64, 4200, 12300)]


@pytest.mark.parametrize("lengths,new,page,spare,most", STEPS, ids=[str(i) for i in range(len(STEPS))])
@pytest.mark.parametrize("inplace", [False, True])
def test_step_matches_oracle(lengths, new, page, spare, most, inplace):
    from klab_b200 import kv_pages

    rng = np.random.default_rng(len(lengths))
    width = -(-max(a + b for a, b in zip(lengths, new)) // page) + 1
    table, free, count = table_state(rng, lengths, page, spare, slack=0)
    table = np.pad(table, ((0, 0), (0, width - table.shape[1])), constant_values=-1)
    want, table_after = ok.build_step(new, lengths, table, free, count, page, most)
    assert want["result"] == 0
    t, ln, fc = i32(table), i32(lengths), i32([count])
    step = kv_pages.build_step(i32(new), ln, t, i32(free), fc, page_size=page, max_tokens=most, inplace=inplace)
    for name, value in want.items():
        assert np.array_equal(getattr(step, name).cpu().numpy(), value), name
    assert np.array_equal(t.cpu().numpy(), table_after)
    if inplace:
        assert step.lengths is ln and step.free_count is fc
    else:
        assert ln.tolist() == list(lengths) and fc.item() == count


@pytest.mark.parametrize("change,result", [({"new": [1, -1, 1]}, 1), ({"lengths": [4, -5, 4]}, 1), ({"new": [70, 1, 1]}, 2),
                                           ({"spare": 1}, 3), ({"most": 33}, 4), ({"new": [2 ** 31 - 1] * 3}, 2)])
def test_step_refusals_change_nothing(native, change, result):
    from klab_b200 import kv_pages

    rng = np.random.default_rng(3)
    c = {"new": [30, 2, 2], "lengths": [30, 14, 16], "spare": 4, "most": 40, **change}
    table, free, count = table_state(rng, np.maximum(c["lengths"], 0), 16, c["spare"])
    t, ln = i32(table), i32(c["lengths"])
    step = kv_pages.build_step(i32(c["new"]), ln, t, i32(free), i32([count]), page_size=16, max_tokens=c["most"])
    assert step.result.item() == result and native.device_status(clear=True) == 5
    assert step.slots.eq(-1).all() and step.rows.eq(-1).all() and step.starts.eq(0).all()
    assert step.lengths.tolist() == c["lengths"] and step.free_count.item() == count
    assert np.array_equal(t.cpu().numpy(), table)


def test_step_and_release_keep_every_page(native):
    """Forty steps of requests that grow, end and begin again: each page is held once or free."""
    from klab_b200 import kv_pages

    rng = np.random.default_rng(5)
    page, pages, requests = 16, 200, 9
    lengths, table = i32([0] * requests), i32(np.full((requests, 30), -1))
    free, count = i32(rng.permutation(pages)), i32([pages])
    host = np.zeros(requests, np.int64)
    for _ in range(40):
        ended = rng.random(requests) < 0.15
        kv_pages.release(torch.from_numpy(ended).cuda(), lengths, table, free, count, page_size=page)
        host[ended] = 0
        new = rng.integers(0, 25, requests)
        new[host + new > 30 * page] = 0
        step = kv_pages.build_step(i32(new), lengths, table, free, count, page_size=page, max_tokens=300, inplace=True)
        assert step.result.item() == 0
        host += new
        assert lengths.tolist() == host.tolist()
        held = table.cpu().numpy()
        held = held[np.arange(30)[None, :] < -(-host // page)[:, None]]
        both = np.concatenate([held, free.cpu().numpy()[:count.item()]])
        assert sorted(both.tolist()) == list(range(pages))
    # A table entry that is no page: nothing is given back.
    table[0, 0] = pages
    lengths[0] = max(1, host[0])
    before = [x.clone() for x in (lengths, table, free, count)]
    kv_pages.release(torch.ones(requests, dtype=torch.bool, device="cuda"), lengths, table, free, count, page_size=page)
    torch.cuda.synchronize()
    assert native.device_status(clear=True) == 4
    assert all(torch.equal(a, b) for a, b in zip(before, (lengths, table, free, count)))


def test_step_with_a_bad_page_gives_no_slot(native):
    from klab_b200 import kv_pages

    table = i32([[7, 1, -1], [99, -1, -1]])
    step = kv_pages.build_step(i32([2, 2]), i32([20, 3]), table, i32([4, 5] + [0] * 8), i32([2]), page_size=16, max_tokens=4)
    torch.cuda.synchronize()
    assert native.device_status(clear=True) == 4
    assert step.slots.tolist() == [20, 21, -1, -1]


# ---------------------------------------------------------------- store and read

@pytest.mark.parametrize("dim,heads,page,dtype,tokens", [(128, 8, 16, "bf16", 1), (128, 2, 32, "bf16", 37), (64, 3, 64, "fp16", 50),
                                                         (256, 1, 16, "bf16", 19), (64, 1, 1024, "bf16", 5), (128, 5, 64, "fp16", 300)])
def test_store_and_read_match_the_format(dim, heads, page, dtype, tokens):
    from klab_b200 import kv_pages

    rng = np.random.default_rng(tokens)
    pages = tokens // page + 3
    slots = rng.permutation(pages * page)[:tokens]
    skip = rng.random(tokens) < 0.2
    skip[0] = False
    qkv = (torch.randn(tokens, (2 + 2 * heads) * dim, generator=torch.Generator().manual_seed(tokens)) * 3).to(DT[dtype])
    qkv[0, 2 * dim:2 * dim + 32] = 0
    if tokens > 4:
        qkv[1, 2 * dim] = float("inf")
        qkv[2, 2 * dim + 1] = float("nan")
        qkv[3, 2 * dim:] = qkv[3, 2 * dim:] * 2.0 ** -20   # subnormal scales
        qkv[4, 2 * dim:] = 7 * 0.5 ** torch.arange(2 * heads * dim).remainder(4)  # exact ties
    dev = qkv.cuda()
    k, v = dev[:, 2 * dim:(2 + heads) * dim].view(tokens, heads, dim), dev[:, (2 + heads) * dim:].view(tokens, heads, dim)
    buf = torch.randint(0, 256, (pages, heads, kv_pages.page_bytes(page, dim)), dtype=torch.uint8, device="cuda")
    before = buf.cpu().numpy().copy()
    kv_pages.store(k, v, buf, i32(np.where(skip, -1, slots)))
    codes, scales = zip(*(ok.quantize(f64(x)) for x in (k, v)))
    got = kv_pages.read(buf, i32(np.where(skip, -1, slots)), dim, dtype=torch.float32)
    for g, c, s in zip(got, codes, scales):
        want = ok.values(c, s)
        want[skip] = 0
        assert np.array_equal(f64(g), want)
    for dt in (torch.bfloat16, torch.float16):
        for g, exact in zip(kv_pages.read(buf, i32(np.where(skip, -1, slots)), dim, dtype=dt), got):
            assert torch.equal(g, exact.to(dt))
    # Every byte: the written tokens' codes and scales at their places, all others as they were.
    after = buf.cpu().numpy()
    for number in range(pages):
        for h in range(heads):
            for block in range(page // 16):
                mine = [(x, slots[x] % 16) for x in range(tokens) if not skip[x] and slots[x] // 16 == number * (page // 16) + block]
                held = np.zeros((4, 16, dim), np.int64)
                sc = np.zeros((2, 16, dim // 32))
                mask = np.zeros((16, dim), np.int64)
                for x, r in mine:
                    held[0, r], held[1, r], mask[r] = codes[0][x, h], codes[1][x, h], 15
                    sc[0, r], sc[1, r] = scales[0][x, h], scales[1][x, h]
                one = np.zeros((16, dim // 32))
                one[[r for _, r in mine]] = np.frombuffer(b"\xff\xff", "<f2")[0]
                bits = ok.pack_block(mask, one, mask, one)
                want = ok.pack_block(held[0], sc[0], held[1], sc[1])
                at = slice(block * 18 * dim, (block + 1) * 18 * dim)
                scale_bits = np.where(bits[16 * dim:] != 0, 255, 0)
                bits = np.concatenate([bits[:16 * dim], scale_bits]).astype(np.uint8)
                old, new = before[number, h, at], after[number, h, at]
                assert np.array_equal(new & ~bits, old & ~bits)
                assert np.array_equal(new & bits, want & bits)


@pytest.mark.parametrize("dim,heads,page,dtype,tokens", [(64, 9, 16, "bf16", 2049), (128, 8, 64, "fp16", 1025), (128, 9, 16, "bf16", 3641),
                                                         (128, 16, 64, "fp16", 2049), (256, 5, 32, "bf16", 3500)])
@pytest.mark.parametrize("order", ["runs", "shuffled", "backwards"])
def test_many_rows_give_what_few_rows_give(dim, heads, page, dtype, tokens, order):
    """One call over many rows against calls over 64: the same bytes, the same rows back."""
    from klab_b200 import kv_pages

    g = torch.Generator(device="cuda").manual_seed(tokens)
    pages = tokens // page + 3
    slots = torch.arange(3, tokens + 3, device="cuda", dtype=torch.int32)
    if order == "shuffled":
        slots = torch.randperm(pages * page, device="cuda", generator=g)[:tokens].int()
    elif order == "backwards":
        slots = slots.flip(0).contiguous()
    slots[torch.rand(tokens, device="cuda", generator=g) < 0.05] = -1
    # Rows on 16 bytes, and (of heads of an odd number) on 8: both ways to load.
    for pad in (0, 4):
        kv = torch.randn(tokens, 2, heads * dim + pad, device="cuda", generator=g).to(DT[dtype])
        kv[7, 0, 40] = float("nan")
        kv[8, 1, 3] = float("inf")
        kv[9] = 0
        kv[10] *= 2.0 ** -20
        k, v = (kv[:, i, :heads * dim].unflatten(1, (heads, dim)) for i in (0, 1))
        many = torch.randint(0, 256, (pages, heads, kv_pages.page_bytes(page, dim)), dtype=torch.uint8, device="cuda", generator=g)
        few = many.clone()
        kv_pages.store(k, v, many, slots)
        for at in range(0, tokens, 64):
            kv_pages.store(k[at:at + 64], v[at:at + 64], few, slots[at:at + 64])
        assert torch.equal(many, few)
        for out in (torch.bfloat16, torch.float16, torch.float32):
            whole = kv_pages.read(many, slots, dim, dtype=out)
            for at in range(0, tokens, 64):
                for a, b in zip(whole, kv_pages.read(many, slots[at:at + 64], dim, dtype=out)):
                    assert torch.equal(a[at:at + 64], b)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_scales_and_codes_of_every_largest_value(dtype):
    """Groups whose max|x| takes every 16-bit pattern from 0 to infinity, at both ways to store."""
    from klab_b200 import kv_pages

    tokens, heads, dim, page = 4096, 8, 128, 64
    top = torch.arange(tokens * heads * 4).div(4, rounding_mode="floor").clamp(max=0x7f80 if dtype == "bf16" else 0x7c00).to(torch.int16).view(DT[dtype])
    top = top.double().nan_to_num().view(tokens, heads, 4, 1)
    part = torch.arange(32) / 14.0 * torch.tensor([1, -1]).repeat(16)  # 0 and near the halves of a step up to the largest
    x = top * part.clamp(-1, 1)
    x[..., 31:] = top
    x = x.to(DT[dtype]).flatten(2)
    codes, scales = ok.quantize(x.double().numpy())
    want = ok.values(codes, scales)
    slots = i32(np.arange(tokens))
    buf = kv_pages.empty_pages(tokens // page, heads, page, dim)
    dev = x.cuda()
    for step in (tokens, 128):
        buf.zero_()
        for at in range(0, tokens, step):
            kv_pages.store(dev[at:at + step], -dev[at:at + step], buf, slots[at:at + step])
        k, v = kv_pages.read(buf, slots, dim, dtype=torch.float32)
        assert np.array_equal(f64(k), want) and np.array_equal(f64(v), -want)


def test_slots_outside_the_pages_touch_nothing(native):
    from klab_b200 import kv_pages

    buf = torch.randint(0, 256, (3, 2, kv_pages.page_bytes(16, 64)), dtype=torch.uint8, device="cuda")
    before = buf.clone()
    k = torch.randn(4, 2, 64, device="cuda").bfloat16()
    bad = i32([48, -2, 2 ** 31 - 1, -2 ** 31])
    kv_pages.store(k, k, buf, bad)
    torch.cuda.synchronize()
    assert native.device_status(clear=True) == 4 and torch.equal(buf, before)
    for x in kv_pages.read(buf, bad, 64):
        assert not x.any()
    assert native.device_status(clear=True) == 4


def test_offsets_past_32_bits():
    """Rows behind the first 4 GiB of the pages."""
    from klab_b200 import kv_pages

    pages, heads, dim, page = 60000, 8, 128, 64
    buf = torch.zeros(pages, heads, kv_pages.page_bytes(page, dim), dtype=torch.uint8, device="cuda")
    assert buf.numel() > 2 ** 32
    slots = i32([pages * page - 1, 0, (pages - 1) * page + 17, 32 * page])
    k, v = (torch.randn(4, heads, dim, device="cuda").bfloat16() for _ in range(2))
    kv_pages.store(k, v, buf, slots)
    for x, got in zip((k, v), kv_pages.read(buf, slots, dim, dtype=torch.float32)):
        assert np.array_equal(f64(got), ok.values(*ok.quantize(f64(x))))
    q = torch.randn(1, heads, dim, device="cuda").bfloat16()
    table = i32([[pages - 1]])
    rows = i32((pages - 1) * page + np.arange(40))
    k, v = (torch.randn(40, heads, dim, device="cuda").bfloat16() for _ in range(2))
    kv_pages.store(k, v, buf, rows)
    out = kv_pages.attention(q, buf, table, i32([40]), i32([0, 1]))
    close(out, q, [0], [40], [1], k, v, "bf16")


# ---------------------------------------------------------------- attention

def close(out, q, starts, lengths, new, k, v, dtype, scale=None):
    """out's rows against the oracle over the quantised rows k, v (all requests behind one another).

    Bounds per element, with A = sum of softmax * |v| and M = sum of softmax * scale_G, for a value scale_G * (u - 8) with
    u <= 15: the FP16 rounding of p and of p * scale, 2^-11 each at most and alike for u and for 8, give 2^-10 A; exp2 and
    the FP32 weights and their sum, 2^-13 A; weights under FP16's normal range add less than 2^-20 of the largest |v|; then
    half a step of the output type. The sums run over P' u and 8 P' apart, so their FP32 accumulators hold up to 23 M and take
    at most length / 16 + 8 truncated additions of 2^-23 each. A score's group of 32 dims is
    scale_G * (sum q u - 8 sum q): its FP32 accumulator holds at most 23 sum |q| and takes four truncated additions (two
    MMAs, 2^-23 each at most, and the start and the scaled sum), so the score is off by at most
    d = 4 * 2^-23 * 23 * scale * sum_G scale_G sum |q| and a weight, numerator and denominator, by 2 d.
    """
    scale = q.shape[2] ** -0.5 if scale is None else scale
    half = torch.finfo(DT[dtype]).eps / 2
    at = 0
    for s, length, n in zip(starts, lengths, new):
        (kc, ks), (vc, vs) = (ok.quantize(f64(x[at:at + length])) for x in (k, v))
        kk, vv = ok.values(kc, ks), ok.values(vc, vs)
        at += length
        if not n or not length:
            continue
        want, size = ok.attention(f64(q[s:s + n]), kk, vv, n, scale)
        mass, _ = ok.attention(f64(q[s:s + n]), kk, np.repeat(vs, 32, -1), n, scale)
        got = f64(out[s:s + n])
        top = np.abs(vv).max(initial=0.0)
        qs = np.abs(f64(q[s:s + n])).reshape(n, ks.shape[1], -1, ks.shape[2], 32).sum(-1)
        d = 92 * 2.0 ** -23 * scale * np.einsum("nhgG,hG->nhg", qs, ks.max(0)).reshape(n, -1, 1)
        tol = half * np.abs(want) + (1 + half) * ((2.0 ** -10 + 2.0 ** -13 + 2 * d) * size + 2.0 ** -20 * top
                                                 + (length / 16 + 8) * 23 * 2.0 ** -23 * mass) + 2.0 ** -24
        assert np.isfinite(got).all()
        worst = np.max(np.abs(got - want) - tol)
        assert worst <= 0, (length, n, worst)


def attention_case(lengths, new, heads, kvh, dim, page, dtype, seed, gap=0, strong=1.0):
    """Pages with garbage where nothing was stored, q as a slice of a fused row, `gap` rows between requests."""
    from klab_b200 import kv_pages

    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    table, _, _ = table_state(rng, lengths, page, 3, slack=1)
    pages = int((table >= 0).sum()) + 3
    buf = torch.randint(0, 256, (pages, kvh, kv_pages.page_bytes(page, dim)), generator=gen, device="cuda", dtype=torch.uint8)
    buf.view(torch.float16)[:, :, 7::11] = float("nan")
    total = int(sum(lengths))
    k, v = (torch.randn(total, kvh, dim, generator=gen, device="cuda").to(DT[dtype]) for _ in range(2))
    k, v = (k * strong).to(DT[dtype]), (v * strong).to(DT[dtype])
    slots = np.concatenate([table[i, np.arange(n) // page] * page + np.arange(n) % page for i, n in enumerate(lengths)])
    if total:
        kv_pages.store(k, v, buf, i32(slots))
    starts = np.concatenate([[0], np.cumsum(new)])
    tokens = int(starts[-1]) + gap
    qkv = torch.randn(max(tokens, 1), (heads + 2 * kvh) * dim, generator=gen, device="cuda").to(DT[dtype])
    return qkv[:, :heads * dim].view(-1, heads, dim), buf, i32(table), i32(lengths), i32(starts), starts, k, v


CASES = [  # lengths, new, heads, kv heads, dim, page, dtype
    ([1], [1], 4, 4, 64, 16, "bf16"), ([300], [1], 32, 8, 64, 16, "bf16"), ([17, 1, 64], [1, 1, 1], 8, 2, 128, 16, "bf16"),
    ([129, 2000, 15, 16], [1, 1, 1, 1], 28, 4, 128, 32, "fp16"), ([500], [1], 16, 1, 128, 64, "bf16"),
    ([5, 33, 260], [5, 3, 4], 8, 2, 128, 16, "bf16"), ([1, 2, 3, 4], [1, 2, 3, 4], 6, 2, 64, 16, "fp16"),
    ([100, 0, 40], [1, 0, 1], 4, 1, 256, 16, "bf16"), ([700, 90], [16, 16], 16, 2, 64, 64, "bf16"),
    ([210], [2], 12, 1, 256, 32, "fp16"), ([4096], [1], 8, 8, 128, 16, "bf16"), ([1000], [7], 64, 1, 128, 16, "bf16"),
    ([50] * 300, [1] * 300, 4, 1, 64, 16, "bf16"), ([16, 32, 48, 128, 256], [1] * 5, 5, 5, 128, 1024, "fp16")]


@pytest.mark.parametrize("lengths,new,heads,kvh,dim,page,dtype", CASES, ids=[str(i) for i in range(len(CASES))])
def test_attention_matches_oracle(lengths, new, heads, kvh, dim, page, dtype):
    from klab_b200 import kv_pages

    q, buf, table, ln, st, starts, k, v = attention_case(lengths, new, heads, kvh, dim, page, dtype, len(lengths) + heads)
    out = kv_pages.attention(q, buf, table, ln, st, max_new=max(new))
    close(out, q, starts, lengths, new, k, v, dtype)
    again = kv_pages.attention(q, buf, table, ln, st, max_new=max(new))
    assert torch.equal(out, again)


@pytest.mark.parametrize("requests,longest,new,heads,kvh,dim", [
    (5, 800, 1, 64, 64, 64), (7, 2500, 3, 16, 2, 64), (33, 900, 1, 8, 2, 64), (64, 600, 2, 8, 2, 128), (60, 1100, 1, 8, 8, 64),
    (65, 700, 1, 8, 4, 64), (2, 9000, 16, 64, 8, 64), (32, 1500, 4, 12, 1, 256)])
def test_batches_that_are_cut_in_different_ways(requests, longest, new, heads, kvh, dim):
    """Segments with CTAs of their own, equal shares across segments, and more requests than a warp holds."""
    rng = np.random.default_rng(requests)
    lengths = [longest, *(int(x) for x in rng.integers(0, longest, requests - 1))]
    fresh = [min(n, int(x)) for n, x in zip(lengths, rng.integers(0, new + 1, requests))]
    fresh[0] = new
    test_attention_matches_oracle(lengths, fresh, heads, kvh, dim, 16, "bf16")


@pytest.mark.parametrize("strong", [2.0 ** -12, 100.0, 3000.0])
def test_attention_over_weak_and_strong_rows(strong):
    """V scales far from 1 move the weights' reference exponent; strong keys make the softmax one-hot."""
    from klab_b200 import kv_pages

    lengths, new = [400, 37], [1, 2]
    q, buf, table, ln, st, starts, k, v = attention_case(lengths, new, 8, 2, 128, 16, "fp16", 9, strong=strong)
    out = kv_pages.attention(q, buf, table, ln, st, max_new=2, scale=0.05 / strong)
    close(out, q, starts, lengths, new, k, v, "fp16", scale=float(np.float32(0.05 / strong)))


def test_attention_with_growing_v_scales_and_far_scores():
    """Each 16 tokens are stronger than the last: the reference moves at every block of a run."""
    from klab_b200 import kv_pages

    n, dim, page = 512, 64, 16
    gen = torch.Generator(device="cuda").manual_seed(4)
    grow = 2.0 ** (torch.arange(n, device="cuda") / 40.0)[:, None, None]
    k = (torch.randn(n, 2, dim, generator=gen, device="cuda") * grow.sqrt()).half()
    v = (torch.randn(n, 2, dim, generator=gen, device="cuda") * grow).half()
    q = torch.randn(1, 8, dim, generator=gen, device="cuda").half()
    for flip in (False, True):
        kk, vv = (x.flip(0).contiguous() if flip else x for x in (k, v))
        buf = kv_pages.empty_pages(n // page, 2, page, dim)
        kv_pages.store(kk, vv, buf, i32(np.arange(n)))
        out = kv_pages.attention(q, buf, i32(np.arange(n // page)[None]), i32([n]), i32([0, 1]))
        close(out, q, [0], [n], [1], kk, vv, "fp16")


def test_rows_that_see_nothing_and_rows_of_nobody():
    from klab_b200 import kv_pages

    # Request 0 has no tokens at all, request 1 fewer tokens than rows, request 2 none to add; one row belongs to nobody.
    q, buf, table, ln, st, starts, k, v = attention_case([0, 2, 40], [1, 4, 0], 8, 2, 64, 16, "bf16", 3, gap=1)
    out = torch.full_like(q, 7.0).contiguous()
    kv_pages.attention(q, buf, table, ln, st, max_new=4, out=out)
    assert not out[0].any() and not out[1:3].any()
    assert out[5:].eq(7.0).all()
    close(out, q, starts, [0, 2, 40], [0, 0, 0], k, v, "bf16")
    kk, vv = (ok.values(*ok.quantize(f64(x[:2]))) for x in (k, v))
    want, _ = ok.attention(f64(q[1:5]), kk, vv, 4, 64 ** -0.5)
    assert np.abs(f64(out[1:5]) - want).max() <= 2.0 ** -6 * np.abs(want).max()


def test_not_a_number_stays_in_its_row():
    from klab_b200 import kv_pages

    q, buf, table, ln, st, starts, k, v = attention_case([90, 70], [2, 1], 8, 2, 128, 16, "bf16", 8)
    clean = kv_pages.attention(q, buf, table, ln, st, max_new=2)
    q = q.contiguous().clone()
    q[0, 3, 5], q[2, 0, 0] = float("nan"), float("inf")
    out = kv_pages.attention(q, buf, table, ln, st, max_new=2)
    assert out[0, 3].isnan().all() and out[2, 0].isnan().any()
    keep = torch.ones(3, 8, dtype=torch.bool, device="cuda")
    keep[0, 3] = keep[2, 0] = False
    assert torch.equal(out[keep], clean[keep])


def test_bad_pages_and_lengths_are_reported(native):
    from klab_b200 import kv_pages

    lengths, new = [100, 60], [1, 1]
    q, buf, table, ln, st, starts, k, v = attention_case(lengths, new, 8, 2, 64, 16, "bf16", 2)
    good = kv_pages.attention(q, buf, table, ln, st)
    bad = table.clone()
    bad[0, 2], bad[0, 5] = buf.shape[0], -1
    out = kv_pages.attention(q, buf, bad, ln, st)
    torch.cuda.synchronize()
    assert native.device_status(clear=True) == 4
    assert torch.equal(out[1], good[1])
    keep = np.r_[0:32, 48:80, 96:100]  # the tokens of the other pages
    kk, vv = (ok.values(*ok.quantize(f64(x[:100]))) for x in (k, v))
    want, size = ok.attention(f64(q[:1]), kk[keep], vv[keep], 1, 0.125)
    assert (np.abs(f64(out[:1]) - want) <= 2.0 ** -7 * (np.abs(want) + size)).all()
    for change in ({"lengths": i32([100, table.shape[1] * 16 + 1])}, {"lengths": i32([100, -1])},
                   {"starts": i32([0, 1, 3])}, {"starts": i32([0, 1, 0])}, {"starts": i32([0, 1, 4])}):
        out = torch.full_like(good, 3.0)
        a = {"lengths": ln, "starts": st, **change}
        kv_pages.attention(q, buf, table, a["lengths"], a["starts"], out=out)
        torch.cuda.synchronize()
        assert native.device_status(clear=True) == 3
        assert torch.equal(out[0], good[0]) and out[1].eq(3.0).all()


# ---------------------------------------------------------------- together

def test_a_captured_step_serves_a_growing_batch():
    """build_step, store and attention of a batch in one graph, replayed while requests grow, wait, end and begin."""
    from klab_b200 import kv_pages

    rng = np.random.default_rng(11)
    requests, heads, kvh, dim, page, most = 5, 8, 2, 64, 16, 20
    buf = kv_pages.empty_pages(60, kvh, page, dim)
    buf.fill_(255)
    lengths, table = i32([0] * requests), i32(np.full((requests, 10), -1))
    free, count = i32(rng.permutation(60)), i32([60])
    new, ended = i32([0] * requests), torch.zeros(requests, dtype=torch.bool, device="cuda")
    qkv = torch.zeros(most, (heads + 2 * kvh) * dim, device="cuda", dtype=torch.bfloat16)
    q, k, v = (x.view(most, -1, dim) for x in qkv.split((heads * dim, kvh * dim, kvh * dim), 1))
    out = torch.zeros(most, heads, dim, device="cuda", dtype=torch.bfloat16)

    def one():
        kv_pages.release(ended, lengths, table, free, count, page_size=page)
        step = kv_pages.build_step(new, lengths, table, free, count, page_size=page, max_tokens=most, inplace=True)
        kv_pages.store(k, v, buf, step.slots)
        kv_pages.attention(q, buf, table, step.lengths, step.starts, max_new=4, out=out)
        return step

    one()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step = one()
    held_k, held_v = [[] for _ in range(requests)], [[] for _ in range(requests)]
    for turn in range(30):
        stop = rng.random(requests) < 0.1
        n = rng.integers(0, 5, requests)
        for i in np.nonzero(stop)[0]:
            held_k[i], held_v[i] = [], []
        n[[len(h) + 4 > 160 for h in held_k]] = 0
        new.copy_(i32(n))
        ended.copy_(torch.from_numpy(stop))
        qkv.copy_(torch.randn(qkv.shape, generator=torch.Generator().manual_seed(turn)))
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert step.result.item() == 0
        starts = step.starts.tolist()
        for i in range(requests):
            held_k[i] += list(k[starts[i]:starts[i + 1]].clone())
            held_v[i] += list(v[starts[i]:starts[i + 1]].clone())
        sizes = [len(h) for h in held_k]
        assert sizes == lengths.tolist()
        flat_k, flat_v = ([x for h in held for x in h] for held in (held_k, held_v))
        empty = torch.zeros(0, kvh, dim, device="cuda")
        close(out, q, starts, sizes, n, torch.stack(flat_k) if flat_k else empty, torch.stack(flat_v) if flat_v else empty, "bf16")
        assert out[starts[-1]:].eq(9.0).all()


def test_two_graphs_and_another_stream_share_nothing():
    """Two captured calls replayed on two streams at once, and eager calls on a third, all give what one call gives."""
    from klab_b200 import kv_pages

    cases = [attention_case([900, 40, 333], [1, 1, 1], 8, 2, 128, 16, "bf16", seed) for seed in (1, 2, 3)]
    want = [kv_pages.attention(*c[:5]) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for c in cases[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(kv_pages.attention(*c[:5]))
        graphs.append(g)
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            other = kv_pages.attention(*cases[2][:5])
    torch.cuda.synchronize()
    for got, w in zip((*outs, other), want):
        assert torch.equal(got, w)


def test_both_launch_paths_agree(monkeypatch):
    """The binding serves plain calls; without it the wrappers launch the same kernels through ctypes."""
    from klab_b200 import _launch, kv_pages

    def everything():
        q, buf, table, ln, st, starts, k, v = attention_case([300, 40], [1, 2], 8, 2, 64, 16, "bf16", 6)
        out = torch.zeros(q.shape, device="cuda", dtype=q.dtype)
        assert kv_pages.attention(q, buf, table, ln, st, max_new=2, out=out) is out
        rows = kv_pages.read(buf, i32([5, -1, 33]), 64, dtype=torch.float16)
        step = kv_pages.build_step(i32([3, 0]), ln, table, i32(np.arange(40)), i32([5]), page_size=16, max_tokens=8)
        count, lengths = i32([5]), ln.clone()
        moved = kv_pages.build_step(i32([1, 1]), lengths, table, i32(np.arange(40)), count, page_size=16, max_tokens=8, inplace=True)
        assert moved.lengths is lengths and moved.free_count is count
        return (out, kv_pages.attention(q, buf, table, ln, st, max_new=2, scale=0.3), *rows, *step, *moved)

    everything()
    assert _launch.fast is not None
    served = []
    with monkeypatch.context() as m:
        class Counting:
            def __getattr__(self, name):
                def call(*a):
                    r = getattr(real, name)(*a)
                    served.append(r is not None)
                    return r
                return call
        real = _launch.fast
        m.setattr(_launch, "fast", Counting())
        first = everything()
    assert served and all(served)
    monkeypatch.setattr(_launch, "fast", None)
    for a, b in zip(first, everything()):
        assert a.shape == b.shape and a.dtype == b.dtype and torch.equal(a, b)


def test_refusals_on_the_gpu():
    """What the binding does not serve is refused by the wrappers, with a device ready."""
    from klab_b200 import kv_pages

    q, buf, table, ln, st, starts, k, v = attention_case([30, 4], [1, 1], 8, 2, 64, 16, "bf16", 6)
    for bad in ({"max_new": 0}, {"max_new": 17}, {"scale": -1.0}, {"scale": float("inf")}, {"out": q}, {"lengths": ln.long()},
                {"lengths": ln.cpu()}, {"starts": st[:2]}, {"q": q.float()}, {"q": q[:, :7]}, {"pages": buf[:, :, :-16]},
                {"pages": buf.cpu()}, {"table": table.t()}, {"q": q.clone().requires_grad_()}):
        a = {"q": q, "pages": buf, "table": table, "lengths": ln, "starts": st, **bad}
        with pytest.raises(ValueError):
            kv_pages.attention(**a)
    slots = i32(np.arange(34))
    for bad in ((k, v.half(), buf, slots), (k, v, buf, slots[:3]), (k, v, buf, slots.long()), (k[:, :1], v[:, :1], buf, slots),
                (k.cpu(), v, buf, slots)):
        with pytest.raises(ValueError):
            kv_pages.store(*bad)
    for bad in ((buf, slots, 96), (buf, slots.long(), 64), (buf, slots, 128)):
        with pytest.raises(ValueError):
            kv_pages.read(*bad)
    with pytest.raises(ValueError):
        kv_pages.read(buf, slots, 64, dtype=torch.float64)
    free, count = i32([0] * 9), i32([3])
    for bad in ({"page_size": 24}, {"max_tokens": 0}, {"new_tokens": i32([1])}, {"lengths": table[:, 0]}, {"free_count": free},
                {"lengths": table.view(-1)[:2]}):
        a = {"new_tokens": i32([1, 1]), "lengths": ln, "table": table, "free_pages": free, "free_count": count,
             "page_size": 16, "max_tokens": 4, **bad}
        with pytest.raises(ValueError):
            kv_pages.build_step(**a)
