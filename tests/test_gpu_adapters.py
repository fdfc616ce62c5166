"""Adapters beside the shared projection against the 64-bit oracle."""

import numpy as np
import pytest
import torch

from oracle import kv_pages as ok

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def native():
    from klab_b200 import _native

    _native.lib()
    assert _native.device_status(clear=True) == 0
    yield _native
    assert _native.device_status(clear=True) == 0


def f64(t):
    return t.double().cpu().numpy()


def case(kind, m, n, k, rank, count, seed=0):
    """(weights for the call, their exact values, x, a, b, c, ids)."""
    from klab_b200 import compressed_bf16 as cb, fp4, int8_weights

    gen = torch.Generator(device="cuda").manual_seed(seed + m + n)
    randn = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    x, a, b = randn(m, k).bfloat16(), (randn(count, rank, k) * 0.05).bfloat16(), (randn(count, n, rank) * 0.05).bfloat16()
    c = torch.rand(count, generator=gen, device="cuda") * 2 - 0.5
    ids = torch.randint(-1, count, (m,), generator=gen, device="cuda", dtype=torch.int32)
    w32 = randn(n, k) * 0.02
    if kind == "bf16":
        w = w32.bfloat16()
        exact = f64(w)
    elif kind == "coded":
        bits = w32.bfloat16().view(torch.int16).cpu().numpy().view(np.uint16)
        w = cb.upload(cb.pack_bits(bits), "cuda")
        exact = f64(w32.bfloat16())
    elif kind in ("int8", "int8_64"):
        w = (int8_weights.quantize_weights_per_row if kind == "int8" else int8_weights.quantize_weights)(w32)
        exact = f64(w.codes) * (f64(w.scales)[:, None] if kind == "int8" else np.repeat(f64(w.scales), 64, 1))
    else:
        w = fp4.quantize_weights_f16(w32)
        exact = f64(w.dequantize())
    return w, exact, x, a, b, c, ids


def close(y, exact, x, a, b, c, ids, dtype):
    """FP32 sums of exact products: 2^-22 of the sum of absolute values at these lengths (chains of at most 256 terms per
    accumulator and a tree, 2^-24 each; the tensor-core routes chain K / 32 truncated FP32 adds, 2^-16 in all); t is
    rounded to FP32 (or to two BF16 terms, 2^-16) before its product; then half a step of the output type."""
    want = f64(x) @ exact.T
    size = np.abs(f64(x)) @ np.abs(exact).T
    more, more_size = ok.adapter_delta(f64(x), f64(a), f64(b), f64(c), ids.tolist())
    half = torch.finfo(dtype).eps / 2
    tol = half * np.abs(want + more) + 2.0 ** -15 * (size + more_size) * (1 + half)
    err = np.abs(f64(y) - want - more)
    assert (err <= tol).all(), float((err - tol).max())


CASES = [("bf16", 1, 256, 512, 16, 3), ("bf16", 1, 4096, 4096, 16, 4), ("bf16", 3, 1000, 1856, 8, 2), ("bf16", 16, 512, 2048, 64, 9),
         ("bf16", 7, 130, 4928, 24, 5), ("bf16", 40, 96, 264, 32, 4), ("bf16", 2, 37, 8, 8, 1), ("bf16", 5, 33, 14336, 256, 2),
         ("int8", 1, 1024, 1024, 16, 2), ("int8", 8, 2000, 4096, 16, 8), ("int8", 16, 512, 1856, 32, 4), ("int8_64", 4, 256, 512, 8, 3),
         ("fp4", 1, 512, 2048, 16, 2), ("fp4", 11, 1000, 4928, 64, 6), ("coded", 2, 300, 1024, 16, 2), ("coded", 16, 64, 512, 8, 2)]


@pytest.mark.parametrize("kind,m,n,k,rank,count", CASES, ids=["-".join(map(str, c)) for c in CASES])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_matches_oracle(kind, m, n, k, rank, count, dtype):
    from klab_b200.adapters import adapter_linear

    w, exact, *rest = case(kind, m, n, k, rank, count)
    y = adapter_linear(rest[0], w, *rest[1:], output_dtype=dtype)
    close(y, exact, *rest, dtype)
    out = torch.empty_like(y)
    assert adapter_linear(rest[0], w, *rest[1:], output_dtype=dtype, out=out) is out and torch.equal(out, y)


@pytest.mark.parametrize("kind,m,n,k,rank,count", [("bf16", 2, 20000, 128, 8, 2), ("int8", 9, 9000, 2048, 24, 12), ("fp4", 16, 4500, 1024, 8, 3),
                                                   ("bf16", 20, 6000, 1000, 40, 5), ("int8", 1, 128, 16384, 16, 1)])
def test_rows_cut_in_different_ways(kind, m, n, k, rank, count):
    """More blocks of rows than there are CTAs, and few blocks over a long K."""
    test_matches_oracle(kind, m, n, k, rank, count, torch.bfloat16)


def test_rows_depend_on_their_own_adapter_alone(native):
    """All rows without one, all with the same one, mixed, and indices outside the stack (counted as none, reported)."""
    from klab_b200.adapters import adapter_linear

    w, exact, x, a, b, c, _ = case("bf16", 12, 300, 1024, 16, 3)
    ids = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    none, same = ids([-1] * 12), ids([1] * 12)
    mixed = ids([-1, 1, 0, 2, 1, 1, -1, 0, 2, 2, 1, 0])
    got = {k: adapter_linear(x, w, a, b, c, v, output_dtype=torch.float32) for k, v in
           (("none", none), ("same", same), ("mixed", mixed))}
    for k, v in (("none", none), ("same", same), ("mixed", mixed)):
        close(got[k], exact, x, a, b, c, v, torch.float32)
    for row, i in enumerate(mixed.tolist()):
        if i in (-1, 1):
            assert torch.equal(got["mixed"][row], got["same" if i == 1 else "none"][row])
    bad = adapter_linear(x, w, a, b, c, ids([3, -2, 2 ** 31 - 1, -2 ** 31] * 3), output_dtype=torch.float32)
    torch.cuda.synchronize()
    assert native.device_status(clear=True) == 6 and torch.equal(bad, got["none"])


def test_not_a_number_stays_in_its_row():
    from klab_b200.adapters import adapter_linear

    for kind, m in (("bf16", 1), ("bf16", 6), ("bf16", 16), ("int8", 5)):
        w, exact, x, a, b, c, ids = case(kind, m, 200, 1024, 16, 4)
        ids = torch.arange(m, device="cuda", dtype=torch.int32) % 3
        a = a.clone()
        a[3] = float("nan")   # an adapter of nobody
        clean = adapter_linear(x, w, a, b, c, ids)
        assert clean.isfinite().all()
        x = x.clone()
        x[0, 3] = float("nan")
        y = adapter_linear(x, w, a, b, c, ids)
        assert y[0].isnan().all() and torch.equal(y[1:], clean[1:])


@pytest.mark.parametrize("captured", [False, True])
def test_weights_that_the_call_before_wrote(captured):
    """Rows out of one call are the weights of the next, with nothing between the two on the stream."""
    from klab_b200.adapters import adapter_linear

    w, _, x, a, b, c, ids = case("bf16", 192, 1024, 512, 16, 3)
    _, _, x2, a2, b2, c2, ids2 = case("bf16", 5, 192, 1024, 16, 2, seed=1)
    xs = [x, x * 2, x * -1, x.roll(1, 0)]
    want = []
    for v in xs:
        y = adapter_linear(v, w, a, b, c, ids)
        torch.cuda.synchronize()
        want.append(adapter_linear(x2, y, a2, b2, c2, ids2))
    y = torch.zeros_like(y)  # one buffer that every pair writes anew

    def run():
        return [adapter_linear(x2, adapter_linear(v, w, a, b, c, ids, out=y), a2, b2, c2, ids2) for v in xs * 4]

    if captured:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = run()
        for _ in range(3):
            g.replay()
    else:
        got = run()
    for i, v in enumerate(got):
        assert torch.equal(v, want[i % len(xs)])


def test_graphs_and_streams():
    from klab_b200.adapters import adapter_linear

    cases = [case(kind, m, 512, 2048, 32, 5, seed) for kind, m, seed in (("int8", 4, 1), ("int8", 8, 2), ("bf16", 16, 3))]
    call = lambda c: adapter_linear(c[2], c[0], *c[3:])  # noqa: E731
    want = [call(c) for c in cases]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for c in cases:  # all captured on one stream, replayed on three at once
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(c))
        graphs.append(g)
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for got, w in zip(outs, want):
        assert torch.equal(got, w)


def test_a_step_of_a_batch_with_adapters():
    """Query, key and value rows with each request's adapter, stored and attended, as one step uses them."""
    from klab_b200 import kv_pages
    from klab_b200.adapters import adapter_linear

    i32 = lambda v: torch.as_tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    requests, heads, kvh, dim, hidden, page = 3, 4, 2, 64, 256, 16
    n = (heads + 2 * kvh) * dim
    w, exact, x, a, b, c, _ = case("bf16", 4, n, hidden, 8, 3)
    of_request = i32([2, -1, 0])
    lengths, table, count = i32([0] * 3), i32([[-1] * 4] * 3), i32([12])
    free = i32(list(range(12)))
    buf = kv_pages.empty_pages(12, kvh, page, dim)
    step = kv_pages.build_step(i32([2, 1, 1]), lengths, table, free, count, page_size=page, max_tokens=4)
    ids = of_request[step.rows.long()]
    qkv = adapter_linear(x, w, a, b, c, ids)
    close(qkv, exact, x, a, b, c, ids, torch.bfloat16)
    q, k, v = (t.view(4, -1, dim) for t in qkv.split((heads * dim, kvh * dim, kvh * dim), 1))
    kv_pages.store(k, v, buf, step.slots)
    out = kv_pages.attention(q, buf, table, step.lengths, step.starts, max_new=2)
    held = kv_pages.read(buf, step.slots, dim, dtype=torch.float32)
    for first, total in ((0, 2), (2, 1), (3, 1)):
        rows = slice(first, first + total)
        want, size = ok.attention(f64(q[rows]), f64(held[0][rows]), f64(held[1][rows]), total, dim ** -0.5)
        assert (np.abs(f64(out[rows]) - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -9 * size + 1e-6).all()
