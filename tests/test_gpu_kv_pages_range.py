"""Attention over 4-bit pages at the ends of its range: one huge value of V, weak values under a long tail, scores and
scales near the largest floats, and rows of no request."""

import numpy as np
import pytest
import torch

from oracle import kv_pages as ok
from test_gpu_kv_pages import DT, attention_case, close, f64, i32, native  # noqa: F401

pytestmark = pytest.mark.gpu


def one_request(k, v, page=16):
    """Pages in order that hold these rows, and the table, lengths and starts of one token's attention over them."""
    from klab_b200 import kv_pages

    n, kvh, dim = k.shape
    pages = -(-n // page)
    buf = kv_pages.empty_pages(pages, kvh, page, dim)
    buf.fill_(255)
    kv_pages.store(k, v, buf, i32(np.arange(n)))
    return buf, i32(np.arange(pages)[None]), i32([n]), i32([0, 1])


@pytest.mark.parametrize("dtype,huge", [("bf16", 3e5), ("bf16", float("inf")), ("bf16", 2.0 ** 18), ("fp16", 6e4), ("fp16", 20.0)])
@pytest.mark.parametrize("at", [5, 650], ids=["first", "late"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_one_huge_value_stays_in_its_group(dtype, huge, at, dim):
    """A V scale up to the largest FP16 value, in the first tokens or behind many, against each group's own magnitude.

    A weight times its V scale s is rounded to FP16 once, 2^-11 of itself or 2^-25 at worst. A warp's weights are taken so
    that its largest is at least 2^(10 - e), with 2^e the end of the range of scales (2^-8, 2^0 or 2^15) that holds its own,
    so the 2^-25 are at most 2^(e - 35) of the largest weight, and a value is s * (u - 8) with |u - 8| <= 8: over n tokens
    8 n 2^(e - 35). The sums: an MMA adds its 16 products to the accumulator in single precision, in an order and with a
    rounding that are not specified, so that beside one large term each of the n smaller ones may be cut, 2^-23 of the
    accumulator a time, where `close` counts one for 16 rows of alike size: (n + 8) * 23 * 2^-23 M. It counts in the huge
    value's own group alone. Everything else as in `close`.
    """
    from klab_b200 import kv_pages

    n, heads, kvh = 700, 8, 2
    gen = torch.Generator(device="cuda").manual_seed(at + dim)
    k, v = (torch.randn(n, kvh, dim, generator=gen, device="cuda").to(DT[dtype]) for _ in range(2))
    q = torch.randn(1, heads, dim, generator=gen, device="cuda").to(DT[dtype])
    v[at, 0, 3] = huge
    out = f64(kv_pages.attention(q, *one_request(k, v)))
    (kc, ks), (vc, vs) = (ok.quantize(f64(x)) for x in (k, v))
    kk, vv = ok.values(kc, ks), ok.values(vc, vs)
    want, size = ok.attention(f64(q), kk, vv, 1, dim ** -0.5)
    mass, _ = ok.attention(f64(q), kk, np.repeat(vs, 32, -1), 1, dim ** -0.5)
    half = torch.finfo(DT[dtype]).eps / 2
    qs = np.abs(f64(q)).reshape(1, kvh, -1, dim // 32, 32).sum(-1)
    d = 92 * 2.0 ** -23 * dim ** -0.5 * np.einsum("nhgG,hG->nhg", qs, ks.max(0)).reshape(1, -1, 1)
    tol = half * np.abs(want) + (1 + half) * ((2.0 ** -11 + 2.0 ** -13 + 2 * d) * size + 8 * n * 2.0 ** (15 - 35)
                                             + (n + 8) * 23 * 2.0 ** -23 * mass)
    assert np.isfinite(out).all()
    err = np.abs(out - want) - tol
    assert (err <= 0).all(), err.max()
    # What no bound of the sums hides: the other groups still hold their own mean to a few per cent.
    others = out[0, :, 32:]
    assert np.abs(others - want[0, :, 32:]).max() <= 0.05 * np.abs(want[0, :, 32:]).max()


def test_weak_values_keep_a_long_tail():
    """V scales of 2^-20: a token that outweighs each of the others by 2^13.4, and the others' sum, which counts.

    All rows behind the first are alike, so the answer has a closed form. Error: the weights' one rounding to FP16 (2^-11;
    their range is the scales', so none of them is an FP16 subnormal: 2^(10 + 8 - 13.5 - 20) is above 2^-16, off by 2^-25 at
    worst, 2^-9 of it), exp2 and the sums in FP32 (2^-13), half a step of BF16.
    """
    from klab_b200 import kv_pages

    n, kvh, dim = 6000, 148, 64
    k = torch.zeros(n, kvh, dim, device="cuda", dtype=torch.bfloat16)
    v = torch.full((n, kvh, dim), 7 * 2.0 ** -20, device="cuda", dtype=torch.bfloat16)
    k[0], v[0] = 1.0, 0.0
    q = torch.ones(1, kvh, dim, device="cuda", dtype=torch.bfloat16)
    kk = ok.values(*ok.quantize(np.ones((1, 32))))[0, 0]
    scale = float(np.float32(np.log(2.0) * (14 - np.log2(1.5)) / (64 * kk)))
    out = f64(kv_pages.attention(q, *one_request(k, v), scale=scale))
    tail = (n - 1) * np.exp(-scale * 64 * kk)
    want = 7 * 2.0 ** -20 * tail / (1 + tail)
    assert np.abs(out / want - 1).max() <= 2.0 ** -8 + 2.0 ** -9 + 2.0 ** -11 + 2.0 ** -12


@pytest.mark.parametrize("dtype,times,scale", [("bf16", 2.0 ** 28, None), ("bf16", 2.0 ** 100, None), ("bf16", 2.0 ** 122, None),
                                               ("bf16", 1.0, 2.9e38), ("fp16", 1.0, 1e30), ("fp16", 2.0 ** 12, 2.0 ** 20),
                                               ("bf16", 2.0 ** -120, 2.0 ** 100), ("bf16", 0.0, 2.9e38)])
def test_far_scores_stay_finite(dtype, times, scale):
    """Scores of 2^30 and far beyond: FP32 holds them to 2^-24 of themselves, so the first token of each row by far is the
    whole result, rounded once; a query of zeros weighs all tokens alike."""
    from klab_b200 import kv_pages

    n, heads, kvh, dim = 300, 8, 2, 128
    gen = torch.Generator(device="cuda").manual_seed(7)
    k, v = (torch.randn(n, kvh, dim, generator=gen, device="cuda").to(DT[dtype]) for _ in range(2))
    q = (torch.randn(1, heads, dim, generator=gen, device="cuda") * times).to(DT[dtype])
    out = kv_pages.attention(q, *one_request(k, v), scale=scale)
    kk, vv = (ok.values(*ok.quantize(f64(x))) for x in (k, v))
    s = np.einsum("hgd,phd->hgp", f64(q)[0].reshape(kvh, 4, dim), kk) * (dim ** -0.5 if scale is None else scale)
    top = np.sort(s, -1)
    if times:  # what decides is far above the rounding of a score
        assert ((top[..., -1] - top[..., -2]) > 2.0 ** -18 * np.abs(s).max(-1)).all()
    if times >= 1.0:
        want = vv[s.argmax(-1), np.arange(kvh)[:, None]].reshape(heads, dim)
        half = torch.finfo(DT[dtype]).eps / 2
        assert (np.abs(f64(out)[0] - want) <= (half + 2.0 ** -10) * np.abs(want)).all()
    else:
        close(out, q, [0], [n], [1], k, v, dtype, scale=scale if times else 1.0)


@pytest.fixture
def dirty_memory():
    """What the allocator gives out next holds NaN."""
    def spoil(*shape, dtype):
        torch.cuda.synchronize()
        for t in [torch.full(shape, float("nan"), device="cuda", dtype=dtype) for _ in range(4)]:
            del t
    return spoil


@pytest.mark.parametrize("binding", [True, False])
@pytest.mark.parametrize("lengths,new,heads,kvh,dim,gap", [([40, 17], [1, 1], 8, 2, 64, 3), ([900, 40, 333], [1, 0, 2], 28, 4, 128, 40),
                                                           ([0, 0], [0, 0], 4, 4, 256, 5), ([700], [16], 16, 1, 128, 700),
                                                           ([30] * 70, [1] * 70, 4, 1, 64, 1)])
def test_rows_of_nobody_are_zeros_in_a_new_result(native, dirty_memory, monkeypatch, binding, lengths, new, heads, kvh, dim, gap):  # noqa: F811
    """A padded batch's rows, before the first request's and behind the last one's; a request whose numbers make no sense."""
    from klab_b200 import _launch, kv_pages

    q, buf, table, ln, st, starts, k, v = attention_case(lengths, new, heads, kvh, dim, 16, "bf16", 3, gap=gap)
    most = max(1, *new)
    want = torch.full(q.shape, 7.0, device="cuda", dtype=q.dtype)
    kv_pages.attention(q, buf, table, ln, st, max_new=most, out=want)
    assert want[starts[-1]:].eq(7.0).all()
    want[starts[-1]:] = 0
    if not binding:
        monkeypatch.setattr(_launch, "fast", None)
    dirty_memory(*q.shape, dtype=q.dtype)
    assert torch.equal(kv_pages.attention(q, buf, table, ln, st, max_new=most), want)
    # The requests begin behind `gap` rows.
    late = torch.cat([q[starts[-1]:], q[:starts[-1]]])
    dirty_memory(*q.shape, dtype=q.dtype)
    got = kv_pages.attention(late, buf, table, ln, st + gap, max_new=most)
    assert not got[:gap].any() and torch.equal(got[gap:], want[:starts[-1]])
    if len(lengths) > 1 and new[0]:
        wrong = ln.clone()
        wrong[0] = -1
        dirty_memory(*q.shape, dtype=q.dtype)
        got = kv_pages.attention(q, buf, table, wrong, st, max_new=most)
        torch.cuda.synchronize()
        assert native.device_status(clear=True) == 3
        assert not got[:new[0]].any() and torch.equal(got[new[0]:], want[new[0]:])


def test_rows_of_nobody_in_a_captured_call():
    """One graph, replayed for fewer and more requests' rows: what an earlier replay left is not there."""
    from klab_b200 import kv_pages

    q, buf, table, ln, st, starts, k, v = attention_case([50, 60, 70], [1, 1, 1], 8, 2, 64, 16, "fp16", 5, gap=4)
    kv_pages.attention(q, buf, table, ln, st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kv_pages.attention(q, buf, table, ln, st)
    graph.replay()
    whole = out.clone()
    for rows in (0, 1, 3, 2):
        st.copy_(i32(np.minimum(np.arange(4), rows)))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[:rows], whole[:rows]) and not out[rows:].any()
