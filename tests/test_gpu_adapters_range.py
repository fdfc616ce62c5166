"""Adapters beside the shared projection: values of x far apart and near the largest, many
rows, operands that the launch before wrote, operands off 16-byte boundaries, and both ways to launch."""

from dataclasses import replace

import pytest
import torch

from test_gpu_adapters import case, close, f64, native  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "int8", "fp4"])
@pytest.mark.parametrize("m", [1, 5, 16])
@pytest.mark.parametrize("far", [2.0 ** 31, 2.0 ** 60, 2.0 ** 100])
def test_a_far_value_of_x_leaves_the_others(kind, m, far):
    """Columns whose weights are 0 may hold anything finite: the rest of the row counts to the last bit."""
    from klab_b200 import fp4, int8_weights
    from klab_b200.adapters import adapter_linear

    n, k = 300, 2048
    _, _, x, a, b, c, ids = case(kind, m, n, k, 16, 3, seed=3)
    w32 = torch.randn(n, k, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda") * 0.02
    w32[:, 7], w32[:, 1500], a[:, :, 7], a[:, :, 1500] = 0, 0, 0, 0
    x[:, 7], x[:, 1500] = far, -far
    if kind == "bf16":
        w = w32.bfloat16()
        exact = f64(w)
    elif kind == "int8":
        w = int8_weights.quantize_weights_per_row(w32)
        exact = f64(w.codes) * f64(w.scales)[:, None]
    else:
        w = fp4.quantize_weights_f16(w32)
        exact = f64(w.dequantize())
    assert not exact[:, 7].any() and not exact[:, 1500].any()
    close(adapter_linear(x, w, a, b, c, ids, output_dtype=torch.float32), exact, x, a, b, c, ids, torch.float32)


@pytest.mark.parametrize("kind", ["bf16", "int8", "fp4"])
@pytest.mark.parametrize("m", [1, 16])
@pytest.mark.parametrize("times", [2.0 ** 124, 2.0 ** 121, 2.0 ** 60, 2.0 ** -60])
def test_x_near_the_ends_of_its_range(kind, m, times):
    """Sums whose value is in range although those of the weights' codes would not be."""
    from klab_b200.adapters import adapter_linear

    w, exact, x, a, b, c, ids = case(kind, m, 200, 1024, 8, 2, seed=4)
    x = x * times
    y = adapter_linear(x, w, a, b, c, ids, output_dtype=torch.float32)
    assert y.isfinite().all()
    close(y.double() / times, exact, x.double() / times, a, b, c, ids, torch.float32)


# Rows around and above a tile of 16; 2100 rows of 9000 outputs are two parts in either form.
@pytest.mark.parametrize("kind,m,n,k,rank", [("bf16", 17, 300, 512, 16), ("int8", 129, 1000, 1024, 8), ("fp4", 129, 200, 2048, 24),
                                             ("bf16", 2048, 520, 256, 16), ("bf16", 2100, 9000, 128, 8), ("int8", 2100, 9000, 128, 8),
                                             ("fp4", 2100, 9000, 128, 8), ("coded", 2100, 9000, 128, 8), ("int8_64", 1870, 9000, 64, 8)])
def test_many_rows(kind, m, n, k, rank):
    from klab_b200.adapters import adapter_linear

    w, exact, *rest = case(kind, m, n, k, rank, 5)
    close(adapter_linear(rest[0], w, *rest[1:]), exact, *rest, torch.bfloat16)


def test_scratch_stays_small(native):  # noqa: F811
    """FP32 sums of 64 MiB at a time, whatever the number of rows."""
    scratch = native.lib().klab_adapter_scratch
    for wfmt in (native.W_BF16, native.W_I8_ROW, native.W_FP4_G32H, native.W_CBF16, native.W_I8_G64):
        for m in (1, 16, 17, 500, 2048, 65535):
            for n, k in ((14336, 4096), (4096, 14336), (100, 131072)):
                for rank in (8, 256):
                    assert 0 < scratch(wfmt, m, n, k, rank) <= 2 ** 26 + 2 ** 22, (wfmt, m, n, k, rank)


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("kind", ["coded", "int8_64", "int8", "fp4", "bf16"])
def test_operands_that_the_launch_before_wrote(kind, captured):
    """x, A, B, the adapters' scales, the ids and the weights' own scales come out of the launches right before the call: each
    in turn is the last one written."""
    from klab_b200.adapters import adapter_linear

    w0, _, x0, a0, b0, c0, ids0 = case("bf16", 12, 1024, 512, 16, 3)
    w, _, x, a, b, c, ids = case(kind, 12, 640, 1024, 16, 3, seed=1)
    side = w.scales if kind in ("int8_64", "int8", "fp4") else c
    held = {"a": a, "b": b, "c": c, "ids": ids, "side": side}
    first = {k: t.clone() for k, t in held.items()}
    ways = [lambda v: v, lambda v: v.flip(0).contiguous()]
    sets = [{k: f(t) for k, t in first.items()} for f in ways]
    xs = [f(x0) for f in ways]

    def one(i, last):
        for k in (*(k for k in held if k != last), *((last,) if last in held else ())):
            held[k].copy_(sets[i][k])
        if last == "x":
            return adapter_linear(adapter_linear(xs[i], w0, a0, b0, c0, ids0, out=y), w, a, b, c, ids)
        return adapter_linear(ys[i], w, a, b, c, ids)

    y = torch.empty(12, 1024, device="cuda", dtype=torch.bfloat16)
    ys = [adapter_linear(v, w0, a0, b0, c0, ids0) for v in xs]
    want = []
    for i in (0, 1):
        for k, t in held.items():
            t.copy_(sets[i][k])
        torch.cuda.synchronize()
        want.append(adapter_linear(ys[i], w, a, b, c, ids))
    assert not torch.equal(*want)
    order = [(i % 2, last) for i, last in enumerate(("x", "a", "b", "c", "ids", "side", "x") * 4)]
    if captured:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = [one(*o) for o in order]
        for _ in range(3):
            g.replay()
    else:
        got = [one(*o) for o in order]
    for v, (i, last) in zip(got, order):
        assert torch.equal(v, want[i]), (i, last)


def moved(t, by):
    """The same values `by` bytes behind a 512-byte boundary."""
    held = torch.empty(t.numel() * t.element_size() + 64, device="cuda", dtype=torch.uint8)
    assert held.data_ptr() % 512 == 0
    out = held[by:by + t.numel() * t.element_size()].view(t.dtype).view(t.shape)
    out.copy_(t)
    return out


@pytest.mark.parametrize("m", [1, 3, 9, 40])
@pytest.mark.parametrize("kind,k,by", [("bf16", 1000, 4), ("bf16", 512, 8), ("int8", 1000, 0), ("int8", 1024, 4), ("int8", 264, 8),
                                       ("fp4", 1024, 4), ("fp4", 992, 8), ("fp4", 1024, 12)])
def test_weights_off_16_byte_boundaries(kind, k, by, m):
    """Rows or addresses that the streamed form does not take run the projection between the two small kernels."""
    from klab_b200 import fp4, int8_weights
    from klab_b200.adapters import adapter_linear

    w, exact, *rest = case(kind, m, 130, k, 16, 3, seed=2)
    if kind == "bf16":
        w = moved(w, by)
    elif kind == "int8":
        w = int8_weights.Int8Weights(moved(w.codes, by), w.scales)
    else:
        w = fp4.FP4F16Weights(moved(w.packed, by), w.scales)
    for dtype in (torch.bfloat16, torch.float32):
        close(adapter_linear(rest[0], w, *rest[1:], output_dtype=dtype), exact, *rest, dtype)


@pytest.mark.parametrize("kind", ["int8", "fp4"])
def test_scales_off_16_byte_boundaries(kind):
    from klab_b200.adapters import adapter_linear

    w, exact, *rest = case(kind, 6, 300, 2048, 16, 3, seed=6)
    want = adapter_linear(rest[0], w, *rest[1:])
    close(want, exact, *rest, torch.bfloat16)
    for by in (w.scales.element_size(), 2 * w.scales.element_size()):
        assert torch.equal(adapter_linear(rest[0], replace(w, scales=moved(w.scales, by)), *rest[1:]), want)


@pytest.mark.parametrize("kind", ["bf16", "int8", "fp4"])
@pytest.mark.parametrize("m", [1, 16, 40])
def test_both_launch_paths_agree(kind, m, monkeypatch):
    """The binding serves streamed formats; without it the wrapper launches the same kernels through ctypes."""
    from klab_b200 import _launch
    from klab_b200.adapters import adapter_linear

    w, _, *rest = case(kind, m, 300, 1024, 16, 3)

    def everything():
        out = torch.empty(m, 300, device="cuda", dtype=torch.float32)
        assert adapter_linear(rest[0], w, *rest[1:], out=out, output_dtype=torch.float32) is out
        return adapter_linear(rest[0], w, *rest[1:]), out

    everything()
    real, served = _launch.fast, []

    class Counting:
        def adapter_linear(self, *a):
            done = real.adapter_linear(*a)
            served.append(done is not None)
            return done

    with monkeypatch.context() as patch:
        patch.setattr(_launch, "fast", Counting())
        first = everything()
    assert served == [True, True]
    monkeypatch.setattr(_launch, "fast", None)
    for a, b in zip(first, everything()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("m", [2, 16])
def test_every_code(m):
    """All INT8 codes, -128 among them, and all pairs of E2M1 codes."""
    from klab_b200 import fp4, int8_weights
    from klab_b200.adapters import adapter_linear

    n, k = 192, 1024
    _, _, x, a, b, c, ids = case("bf16", m, n, k, 8, 2, seed=9)
    gen = torch.Generator(device="cuda").manual_seed(9)
    codes = torch.arange(n * k, device="cuda").view(n, k).add(torch.arange(n, device="cuda")[:, None]).sub(128).to(torch.int8)
    scales = torch.rand(n, generator=gen, device="cuda") * 1e-3 + 1e-3
    assert codes.unique().numel() == 256
    y = adapter_linear(x, int8_weights.Int8Weights(codes, scales), a, b, c, ids, output_dtype=torch.float32)
    close(y, f64(codes) * f64(scales)[:, None], x, a, b, c, ids, torch.float32)
    packed = (torch.arange(n * k // 2, device="cuda").view(n, k // 2) + torch.arange(n, device="cuda")[:, None] * 7).to(torch.uint8)
    w = fp4.FP4F16Weights(packed, (torch.rand(n, k // 32, generator=gen, device="cuda") * 0.01 + 0.01).half())
    assert packed.unique().numel() == 256
    close(adapter_linear(x, w, a, b, c, ids, output_dtype=torch.float32), f64(w.dequantize()), x, a, b, c, ids, torch.float32)
