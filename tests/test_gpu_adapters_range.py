"""Adapters beside the shared projection: values of x far apart and near the largest, and
many rows."""

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
