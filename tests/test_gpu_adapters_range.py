"""Adapters beside the shared projection: values of x far apart and near the largest."""

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
