"""adapter_linear's refusals without a GPU: the C entry before any device call, and the Python layer's checks."""

import pytest
import torch

from klab_b200 import _native, adapters, fp4, int8_weights

FAKE = 1 << 20


def call(**k):
    return _native.lib().klab_adapter_linear(
        k.get("wfmt", _native.W_BF16), k.get("x", FAKE), k.get("w", FAKE), None, k.get("a", FAKE), FAKE, k.get("c", FAKE),
        k.get("ids", FAKE), FAKE, k.get("dt", 0), k.get("m", 2), k.get("n", 32), k.get("k", 64), k.get("rank", 8),
        k.get("adapters", 3), k.get("scratch", FAKE), k.get("bytes", 1 << 20), None, 0, None)


def test_c_refusals():
    for bad in ({"x": None}, {"a": None}, {"c": None}, {"ids": None}, {"scratch": None}, {"m": 0}, {"rank": 0}, {"adapters": 0},
                {"bytes": 2 * 8 * 4, "wfmt": _native.W_CBF16}):
        assert call(**bad) == _native.E_INVALID, bad
    for bad in ({"rank": 12}, {"rank": 264}, {"k": 60}, {"m": 65536}):
        assert call(**bad) == _native.E_SHAPE, bad
    for bad in ({"x": FAKE + 8}, {"a": FAKE + 2}, {"scratch": FAKE + 4}):
        assert call(**bad) == _native.E_ALIGN, bad
    for bad in ({"wfmt": _native.W_F32}, {"wfmt": _native.W_FP4_G16E}, {"dt": _native.DT_F16}):
        assert call(**bad) == _native.E_UNSUPPORTED, bad
    scratch = _native.lib().klab_adapter_scratch
    assert scratch(_native.W_CBF16, 2, 32, 64, 8) == 128 + 256 and scratch(_native.W_BF16, 0, 1, 64, 8) == _native.E_INVALID


def test_arguments():
    m, n, k, r, s = 2, 32, 64, 8, 3
    bf = dict(dtype=torch.bfloat16)
    good = dict(x=torch.zeros(m, k, **bf), w=torch.zeros(n, k, **bf), a=torch.zeros(s, r, k, **bf), b=torch.zeros(s, n, r, **bf),
                scales=torch.ones(s), ids=torch.zeros(m, dtype=torch.int32))
    for bad in ({"x": good["x"].float()}, {"x": good["x"][0]}, {"w": good["w"].half()}, {"w": good["w"][:, :32]},
                {"a": good["a"].float()}, {"a": good["a"][:, :7]}, {"b": good["b"][:, :31]}, {"b": good["b"].transpose(1, 2)},
                {"scales": good["scales"].half()}, {"scales": good["scales"][:2]}, {"ids": good["ids"].long()},
                {"ids": good["ids"][:1]}, {"x": torch.zeros(k, m, **bf).t()}, {"output_dtype": torch.float16},
                {"out": torch.zeros(m, n)}, {"out": torch.zeros(m, n + 1, **bf)}, {"out": good["w"].view(-1)[:m * n].view(m, n)},
                {"w": int8_weights.Int8Weights(torch.zeros(n, k, dtype=torch.int8), torch.zeros(n, 3))},
                {"w": int8_weights.Int8Weights(torch.zeros(n, k, dtype=torch.uint8), torch.zeros(n))},
                {"w": fp4.FP4F16Weights(torch.zeros(n, k // 2, dtype=torch.uint8), torch.zeros(n, k // 32))},
                {"a": torch.zeros(s, 12, k, **bf), "b": torch.zeros(s, n, 12, **bf)},
                {"x": good["x"].clone().requires_grad_()}):
        with pytest.raises(ValueError):
            adapters.adapter_linear(**{**good, **bad})
    with pytest.raises(ValueError, match="CUDA"):
        adapters.adapter_linear(**good)
