"""Host side of the batched operators on the GPU: what a caller sees when something runs out or is missing."""

import pytest
import torch

from test_gpu_kv_pages import i32, native  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture
def little_memory():
    """The caching allocator refuses more than 64 MiB above what it holds; nothing of the GPU's memory is used up."""
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + 2 ** 26) / total)
    yield
    torch.cuda.set_per_process_memory_fraction(1.0)


@pytest.mark.parametrize("binding", [True, False])
def test_out_of_memory_is_torchs_error(little_memory, binding, monkeypatch):
    """What a server catches to evict or retry, whichever way the call takes."""
    from klab_b200 import _launch, kv_pages
    from klab_b200.adapters import adapter_linear

    bf = dict(device="cuda", dtype=torch.bfloat16)
    buf = kv_pages.empty_pages(2, 8, 16, 256)
    buf.zero_()
    lengths, table, free, count = i32([0]), i32([[-1]]), i32([0, 1]), i32([2])
    slots = torch.zeros(2 ** 17, device="cuda", dtype=torch.int32)
    x, w, a, b = torch.zeros(2 ** 14, 16, **bf), torch.zeros(2 ** 16, 16, **bf), torch.zeros(1, 8, 16, **bf), torch.zeros(1, 2 ** 16, 8, **bf)
    c, ids = torch.zeros(1, device="cuda"), torch.zeros(2 ** 14, device="cuda", dtype=torch.int32)
    kv_pages.read(buf, slots[:1], 256)
    assert _launch.fast is not None
    if not binding:
        monkeypatch.setattr(_launch, "fast", None)
    for call in (lambda: kv_pages.read(buf, slots, 256, dtype=torch.float32),
                 lambda: kv_pages.build_step(i32([1]), lengths, table, free, count, page_size=16, max_tokens=2 ** 27),
                 lambda: adapter_linear(x, w, a, b, c, ids)):
        with pytest.raises(torch.OutOfMemoryError):
            call()
    assert not kv_pages.read(buf, slots[:3], 256)[0].any()  # and goes on


def test_without_the_binding(monkeypatch, tmp_path):
    """A build without it (no headers of torch): the same results through ctypes, and a warning once."""
    from klab_b200 import _launch, kv_pages

    buf = kv_pages.empty_pages(2, 2, 16, 64)
    k = torch.randn(5, 2, 64, device="cuda").bfloat16()
    slots = i32([3, 17, -1, 4, 30])
    kv_pages.store(k, k, buf, slots)
    want = kv_pages.read(buf, slots, 64)
    monkeypatch.setattr(_launch, "fast", None)
    monkeypatch.setattr(_launch, "_ready", set())
    monkeypatch.setattr(_launch, "BINDING", tmp_path / "klab_torch.so")
    buf.zero_()
    with pytest.warns(RuntimeWarning, match="ctypes"):
        kv_pages.store(k, k, buf, slots)
    assert _launch.fast is None
    for got, w in zip(kv_pages.read(buf, slots, 64), want):
        assert torch.equal(got, w)
