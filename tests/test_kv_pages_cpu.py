"""Batched 4-bit pages without a GPU: the oracle's own arithmetic, the host side of the C entry points (block offsets of
good and bad slots, refusals before any device call) and the Python layer's checks of arguments."""

import numpy as np
import pytest
import torch

from klab_b200 import _native, kv_pages
from oracle import kv_pages as ok

FAKE = 1 << 20  # an aligned address that no refused call may touch


def test_quantizer_bounds_and_ties():
    x = np.array([[7.0, 3.5, -3.5, 0.5, 1.5, -7.0, 2.5, 0.0] + [0.0] * 24])
    codes, scales = ok.quantize(x)
    assert scales[0, 0] == 1.0
    assert codes[0, :8].tolist() == [15, 12, 4, 8, 10, 1, 10, 8]  # ties to the even code value
    x = np.array([[np.nan, np.inf, -np.inf, 1.0] + [0.0] * 28, [0.0] * 32])
    codes, scales = ok.quantize(x)
    assert scales[:, 0].tolist() == [65504.0, 0.0]
    assert codes[0, :4].tolist() == [8, 15, 1, 8] and (codes[1] == 8).all()
    x = np.random.default_rng(0).standard_normal((50, 128))
    codes, scales = ok.quantize(x)
    step = np.repeat(scales, 32, -1).reshape(x.shape)
    assert (np.abs(ok.values(codes, scales) - x) <= step * (0.5 + 7 * 2.0 ** -11)).all()
    assert codes.min() >= 1 and codes.max() <= 15


@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_block_offsets_of_good_and_bad_slots(page, dim):
    offset = _native.lib().klab_kv_block_offset
    pages, heads = 5, 3
    size = page * dim * 9 // 8
    for slot in (0, 1, 15, 16, page - 1, page, 3 * page + page // 2, 5 * page - 1):
        for head in range(heads):
            want = (slot // page * heads + head) * size + slot % page // 16 * 18 * dim
            got = offset(slot, head, pages, heads, page, dim)
            assert got == want and got + 18 * dim <= pages * heads * size
    for slot in (-1, -2, -2 ** 31, 5 * page, 5 * page + 1, 2 ** 31 - 1):
        assert offset(slot, 0, pages, heads, page, dim) == -1
    assert offset(0, heads, pages, heads, page, dim) == offset(0, -1, pages, heads, page, dim) == -1
    # A long cache: the offset passes 32 bits.
    many = 2 ** 31 // page - 1
    slot = many * page - 1
    assert offset(slot, 7, many, 8, page, dim) == ((many - 1) * 8 + 7) * size + (page // 16 - 1) * 18 * dim > 2 ** 32
    for wrong in (0, 8, 24, 48, 2048):
        assert offset(0, 0, pages, heads, wrong, dim) == -1
    assert offset(0, 0, pages, heads, page, 96) == -1


def test_packed_order_is_a_permutation():
    for dim in (64, 128, 256):
        rng = np.random.default_rng(dim)
        codes = rng.integers(0, 16, (2, 16, dim))
        scales = rng.random((2, 16, dim // 32)).astype(np.float16).astype(float)
        block = ok.pack_block(codes[0], scales[0], codes[1], scales[1])
        nib = np.concatenate([block[:16 * dim] & 15, block[:16 * dim] >> 4])
        assert sorted(nib.tolist()) == sorted(codes.reshape(-1).tolist())
        assert sorted(block[16 * dim:].view("<f2").tolist()) == sorted(scales.reshape(-1).tolist())


def test_step_oracle_gives_pages_once():
    rng = np.random.default_rng(1)
    lengths, new = rng.integers(0, 90, 7), rng.integers(0, 60, 7)
    ids = rng.permutation(100)
    table = np.full((7, 12), -1)
    at = 0
    for i, n in enumerate(-(-lengths // 16)):
        table[i, :n] = ids[at:at + n]
        at += n
    out, after = ok.build_step(new, lengths, table, ids[at:], 100 - at, 16, 500)
    slots = out["slots"][:new.sum()]
    assert len(set(slots.tolist())) == new.sum() and out["result"] == 0
    used = after[after >= 0]
    assert len(set(used.tolist())) == len(used) == (-(-(lengths + new) // 16)).sum()


def refused(name, *args):
    return getattr(_native.lib(), name)(*args)


def test_c_refusals_come_before_any_device_call():
    step = lambda **k: refused("klab_kv_build_step", *[k.get(n, FAKE) for n in ("new", "len", "table", "free", "count")],  # noqa: E731
                               k.get("requests", 4), k.get("width", 4), k.get("pages", 8), k.get("page", 16),
                               k.get("most", 10), *[FAKE] * 7, None)
    assert step(new=None) == step(table=None) == step(most=0) == step(requests=0) == step(width=-1) == _native.E_INVALID
    assert step(requests=8193) == step(page=24) == step(page=8) == step(page=2048) == _native.E_SHAPE
    assert step(pages=2 ** 27) == step(width=2 ** 27) == _native.E_SHAPE
    free = lambda **k: refused("klab_kv_release", k.get("ended", FAKE), FAKE, FAKE, FAKE, k.get("count", FAKE),  # noqa: E731
                               k.get("requests", 4), 4, 8, k.get("page", 16), None)
    assert free(ended=None) == free(count=None) == free(requests=-1) == _native.E_INVALID
    assert free(page=20) == _native.E_SHAPE
    store = lambda **k: refused("klab_kv_store", k.get("k", FAKE), FAKE, k.get("dt", 0), k.get("ks", 256), 256, 128, 128,  # noqa: E731
                                k.get("pages", FAKE), k.get("slots", FAKE), k.get("tokens", 3), k.get("n", 9),
                                k.get("page", 16), k.get("heads", 2), k.get("dim", 128), None)
    assert store(k=None) == store(pages=None) == store(slots=None) == store(tokens=0) == store(n=0) == _native.E_INVALID
    assert store(dim=96) == store(page=17) == store(n=2 ** 28) == store(tokens=2 ** 30) == _native.E_SHAPE
    assert store(k=FAKE + 4) == store(ks=254) == store(pages=FAKE + 8) == _native.E_ALIGN
    assert store(dt=2) == _native.E_UNSUPPORTED
    read = lambda **k: refused("klab_kv_read", k.get("pages", FAKE), FAKE, k.get("out", FAKE), FAKE, k.get("dt", 0), 3, 9,  # noqa: E731
                               16, 2, k.get("dim", 128), None)
    assert read(pages=None) == read(out=None) == _native.E_INVALID
    assert read(dim=32) == _native.E_SHAPE and read(out=FAKE + 8) == _native.E_ALIGN

    def attend(**k):
        return refused("klab_kv_attention", k.get("q", FAKE), k.get("qs", 1024), k.get("dt", 0), FAKE, FAKE,
                       k.get("len", FAKE), FAKE, FAKE, k.get("scratch", FAKE), 1 << 40, k.get("tokens", 4),
                       k.get("requests", 4), k.get("width", 4), 8, k.get("page", 16), k.get("heads", 8), k.get("kvh", 2),
                       k.get("dim", 128), k.get("new", 1), 0.1, None)

    assert attend(q=None) == attend(len=None) == attend(scratch=None) == attend(tokens=0) == _native.E_INVALID
    assert attend(requests=0) == attend(new=0) == attend(heads=0) == _native.E_INVALID
    assert attend(dt=2) == _native.E_UNSUPPORTED
    for bad in ({"heads": 7}, {"heads": 130}, {"dim": 80}, {"new": 17}, {"page": 48}, {"requests": 8193}, {"width": 2 ** 28}):
        assert attend(**bad) == _native.E_SHAPE, bad


def tables(requests=3, width=4, pages=20):
    i32 = dict(dtype=torch.int32)
    return dict(lengths=torch.zeros(requests, **i32), table=torch.zeros((requests, width), **i32),
                free_pages=torch.arange(pages, **i32), free_count=torch.tensor([pages], **i32))


def test_step_arguments():
    t = tables()
    new = torch.ones(3, dtype=torch.int32)
    step = lambda new=new, page_size=16, max_tokens=9, **k: kv_pages.build_step(new, **{**t, **k}, page_size=page_size,  # noqa: E731
                                                                              max_tokens=max_tokens)
    for bad in ({"new": new.long()}, {"new": new[:2]}, {"lengths": t["lengths"].float()}, {"table": t["table"][:2]},
                {"table": t["table"].t()}, {"free_count": t["free_pages"][:2]}, {"page_size": 20}, {"page_size": 8},
                {"page_size": 16.0}, {"max_tokens": 0}, {"max_tokens": 2 ** 31}, {"lengths": t["lengths"][None]}):
        with pytest.raises(ValueError):
            step(**bad)
    with pytest.raises(ValueError, match="overlap"):
        step(lengths=t["table"].view(-1)[:3])
    with pytest.raises(ValueError, match="CUDA"):
        step()
    with pytest.raises(ValueError, match="ended"):
        kv_pages.release(new, **t, page_size=16)
    with pytest.raises(ValueError, match="CUDA"):
        kv_pages.release(new.bool(), **t, page_size=16)


def test_store_and_read_arguments():
    pages = kv_pages.empty_pages(4, 2, 16, 128, device="cpu")
    assert pages.shape == (4, 2, kv_pages.page_bytes(16, 128)) == (4, 2, 2304)
    k = torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    slots = torch.zeros(3, dtype=torch.int32)
    for args in ((k.float(), k.float(), pages, slots), (k, k.half(), pages, slots), (k[0], k[0], pages, slots),
                 (k, k, pages, slots.long()), (k, k, pages, slots[:2]), (k[:, :1], k[:, :1], pages, slots),
                 (k[:, :, :64], k[:, :, :64], pages, slots), (k, k, pages.float(), slots), (k, k, pages[:, :, :2300], slots),
                 (k.transpose(1, 2).contiguous().transpose(1, 2), k, pages, slots), (k[:0], k[:0], pages, slots[:0]),
                 (torch.zeros(3, 2, 130, dtype=torch.bfloat16)[:, :, 1:129], k, pages, slots)):
        with pytest.raises(ValueError):
            kv_pages.store(*args)
    with pytest.raises(ValueError, match="CUDA"):
        kv_pages.store(k, k, pages, slots)
    for bad in ((pages, slots, 96), (pages, slots.long(), 128), (pages, slots, 256), (pages, slots[None], 128)):
        with pytest.raises(ValueError):
            kv_pages.read(*bad)
    with pytest.raises(ValueError):
        kv_pages.read(pages, slots, 128, dtype=torch.float64)
    with pytest.raises(ValueError, match="CUDA"):
        kv_pages.read(pages, slots, 128)
    for bad in ((0, 2, 16, 128), (4, 2, 24, 128), (4, 2, 16, 100), (2 ** 27, 2, 16, 128)):
        with pytest.raises(ValueError):
            kv_pages.empty_pages(*bad, device="cpu")


def test_attention_arguments():
    pages = kv_pages.empty_pages(4, 2, 16, 128, device="cpu")
    q = torch.zeros(3, 8, 128, dtype=torch.bfloat16)
    t = tables()
    good = dict(q=q, pages=pages, table=t["table"], lengths=t["lengths"], starts=torch.arange(4, dtype=torch.int32))
    for bad in ({"q": q.float()}, {"q": q[:, :7]}, {"q": q[:, :, :64]}, {"q": q[0]}, {"q": q[:0]},
                {"q": q.transpose(0, 1).contiguous().transpose(0, 1)}, {"lengths": t["lengths"][:2]},
                {"starts": good["starts"][:3]}, {"starts": good["starts"].long()}, {"table": t["table"][0]},
                {"max_new": 0}, {"max_new": 17}, {"scale": 0.0}, {"scale": float("nan")}, {"scale": -1.0},
                {"out": q.half()}, {"out": q[:, :4]}, {"out": q}, {"q": torch.zeros(3, 130, 128, dtype=torch.bfloat16)}):
        with pytest.raises(ValueError):
            kv_pages.attention(**{**good, **bad})
    with pytest.raises(ValueError, match="CUDA"):
        kv_pages.attention(**good)
    with pytest.raises(ValueError, match="requires_grad"):
        kv_pages.attention(**{**good, "q": q.clone().requires_grad_()})


def test_binding_leaves_what_it_does_not_serve_to_the_wrappers():
    """Without a ready device every call comes back None (the wrapper's checks then decide); its own setup is checked."""
    from klab_b200 import _launch

    module = _launch.load_binding()
    pages = kv_pages.empty_pages(4, 2, 16, 128, device="cpu")
    k, slots = torch.zeros(3, 2, 128, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    t = tables()
    assert module.store(k, k, pages, slots) is None and module.store(k, k) is None and module.store(1, k, pages, None) is None
    assert module.read(pages, slots, 128, 0) is None and module.read(pages, slots, 128, None) is None
    q, starts = torch.zeros(3, 8, 128, dtype=torch.bfloat16), torch.arange(4, dtype=torch.int32)
    for scale, out in ((None, None), (0.5, q), (-1.0, None), ("x", None), (None, 3)):
        assert module.attention(q, pages, t["table"], t["lengths"], starts, 1, scale, out) is None
    assert module.build_step(t["lengths"], *t.values(), 16, 9, False) is None
    assert module.build_step(t["lengths"], *t.values(), 16.0, 9, None) is None
    x, a = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(3, 8, 64, dtype=torch.bfloat16)
    assert module.adapter_linear(0, x, x, None, a, a, t["lengths"], slots, None, False) is None
    with pytest.raises(ValueError):
        module.bind(0, 0, 0, 0, 0, 0, 0)
    with pytest.raises(ValueError):
        module.bind(1)
    with pytest.raises(ValueError):
        module.mark_ready(64)
