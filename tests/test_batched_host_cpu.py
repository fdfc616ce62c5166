"""Host side of the batched operators without a GPU: sizes of scratch."""

from klab_b200 import _native


def test_plain_scratch_stays_small():
    """t and the projection in FP32 for 64 MiB of rows at a time, and the few behind the last part."""
    scratch = _native.lib().klab_adapter_scratch
    for wfmt in (_native.W_CBF16, _native.W_I8_G64):
        for m in (1, 300, 1169, 1185, 2048, 65535):
            assert 4 * min(m, 1024) * 14336 < scratch(wfmt, m, 14336, 4096, 16) <= 2 ** 26 + 2 ** 21
        # Rows that are each past a part's size: two tiles and the rest of a third.
        assert scratch(wfmt, 100, 2 ** 24, 64, 8) == 48 * 4 * (2 ** 24 + 8)
