"""Batches whose sizes 32 bits do not hold are refused (tensors without memory)."""
import ctypes

import pytest
import torch

from fleet import mk
from fleet.latent import LatentBatch, LatentCache


def test_sizes_past_32_bits_are_refused():
    meta = lambda *s: torch.empty(*s, dtype=torch.int32, device="meta")  # noqa: E731
    LatentBatch(meta(2 ** 31 - 1, 1), meta(2 ** 31 - 1), meta(2 ** 31))
    for big in (2 ** 31, 2 ** 32 + 3):                    # (the second is 3 in 32 bits)
        for args in ((meta(big, 1), meta(big)), (meta(big, 1), meta(big), meta(big + 1)), (meta(2, big), meta(2))):
            with pytest.raises(ValueError):
                LatentBatch(*args)
    cache = LatentCache(2, 16, 64, 16, device="cpu")
    for args in ((2 ** 32 + 1, 1, 16), (1, 2 ** 32 + 1, 16), (1, 1, 2 ** 32 + 1)):
        with pytest.raises(ValueError):
            cache.workspace_bytes(*args)


def test_too_many_groups_are_refused():
    """Sequences are a group of the attention's work each, and these are counted in 31 bits at 5 and more a group."""
    if not mk.LIB_PATH.exists():
        pytest.skip("library not built")
    P, n = 1 << 20, 2 ** 29                               # an address that nothing reads
    l, b = mk.MkLatent(P, P, P, 4, 64, 512, 64), mk.MkLatentBatch(P, P, None, 1, n, 1)
    assert mk.lib().mk_latent_attend(ctypes.addressof(l), ctypes.addressof(b), P, 576, 576, n, 1, 0, 1.0, P, 512, 512, None, P, 1 << 40,
                                     None) == mk.MK_EINVAL
    assert b"groups" in mk.lib().mk_last_error()
