"""Batches whose sizes 32 bits do not hold are refused (tensors without memory)."""
import pytest
import torch

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
