"""Calls whose rows or heads 32 bits do not hold are refused before anything is done (rows that are one row in memory: 2^32 + 3
of them are 3 in 32 bits)."""
import pytest
import torch

from fleet.latent import LatentBatch, LatentCache
from fleet.rope import Rope

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
MANY = 2 ** 32 + 3


def call(name):
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    cache = LatentCache(4, 16, 8, 8, device=DEV)
    batch = LatentBatch(ints([[0], [1]]), ints([2, 1]), ints([0, 2, 3]))
    row = torch.ones(1, 8, dtype=torch.bfloat16, device=DEV)
    rows = row.expand(MANY, 8)
    if name == "append":
        return cache, lambda: cache.append(rows, rows, batch)
    if name == "read":
        return cache, lambda: cache.read(batch, MANY)
    if name == "attend rows":
        return cache, lambda: cache.attend(torch.ones(1, 1, 16, dtype=torch.bfloat16, device=DEV).expand(MANY, 1, 16), batch, 1.0)
    if name == "attend heads":
        return cache, lambda: cache.attend(torch.ones(1, 1, 16, dtype=torch.bfloat16, device=DEV).expand(3, MANY, 16), batch, 1.0)
    rope = Rope(torch.ones(4, dtype=torch.float64, device=DEV))
    x = row[:, None]
    if name == "rope tokens":
        return cache, lambda: rope(x.expand(MANY, 1, 8), torch.zeros(1, dtype=torch.int64, device=DEV).expand(MANY))
    return cache, lambda: rope(x.expand(1, MANY, 8), ints([0]))


@pytest.mark.parametrize("name", ["append", "read", "attend rows", "attend heads", "rope tokens", "rope heads"])
def test_refused(name):
    cache, f = call(name)
    torch.cuda.reset_peak_memory_stats()
    with pytest.raises(ValueError):
        f()
    torch.cuda.synchronize()
    assert not cache._c.any() and not cache.scales.any() and torch.cuda.max_memory_allocated() < 2 ** 30
