"""The latent attention where a table is so wide, for so many heads, that a place of its work is several units: short sequences
behind a table of 2^30 tokens, one row of it for all sequences (stride 0), split within their groups by the blocks' runs."""
import numpy as np
import pytest
import torch

import latent_ref as R
from fleet.latent import LatentBatch
from test_gpu_latent import check_attend, filled, ints

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HEADS = 1024


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens", [[300, 0, 3000, 65], [1] * 3 + [1025], [64 + 200 * i for i in range(16)]])       # places of 4, 4 and 16 units
def test_coarse_places(lens, dtype):
    n = len(lens)
    cache, table = filled([max(lens)], 64, 40, 16, seed=n)
    wide = torch.full((1, 2 ** 24), -1, dtype=torch.int32, device=DEV)
    wide[0, :len(table[0])] = ints(table[0])
    batch = LatentBatch(wide.expand(n, 2 ** 24), ints(lens))
    q = torch.randn(n, HEADS, 56, generator=torch.Generator(device=DEV).manual_seed(n), device=DEV).to(dtype)
    # (the bound's floor: weights within 2^-30 of a row's largest, see test_gpu_latent_groups.py)
    ref = R.Cache(cache)
    spread = float(cache.scales[:, 0].max() / cache.scales[:, 0].min())
    floor = 2.0 ** -30 * spread * np.array([np.abs(ref.tokens(table[0], m)[0]).sum(0) for m in lens])[:, None]
    check_attend(cache, q, table * n, lens, None, 0.3, batch=batch, ref=ref, floor=floor)
    assert cache.status() == {"error": 0}
