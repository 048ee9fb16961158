"""Lengths past the table, several rows a sequence: the rows' tokens go by the length as given, and those past the table are none."""
import numpy as np
import pytest
import torch

import latent_ref as R
from test_gpu_latent import batch_of, check_attend, f64, filled, same

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("lens,counts", [([70, 30], [10, 2]), ([65, 64], [1, 1]), ([200, 64], [300, 64]), ([66, 67], [2, 3]), ([64 + 1000, 5], [999, 5])])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_past_the_table(lens, counts, dtype):
    page, d_c, d_r = 16, 64, 16
    cache, table = filled([64, 64], page, d_c, d_r, seed=sum(lens))         # 4 pages each: 64 tokens
    ref = R.Cache(cache)
    T = sum(counts)
    g = torch.Generator(device=DEV).manual_seed(2)
    batch = batch_of(table, lens, counts)
    q = torch.randn(T, 20, d_c + d_r, generator=g, device=DEV).to(dtype)
    check_attend(cache, q, table, lens, counts, 0.2)
    c, r = torch.randn(T, d_c, generator=g, device=DEV).to(dtype), torch.randn(T, d_r, generator=g, device=DEV).to(dtype)
    cache.append(c, r, batch)
    ref.append((f64(c), f64(r)), table, lens, counts)
    same(cache, ref)
    got = cache.read(batch, T, dtype=dtype)
    row = 0
    for t, n, k in zip(table, lens, counts):
        tokens = ref.tokens(t, n)[:2]
        for i in range(k):
            at = n - k + i
            for v, w in zip(got, tokens):
                want = w[at] if 0 <= at < 64 else np.zeros(w.shape[1])
                assert torch.equal(v[row].cpu(), torch.tensor(want).to(dtype))
            row += 1
