"""Waits of the latent attention that run out: each ends after the cache's limit, here of a nanosecond, which any wait for memory
or for a product is past. The kernel ends all the same (a block waits for its own copies and products in flight, whatever the
limit), leaves NaN where a block gave up, and says so."""
import pytest
import torch

from fleet import mk
from test_gpu_latent import batch_of, filled

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("lens,heads,dtype", [([4000], 16, torch.bfloat16), ([700, 0, 3000], 20, torch.float16), ([9000], 128, torch.bfloat16)])
def test_a_wait_that_runs_out_is_reported(lens, heads, dtype):
    cache, table = filled(lens, 64, 128, 32, seed=heads)
    table = [list(t) + [-1] * (2 ** 14 - len(t)) for t in table]
    batch = batch_of(table, lens)
    q = torch.randn(len(lens), heads, 160, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(dtype)
    want, want_lse = cache.attend(q, batch, 0.1, return_lse=True)
    assert cache.status() == {"error": 0}
    limit, cache.wait_ns = cache.wait_ns, 1
    got, got_lse = cache.attend(q, batch, 0.1, return_lse=True)
    cache.wait_ns = limit
    with pytest.raises(mk.MkError) as e:
        cache.status()
    assert e.value.code == mk.MK_EDEVICE and e.value.status == {"error": 1}
    assert got.isnan().any() and (got.isnan() | (got == want)).all() and (got_lse.isnan() | (got_lse == want_lse)).all()
    again, again_lse = cache.attend(q, batch, 0.1, return_lse=True)      # the next call is sound, and the word stays
    assert torch.equal(again, want) and torch.equal(again_lse, want_lse)
    assert cache.status(raise_on_error=False) == {"error": 1}
    cache.reset()
    cache.attend(q, batch, 0.1)
    assert cache.status() == {"error": 0}
