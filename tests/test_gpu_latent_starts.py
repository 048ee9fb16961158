"""Starts that go down: what the call's rows and pages hold is undefined, but nothing else is touched, and the calls end."""
import pytest
import torch

from fleet.latent import LatentBatch
from test_gpu_latent import check_attend, filled, ints

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("starts", [[0, 3, 1, 4], [4, 0, 4, 0], [-5, 9, -5, 9], [0, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1], [2, 2, 2, 2], [3, 2, 1, 0]])
@pytest.mark.parametrize("many", [1, 40])
def test_nothing_else_is_touched(starts, many):
    lens = [70, 9, 130] * many
    cache, table = filled(lens + [20], 16, 64, 16, seed=3)
    other, mine = table[-1][:2], sorted({p for t in table[:-1] for p in t if p >= 0})
    before = cache._c.clone(), cache._r.clone(), cache.scales.clone()
    batch = LatentBatch(ints(table[:-1]), ints(lens), ints(starts[:3] * many + starts[3:]))
    rows = 4
    g = torch.Generator(device=DEV).manual_seed(1)
    c, r = torch.randn(rows, 64, generator=g, device=DEV).bfloat16(), torch.randn(rows, 16, generator=g, device=DEV).bfloat16()
    q = torch.randn(rows, 20, 80, generator=g, device=DEV).bfloat16()
    out = torch.full((rows + 2, 20, 64), 7.0, device=DEV).bfloat16()
    pair = torch.full((rows + 2, 64), 7.0, device=DEV).bfloat16(), torch.full((rows + 2, 16), 7.0, device=DEV).bfloat16()
    cache.attend(q, batch, 0.1, out=out[1:-1])
    cache.read(batch, rows, out=(pair[0][1:-1], pair[1][1:-1]))
    cache.append(c, r, batch)
    for t in (out, *pair):
        assert (t[[0, -1]] == 7).all()
    rest = [p for p in range(cache.pages) if p not in mine]
    assert set(other) <= set(rest)
    for now, then in zip((cache._c, cache._r, cache.scales), before):
        assert torch.equal(now[rest], then[rest])
    assert cache.status() == {"error": 0}
    check_attend(cache, q[:1], table[-1:], [20], None, 0.1)
