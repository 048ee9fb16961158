"""How near the attention's weights are in FP16, whose outputs have 11 bits themselves.

Every key is the rotary part's first value alone, so a score is one product of codes and pieces, exact until its factors:
with u = 2^-24 its logarithm to base 2, at most 32 in size, is off by 5 u 32 and its exponential by 4 u, together by
164 u < 2^-16 of a weight. The weights' four pieces are within 2^-15 + 2^-18 of each, or of 2^-33 of the row's largest, and
the products and sums of L tokens within 2 L u. So a value before its rounding is off by at most
b = (2 x 2^-16 + 2^-15 + 2^-18 + 2 L u + 2^-20) sum p |c| + 2^-33 L max |c|, and an output by that and half of the distance
between FP16's values there. Weights of 11 bits leave this bound: a weight that outweighs the others and is no power of two is
off by up to 2^-11, which is from half of that distance to all of it."""
import numpy as np
import pytest
import torch

import latent_ref as R
from test_gpu_latent import batch_of, f64, filled

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def half_step(v):
    """Half the distance between FP16's values at |v|, subnormal ones included."""
    return np.exp2(np.maximum(np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -24))), -14) - 11)


@pytest.mark.parametrize("n,d_c,heads", [(129, 128, 16), (256, 512, 16), (300, 200, 20), (640, 64, 5)])
def test_weights_of_fp16(n, d_c, heads):
    page, d_r = 64, 8
    cache, table = filled([n], page, d_c, d_r, seed=n)
    cache.scales.fill_(2.0 ** -7)
    # one key above the others, in the second tile: within 2^8 of the first tile's largest, so that its weight keeps its fraction;
    # two to share with, and the rest far below
    cache.scales[:, 1] = 2.0 ** -5
    cache.r_codes.zero_()
    ramp = torch.zeros(n, d_r, device=DEV)
    ramp[:, 0] = -14
    ramp[[0, n // 3], 0] = 0
    ramp[128, 0] = 3.5
    place = torch.arange(n, device=DEV)
    cache.r_codes[torch.tensor(table[0], device=DEV)[place // page].long(), place % page] = (ramp * 32).to(torch.float8_e4m3fn).view(torch.uint8)
    # as many sequences over these pages as there are blocks, so that a block takes one's tiles one after the other
    B = 148
    q = torch.zeros(B, heads, d_c + d_r, device=DEV).half()
    q[..., d_c] = torch.linspace(0.02, 1.5, B * heads, device=DEV).half().view(B, heads)      # (scores up to 5.25 e-folds: 7.6 doublings)
    out, lse = cache.attend(q, batch_of(table * B, [n] * B), 1.0, return_lse=True)
    want, want_lse, size, spread = R.attend(R.Cache(cache), f64(q), table * B, [n] * B, [1] * B, 1.0)
    assert spread.max() * np.log2(np.e) <= 32
    u = 2.0 ** -24
    b = (2 * 2.0 ** -16 + 2.0 ** -15 + 2.0 ** -18 + 2 * n * u + 2.0 ** -20) * size + 2.0 ** -33 * n * 448 * 2.0 ** -7
    off = np.abs(f64(out) - want)
    bound = half_step(np.abs(want) + b) + b
    assert (off <= bound).all(), ((off > bound).mean(), (off / bound).max())
    assert (np.abs(f64(lse) - want_lse) <= 2 * 2.0 ** -16 + 2 * n * u).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_what_is_not_finite_keeps_to_its_row(dtype):
    """Weights of neighbouring heads are packed side by side: a NaN or an infinity in one head's query, in every place of a group, and a
    NaN in a token that only the later rows see leave the others' bits as they were."""
    lens, counts, heads = [300, 70], [1, 3], 20
    cache, table = filled(lens, 64, 64, 16, seed=5)
    q = torch.randn(4, heads, 80, generator=torch.Generator(device=DEV).manual_seed(5), device=DEV).to(dtype)
    batch = batch_of(table, lens, counts)
    clean, clean_lse = cache.attend(q, batch, 0.1, return_lse=True)
    assert torch.isfinite(clean).all()
    for h in range(heads):
        bad = q.clone()
        bad[0, h, 3], bad[2, h, 70] = float("nan"), float("inf") if h % 2 else -float("inf")
        got, lse = cache.attend(bad, batch, 0.1, return_lse=True)
        hit = torch.zeros(4, heads, dtype=torch.bool, device=DEV)
        hit[0, h] = hit[2, h] = True
        assert got[hit].isnan().all() and lse[hit].isnan().all()
        assert torch.equal(got[~hit], clean[~hit]) and torch.equal(lse[~hit], clean_lse[~hit])
    cache.c_codes[table[1][1], 5, 9] = 127                  # token 69 of the second: its last row alone sees it
    got, lse = cache.attend(q, batch, 0.1, return_lse=True)
    assert got[3].isnan().all() and torch.equal(got[:3], clean[:3]) and torch.equal(lse[:3], clean_lse[:3])
