"""The latent attention with 32 rows a group: BF16, 64 rows or more for each sequence, and a table that is wide enough
for that many tokens (here 2^20, its places behind the sequences' pages being in no cache)."""
import numpy as np
import pytest
import torch

import latent_ref as R
from test_gpu_latent import batch_of, filled
from test_gpu_latent import check_attend as check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TOKENS = 2 ** 20


def widened(table, page):
    return [list(t) + [-1] * (TOKENS // page - len(t)) for t in table]


def check_attend(cache, q, table, lens, counts, scale):
    """check_attend, and where a value's heavy tokens are all zero there: the weights are within 2^-30 of the row's largest,
    not nearer. x = 2^7 p (p: softmax x the page's scale, over its largest so far, which the running one is at most 2^8
    above) is three E5M2 pieces x1 + x2 / 8 + x3 / 64, whose last step is E5M2's smallest, 2^-16, over 64: x is off by at
    most 2^-23, p by 2^-30. So a value is off by at most 2^-30 max(p) sum |code|, which is no more than
    2^-30 (largest scale / smallest) sum |code x scale| of the sequence's tokens."""
    ref, rows = R.Cache(cache), []
    for t, n, k in zip(table, lens, counts or [1] * len(lens)):
        c = ref.tokens(t, max(n, 0))[0]
        rows += [np.abs(c).sum(0)] * k
    spread = float(cache.scales[:, 0].max() / cache.scales[:, 0].min())
    return check(cache, q, table, lens, counts, scale, ref=ref, floor=2.0 ** -30 * spread * np.array(rows)[:, None])


def queries(rows, heads, d, seed, dtype=torch.bfloat16):
    return torch.randn(rows, heads, d, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


@pytest.mark.parametrize("lens,counts,heads", [([1], None, 64), ([1027, 1], None, 65), ([500, 0, 33, 257], None, 128), ([300], [300], 16), ([300], [300], 7),
                                               ([6, 200, 64, 0, 129, 1], [5, 3, 1, 0, 129, 1], 20), ([3, 4, 90], [5, 4, 2], 128),
                                               ([2000, 5], [2, 4], 80), ([-3, 40], [1, 1], 80), ([0, 0], None, 128), ([9000], None, 128)])
@pytest.mark.parametrize("page,d_c,d_r", [(64, 512, 64), (16, 200, 24), (128, 8, 8)])
def test_attend(lens, counts, heads, page, d_c, d_r):
    cache, table = filled(lens, page, d_c, d_r, seed=heads)
    q = queries(sum(counts or [1] * len(lens)), heads, d_c + d_r, heads)
    check_attend(cache, q, widened(table, page), lens, counts, 2.75 / (d_c + d_r) ** 0.5)


def test_scores_that_rise_along_the_context():
    page, d_c, d_r, n = 64, 64, 16, 1000
    cache, table = filled([n], page, d_c, d_r, seed=9)
    ramp = torch.zeros(n, d_r)
    ramp[:, 0] = torch.arange(n) * 0.4
    cache.append(torch.randn(n, d_c, device=DEV).bfloat16(), ramp.to(DEV).bfloat16(), batch_of(table, [n], [n]))
    q = torch.zeros(1, 64, 80, device=DEV).bfloat16()
    q[..., 64] = torch.tensor([1.0, -1.0, 0.1, 8.0] * 16)
    check_attend(cache, q, widened(table, page), [n], None, 1.0)


def test_nothing_of_masked_places_comes_through():
    lens, counts, heads = [70, 100, 0], [1, 4, 1], 64
    cache, table = filled(lens, 64, 512, 64, seed=12)
    wide = widened(table, 64)
    q = queries(6, heads, 576, 12)
    clean, lse = check_attend(cache, q, wide, lens, counts, 0.1)
    unused = [p for p in range(cache.pages) if p not in table[0] + table[1]]
    for codes in (cache.c_codes, cache.r_codes):
        codes[table[0][1], 6:] = 127
        codes[table[1][1], 36:] = 255
        codes[unused] = 127
    cache.scales[unused] = float("nan")
    got, got_lse = cache.attend(q, batch_of(wide, lens, counts), 0.1, return_lse=True)
    assert torch.equal(got, clean) and torch.equal(got_lse, lse)
    cache.c_codes[table[1][1], 34, 5] = 127                 # token 98 of the second: its rows 2 and 3 see it
    cache.r_codes[table[1][1], 35, 0] = 127                 # token 99: its row 3 alone
    q[0, 3, 7], q[1, 63, 570] = float("nan"), float("inf")  # and two heads of their own
    got, got_lse = cache.attend(q, batch_of(wide, lens, counts), 0.1, return_lse=True)
    bad = torch.zeros(6, heads, dtype=torch.bool, device=DEV)
    bad[3:5] = True
    bad[0, 3] = bad[1, 63] = True
    assert got[bad].isnan().all() and got_lse[bad].isnan().all()
    assert torch.equal(got[~bad], clean[~bad]) and torch.equal(got_lse[~bad], lse[~bad])


def test_strides_pages_outside_and_rows_of_nobody():
    lens, counts = [150, 64], [3, 1]
    cache, table = filled(lens, 16, 512, 64, seed=11, extra=1)
    table[0][3], table[1][0] = cache.pages, 2 ** 31 - 1
    wide = widened(table, 16)
    for off in (0, 3):
        base = queries(6, 64 * 600 + 8, 1, 11)[..., 0]
        q = base[:, off:off + 38400].unflatten(1, (64, 600))[..., :576]
        big = torch.full((64, 6, 520), 7.0, device=DEV).bfloat16()
        out = big.transpose(0, 1)[..., off:off + 512]
        cache.attend(q, batch_of(wide, lens, counts), 0.1, out=out)
        want, _ = check_attend(cache, q.contiguous(), wide, lens, counts, 0.1)
        assert torch.equal(out[:4], want[:4])
        assert (out[4:] == 7).all() and (big[..., :off] == 7).all() and (big[..., off + 512:] == 7).all()


def test_a_workspace_is_enough_for_any_table():
    """What a call asks for does not go by the table: the same cache, rows and heads behind a narrow and a wide one."""
    cache, table = filled([777], 32, 128, 32, seed=3)
    q = queries(1, 64, 160, 3)
    for t in (table, widened(table, 32), table):
        check_attend(cache, q, t, [777], None, 0.1)
    assert np.isfinite(cache.attend(q, batch_of(table, [777]), 0.1).float().cpu().numpy()).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,heads,d_c", [([20000], 16, 512), ([12345], 3, 200), ([15000, 9000], 16, 136), ([20000, 0, 70], 5, 64), ([9600], 40, 128)])
def test_few_rows_of_long_sequences(lens, heads, d_c, dtype):
    """Partial sums of all blocks for few groups: the join that reads several of a row's side by side."""
    cache, table = filled(lens, 64, d_c, 32, seed=heads)
    check_attend(cache, queries(len(lens), heads, d_c + 32, heads, dtype), widened(table, 64), lens, None, 2.75 / (d_c + 32) ** 0.5)


@pytest.mark.parametrize("heads", [16, 20])
def test_empty_sequences_behind_shared_groups(heads):
    """A run that ends a group of several and goes on with sequences that hold nothing, again and again."""
    lens = [2000, 0, 0, 1500, 0, 900, 0, 0, 0] * 3
    cache, table = filled(lens, 64, 256, 32, seed=heads)
    q = queries(len(lens), heads, 288, heads)
    first = None
    for _ in range(20):
        out, lse = cache.attend(q, batch_of(table, lens), 0.1, return_lse=True)
        first = first or (out, lse)
        assert torch.equal(out, first[0]) and torch.equal(lse, first[1])
    check_attend(cache, q, table, lens, None, 0.1)
