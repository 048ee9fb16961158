"""LatentCache on the GPU against the cache and the attention in 64 bits (latent_ref).

Codes and scales are whole numbers of a kind: equal. The attention's bounds, with u = 2^-24, for a row that
sees L tokens, d = d_c + d_r: a score is a sum of d products, off by at most (d + 8) u sum |q k| scale with the scales'
roundings, and q's pieces by 2^-22 of its row's largest value, below that; e = 2 (d + 64) u max_j (scale sum |q k|_j)
bounds twice that. A weight is exp of it, off by 2 e in all with its share of the sum, by 4 u from the exponential and by
2^-11 from its pieces; the products and sums with L tokens by 2 L u. So an output is off by at most
(2 e + 2^-11 + 2^-20 + 2 L u) sum p |c| and its own rounding, half a step; the log of the sum by e + (L + 64) u +
4 u |lse|."""
import numpy as np
import pytest
import torch

import latent_ref as R
from fleet.latent import LatentBatch, LatentCache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def offsets(counts):
    return [sum(counts[:i]) for i in range(len(counts) + 1)]


def batch_of(table, lens, counts=None):
    return LatentBatch(ints(table).view(len(lens), -1), ints(lens), None if counts is None else ints(offsets(counts)))


def f64(t):
    return t.double().cpu().numpy()


def filled(lens, page, d_c, d_r, seed=0, extra=0):
    """A cache of random codes for sequences of these lengths, and their table."""
    g = torch.Generator().manual_seed(seed)
    table, pages = R.pool(lens, page, g, extra=extra)
    cache = LatentCache(pages, page, d_c, d_r, device=DEV)
    gd = torch.Generator(device=DEV).manual_seed(seed)
    for codes in (cache.c_codes, cache.r_codes):
        codes.copy_((torch.randn(codes.shape, generator=gd, device=DEV) * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8))
    cache.scales.copy_(torch.exp2(torch.randint(-8, -5, (pages, 2), generator=gd, device=DEV).float()))
    return cache, table


def same(cache, ref):
    assert np.array_equal(f64(cache.scales), ref.scales)
    for got, want in zip((cache.c_codes, cache.r_codes), ref.codes):
        assert R.same_codes(got.cpu().numpy(), want)


def padding_is_zero(cache):
    assert not cache._c[..., cache.d_c:].any() and not cache._r[..., cache.d_r:].any()


SEQS = [([1], None), ([64], None), ([65], None), ([1, 130, 64, 0, 17], None), ([5, 200, 64, 0, 129, 1], [5, 100, 1, 0, 129, 1]),
        ([300], [300]), ([300], [173]), ([3, 4], [5, 4]), ([-2, 9], [1, 2])]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,counts", SEQS)
@pytest.mark.parametrize("page,d_c,d_r", [(64, 512, 64), (16, 200, 24), (128, 8, 8), (32, 136, 56)])
def test_append_and_read(lens, counts, page, d_c, d_r, dtype):
    cache, table = filled(lens, page, d_c, d_r, seed=len(lens))
    ref = R.Cache(cache)
    ks = counts or [1] * len(lens)
    T = sum(ks)
    g = torch.Generator(device=DEV).manual_seed(9)
    for spread in (1.0, 30.0, 0.01):              # scales that stay, grow and are far too wide
        c = (torch.randn(T, d_c, generator=g, device=DEV) * spread).to(dtype)
        r = (torch.randn(T, d_r, generator=g, device=DEV) * spread * 2).to(dtype)
        batch = batch_of(table, lens, counts)
        cache.append(c, r, batch)
        ref.append((f64(c), f64(r)), table, lens, ks)
        same(cache, ref)
        for out_dtype in (torch.bfloat16, torch.float16):
            got = cache.read(batch, T, dtype=out_dtype)
            row = 0
            for t, n, k in zip(table, lens, ks):
                want = ref.tokens(t, max(n, 0))[:2]
                for i in range(k):
                    pos = max(n, 0) - k + i
                    for v, w in zip(got, want):
                        w = torch.tensor(w[pos]).to(out_dtype) if pos >= 0 else torch.zeros_like(v[row])
                        assert torch.equal(v[row].cpu(), w.cpu())
                    row += 1
    padding_is_zero(cache)


def test_token_by_token_and_drafts_taken_back():
    """200 tokens one by one, with three drafts written beyond and taken back at every fifth."""
    page, d_c, d_r = 16, 64, 16
    cache, table = filled([210], page, d_c, d_r)
    ref = R.Cache(cache)
    g = torch.Generator(device=DEV).manual_seed(1)
    for n in range(1, 201):
        k = 4 if n % 5 == 0 else 1
        c = (torch.randn(k, d_c, generator=g, device=DEV) * torch.exp2(torch.randn(k, 1, generator=g, device=DEV) * 3)).bfloat16()
        r = torch.randn(k, d_r, generator=g, device=DEV).bfloat16()
        cache.append(c, r, batch_of(table, [n + k - 1], [k]))
        ref.append((f64(c), f64(r)), table, [n + k - 1], [k])
    same(cache, ref)


def test_one_append_is_many():
    """A chunk in one call holds the values of the same chunk page by page."""
    page, d_c, d_r = 32, 128, 64
    g = torch.Generator(device=DEV).manual_seed(2)
    c, r = torch.randn(100, d_c, generator=g, device=DEV).bfloat16(), torch.randn(100, d_r, generator=g, device=DEV).bfloat16()
    a, table = filled([100], page, d_c, d_r)
    b, _ = filled([100], page, d_c, d_r, seed=5)
    b.scales.fill_(1e9)                            # of other use: not this sequence's
    a.append(c, r, batch_of(table, [100], [100]))
    for at in range(0, 100, 32):
        n = min(100, at + 32)
        b.append(c[at:n], r[at:n], batch_of(table, [n], [n - at]))
    live = table[0][:4]
    assert torch.equal(a.scales[live], b.scales[live])
    got, want = a.read(batch_of(table, [100], [100]), 100), b.read(batch_of(table, [100], [100]), 100)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_extreme_values():
    page, d_c, d_r = 16, 16, 8
    cache, table = filled([16] * 9, page, d_c, d_r)
    ref = R.Cache(cache)
    inf, nan = float("inf"), float("nan")
    rows = [[0.0] * 16, [448.0] + [0.0] * 15, [449.0] + [1.0] * 15, [nan] * 16, [inf, -inf, 3.0, nan] * 4, [3e38] * 8 + [-3e38] * 8,
            [1e-38] * 16, [-0.0, 1e-12] * 8, [2.0 ** i for i in range(-20, -4)]]
    c = torch.tensor(rows, device=DEV).bfloat16()
    r = c[:, :8].contiguous()
    for n in (1, 2, 5):
        batch = batch_of(table, [n] * 9)
        cache.append(c, r, batch)
        ref.append((f64(c), f64(r)), table, [n] * 9, [1] * 9)
        same(cache, ref)
    read = cache.read(batch_of(table, [1] * 9), 9)[0]
    assert read[3].isnan().all() and read[4, :4].isnan().tolist() == [True, True, False, True] and read[4, 2] == 3


def test_what_is_outside_is_left_alone():
    """Pages outside the cache, lengths past the table, rows of nobody: nothing of it is written or read."""
    page, d_c, d_r = 16, 24, 8
    cache, _ = filled([64], page, d_c, d_r)
    before = R.Cache(cache)
    table = [[0, -1], [cache.pages, 1], [2, 2 ** 31 - 1], [3, -2 ** 31]]
    lens, counts = [20, 20, 40, 2 ** 31 - 1], [10, 10, 12, 2]
    T = sum(counts) + 3
    c, r = torch.randn(T, d_c, device=DEV).bfloat16(), torch.randn(T, d_r, device=DEV).bfloat16()
    batch = batch_of(table, lens, counts)
    cache.append(c, r, batch)
    before.append((f64(c), f64(r)), table, lens, counts)
    same(cache, before)
    out = torch.full((T, d_c), 7.0, device=DEV).bfloat16(), torch.full((T, d_r), 7.0, device=DEV).bfloat16()
    got = cache.read(batch, T, out=out)
    assert got[0] is out[0] and (out[0][-3:] == 7).all() and (out[1][-3:] == 7).all()
    fresh = cache.read(batch, T)
    assert not fresh[0][-3:].any()
    assert torch.equal(fresh[0][:-3], out[0][:-3])
    row = 0
    for t, n, k in zip(table, lens, counts):
        for i in range(k):
            pos = n - k + i
            p = t[pos // page] if pos < 2 * page else -1
            if not 0 <= p < cache.pages:
                assert not out[0][row].any() and not out[1][row].any()
            row += 1


def test_strides():
    page, d_c, d_r = 64, 512, 64
    a, table = filled([70, 3], page, d_c, d_r)
    b, _ = filled([70, 3], page, d_c, d_r)
    g = torch.Generator(device=DEV).manual_seed(3)
    for off, width in ((0, 584), (8, 592), (5, 585)):
        base = torch.randn(12, width, generator=g, device=DEV).bfloat16()
        c, r = base[:, off:off + 512], base[:, off + 512:off + 576]
        batch = batch_of(table, [70, 3], [10, 2])
        a.append(c, r, batch)
        b.append(c.contiguous(), r.contiguous(), batch)
        assert torch.equal(a._c, b._c) and torch.equal(a._r, b._r) and torch.equal(a.scales, b.scales)
        out = torch.zeros_like(base)
        a.read(batch, 12, out=(out[:, off:off + 512], out[:, off + 512:off + 576]))
        want = a.read(batch, 12)
        assert torch.equal(out[:, off:off + 512], want[0]) and torch.equal(out[:, off + 512:off + 576], want[1])
        assert not out[:, :off].any() and not out[:, off + 576:].any()


def check_attend(cache, q, table, lens, counts, scale, batch=None, ref=None, floor=0.0):
    ks = counts or [1] * len(lens)
    batch = batch or batch_of(table, lens, counts)
    out, lse = cache.attend(q, batch, scale, return_lse=True)
    T = sum(ks)
    want, want_lse, size, spread = R.attend(ref or R.Cache(cache), f64(q), table, lens, ks, scale)
    got, got_lse = f64(out)[:T], f64(lse)[:T]
    want, want_lse, size, spread = want[:T], want_lse[:T], size[:T], spread[:T]
    d, L = cache.d_c + cache.d_r, max(1, *lens)
    e = 2 * (d + 64) * U * spread
    eps = torch.finfo(q.dtype).eps
    bound = eps / 2 * np.abs(want) + (1 + eps) * (2 * e[..., None] + 2.0 ** -11 + 2.0 ** -20 + 2 * L * U) * size
    tiny = float(torch.finfo(q.dtype).smallest_normal) * eps / 2
    assert (np.abs(got - want) <= bound + floor + tiny).all(), (np.abs(got - want) - bound - floor).max()
    empty = np.isneginf(want_lse)
    assert np.array_equal(np.isneginf(got_lse), empty)
    d = np.abs(got_lse[~empty] - want_lse[~empty])
    assert (d <= (e + (L + 64) * U + 4 * U * np.abs(want_lse))[~empty]).all(), d.max()
    assert torch.equal(out[:T], cache.attend(q, batch, scale)[:T])          # the same bits again
    return out, lse


ATTEND = [([1], None), ([64], None), ([63, 65, 128, 129], None), ([1, 500, 0, 33, 257], None), ([0, 0], None), ([1027], None),
          ([6, 200, 64, 0, 129, 1], [5, 3, 1, 0, 129, 1]), ([300], [300]), ([3, 4, 90], [5, 4, 2]), ([2000, 5], [2, 4]), ([-3, 40], [1, 1])]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,counts", ATTEND)
@pytest.mark.parametrize("page,d_c,d_r,heads", [(64, 512, 64, 16), (16, 200, 24, 20), (128, 8, 8, 1), (32, 264, 40, 7), (64, 128, 64, 128)])
def test_attend(lens, counts, page, d_c, d_r, heads, dtype):
    cache, table = filled(lens, page, d_c, d_r, seed=heads)
    ks = counts or [1] * len(lens)
    q = torch.randn(sum(ks), heads, d_c + d_r, generator=torch.Generator(device=DEV).manual_seed(heads), device=DEV).to(dtype)
    check_attend(cache, q, table, lens, counts, 2.75 / (d_c + d_r) ** 0.5)


@pytest.mark.parametrize("scale", [0.0, 1e-4, 0.5, -0.1])
def test_attend_flat_and_steep(scale):
    cache, table = filled([700, 90], 64, 512, 64, seed=4)
    q = torch.randn(2, 16, 576, generator=torch.Generator(device=DEV).manual_seed(4), device=DEV).bfloat16()
    check_attend(cache, q, table, [700, 90], None, scale)


def test_attend_many_sequences():
    g = torch.Generator().manual_seed(6)
    lens = torch.randint(0, 300, (600,), generator=g).tolist()
    cache, table = filled(lens, 32, 64, 16, seed=6)
    q = torch.randn(600, 4, 80, generator=torch.Generator(device=DEV).manual_seed(6), device=DEV).bfloat16()
    check_attend(cache, q, table, lens, None, 0.3)


def test_attend_a_long_context():
    cache, table = filled([40000], 64, 512, 64, seed=7)
    q = torch.randn(1, 16, 576, generator=torch.Generator(device=DEV).manual_seed(7), device=DEV).bfloat16()
    check_attend(cache, q, table, [40000], None, 0.1147)


def test_attend_pages_of_very_different_scales():
    """Scales from 2^-32 to 2^32 side by side: what weighs is the product of weight and value."""
    lens = [400, 333]
    cache, table = filled(lens, 16, 128, 32, seed=8)
    g = torch.Generator(device=DEV).manual_seed(8)
    q = torch.randn(2, 16, 160, generator=g, device=DEV).bfloat16()
    for spread in (6, 32):
        cache.scales.copy_(torch.exp2(torch.randint(-spread, spread + 1, (cache.pages, 2), generator=g, device=DEV).float()))
        # scores that stay near one another however wide a page is
        check_attend(cache, q, table, lens, None, 2.0 ** -(spread + 12))


def test_attend_scores_that_rise_along_the_context():
    """The largest score comes last and far above what came before, tile after tile."""
    page, d_c, d_r, n = 64, 64, 16, 1000
    cache, table = filled([n], page, d_c, d_r, seed=9)
    ramp = torch.zeros(n, d_r)
    ramp[:, 0] = torch.arange(n) * 0.4
    cache.append(torch.randn(n, d_c, device=DEV).bfloat16(), ramp.to(DEV).bfloat16(), batch_of(table, [n], [n]))
    q = torch.zeros(1, 16, 80, device=DEV).bfloat16()
    q[..., 64] = torch.tensor([1.0, -1.0, 0.1, 8.0] * 4)
    check_attend(cache, q, table, [n], None, 1.0)


def test_attend_widely_spread_queries():
    cache, table = filled([300], 64, 512, 64, seed=10)
    g = torch.Generator(device=DEV).manual_seed(10)
    q = torch.randn(1, 16, 576, generator=g, device=DEV)
    q = (q * torch.exp2(torch.randint(-12, 3, q.shape, generator=g, device=DEV).float())).bfloat16()
    check_attend(cache, q, table, [300], None, 0.1)
    for power in (-60, 60):
        check_attend(cache, (q.float() * 2.0 ** power).bfloat16(), table, [300], None, 0.1 * 2.0 ** -power)


def test_attend_strides_and_rows_of_nobody():
    cache, table = filled([100, 30], 64, 512, 64, seed=11)
    g = torch.Generator(device=DEV).manual_seed(11)
    for off in (0, 3):
        base = torch.randn(6, 16 * 600 + 8, generator=g, device=DEV).bfloat16()
        q = base[:, off:off + 9600].unflatten(1, (16, 600))[..., :576]
        big = torch.full((16, 6, 520), 7.0, device=DEV).bfloat16()
        out = big.transpose(0, 1)[..., off:off + 512]
        batch = batch_of(table, [100, 30], [3, 1])
        got = cache.attend(q, batch, 0.1, out=out)
        assert got is out
        want, _ = check_attend(cache, q.contiguous(), table, [100, 30], [3, 1], 0.1)
        assert torch.equal(out[:4], want[:4])
        assert (out[4:] == 7).all() and (big[..., :off] == 7).all() and (big[..., off + 512:] == 7).all()


def test_attend_nothing_of_masked_places_comes_through():
    """NaN codes behind a sequence's end, in later drafts' tokens, in unused pages; scales that are NaN there."""
    lens, counts = [70, 100, 0], [1, 4, 1]
    cache, table = filled(lens, 64, 512, 64, seed=12)
    q = torch.randn(6, 16, 576, generator=torch.Generator(device=DEV).manual_seed(12), device=DEV).bfloat16()
    clean, lse = check_attend(cache, q, table, lens, counts, 0.1)
    for codes in (cache.c_codes, cache.r_codes):
        codes[table[0][1], 6:] = 127
        codes[table[1][1], 36:] = 255
        codes[[p for p in range(cache.pages) if p not in table[0] + table[1]]] = 127
    cache.scales[[p for p in range(cache.pages) if p not in table[0] + table[1]]] = float("nan")
    got, got_lse = cache.attend(q, batch_of(table, lens, counts), 0.1, return_lse=True)
    assert torch.equal(got, clean) and torch.equal(got_lse, lse)
    cache.c_codes[table[1][1], 34, 5] = 127                 # token 98 of the second: its rows 2 and 3 see it
    cache.r_codes[table[1][1], 35, 0] = 127                 # token 99: its row 3 alone
    got, got_lse = cache.attend(q, batch_of(table, lens, counts), 0.1, return_lse=True)
    assert torch.equal(got[:3], clean[:3]) and got[3:5].isnan().all() and not got[5].any()
    assert got_lse[3:5].isnan().all() and torch.equal(got_lse[:3], lse[:3])


def test_attend_a_query_that_is_not_finite_keeps_to_its_head():
    cache, table = filled([90, 80], 64, 512, 64, seed=13)
    q = torch.randn(2, 16, 576, generator=torch.Generator(device=DEV).manual_seed(13), device=DEV).bfloat16()
    batch = batch_of(table, [90, 80])
    clean = cache.attend(q, batch, 0.1)
    q[0, 3, 7], q[1, 15, 570] = float("nan"), float("inf")
    got = cache.attend(q, batch, 0.1)
    hit = torch.zeros(2, 16, dtype=torch.bool)
    hit[0, 3] = hit[1, 15] = True
    assert got[hit].isnan().all() and torch.equal(got[~hit], clean[~hit])


def test_attend_pages_outside_hold_no_token():
    lens = [150, 64, 20]
    cache, table = filled(lens, 16, 64, 16, seed=14, extra=1)
    q = torch.randn(3, 16, 80, generator=torch.Generator(device=DEV).manual_seed(14), device=DEV).bfloat16()
    table[0][3], table[0][9], table[1][0] = -1, cache.pages, 2 ** 31 - 1
    table[2] = [-5] * len(table[2])
    check_attend(cache, q, table, lens, None, 0.2)
    long = [2 ** 31 - 1, 64, 20]                            # past the table: the table's end
    cut = [len(table[0]) * 16, 64, 20]
    got = cache.attend(q, batch_of(table, long), 0.2)
    assert torch.equal(got, cache.attend(q, batch_of(table, cut), 0.2))


def test_a_step_together():
    """Append, then attend over what was written, step after step, several sequences at different places."""
    page, d_c, d_r, heads = 32, 128, 64, 16
    lens = [1, 30, 95]
    cache, table = filled([n + 8 for n in lens], page, d_c, d_r, seed=15)
    ref = R.Cache(cache)
    g = torch.Generator(device=DEV).manual_seed(15)
    for _ in range(6):
        c, r = torch.randn(3, d_c, generator=g, device=DEV).bfloat16(), torch.randn(3, d_r, generator=g, device=DEV).bfloat16()
        q = torch.randn(3, heads, d_c + d_r, generator=g, device=DEV).bfloat16()
        batch = batch_of(table, lens)
        cache.append(c, r, batch)
        ref.append((f64(c), f64(r)), table, lens, [1] * 3)
        same(cache, ref)
        check_attend(cache, q, table, lens, None, 0.15, batch, ref)
        lens = [n + 1 for n in lens]


def test_streams_and_a_captured_graph():
    lens = [90, 200, 0, 31]
    cache, table = filled([n + 4 for n in lens], 64, 512, 64, seed=16)
    g = torch.Generator(device=DEV).manual_seed(16)
    c, r = torch.randn(4, 512, generator=g, device=DEV).bfloat16(), torch.randn(4, 64, generator=g, device=DEV).bfloat16()
    q = torch.randn(4, 16, 576, generator=g, device=DEV).bfloat16()
    batch = batch_of(table, lens)

    def step(**kw):
        cache.append(c, r, batch, **kw)
        return cache.attend(q, batch, 0.1, **kw), *cache.read(batch, 4, **kw)
    want = step()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for s in (side, side.cuda_stream):
        got = step(stream=s)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step())
    for grow in (1, 0, 2):
        batch.lens.add_(grow)
        q.copy_(torch.randn(4, 16, 576, generator=g, device=DEV))
        c.copy_(torch.randn(4, 512, generator=g, device=DEV))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = cache.attend(q, batch, 0.1), *cache.read(batch, 4)
        assert all(torch.equal(a, b) for out in outs for a, b in zip(out, want))


def test_two_calls_at_once():
    cache, table = filled([3000, 20], 64, 512, 64, seed=17)
    qs = [torch.randn(2, 16, 576, generator=torch.Generator(device=DEV).manual_seed(i), device=DEV).bfloat16() for i in range(2)]
    batch = batch_of(table, [3000, 20])
    want = [cache.attend(q, batch, 0.1) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [cache.attend(qs[i % 2], batch, 0.1, stream=streams[i % 2]) for i in range(60)]
    torch.cuda.synchronize()
    assert all(torch.equal(v, want[i % 2]) for i, v in enumerate(got))


def test_nothing_to_do():
    cache = LatentCache(2, 16, 64, 16, device=DEV)
    empty = LatentBatch(ints([]).view(0, 1), ints([]))
    cache.append(torch.empty(0, 64, device=DEV).half(), torch.empty(0, 16, device=DEV).half(), empty)
    assert cache.read(empty, 0)[0].shape == (0, 64)
    assert cache.attend(torch.empty(0, 16, 80, device=DEV).half(), empty, 1.0).shape == (0, 16, 64)
    rows = LatentBatch(ints([]).view(0, 1), ints([]), ints([0]))
    assert not cache.read(rows, 3)[0].any()
    out = torch.full((3, 16, 64), 7.0, device=DEV).half()
    cache.attend(torch.zeros(3, 16, 80, device=DEV).half(), rows, 1.0, out=out)
    cache.append(torch.ones(3, 64, device=DEV).half(), torch.ones(3, 16, device=DEV).half(), rows)
    assert (out == 7).all() and not cache._c.any() and not cache.scales.any()
