"""Calls of the latent attention's operators that no shape of test_gpu_latent.py makes: caches past 4 GiB and never written,
streams that a captured graph forks and joins, tensors dropped while a stream is busy, and what is refused on the GPU."""
import numpy as np
import pytest
import torch

import latent_ref as R
from fleet.latent import LatentBatch, LatentCache
from fleet.rope import Rope
from test_gpu_latent import U, batch_of, check_attend, f64, filled, ints, same

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def randn(*s, seed=0, dtype=torch.bfloat16):
    return torch.randn(*s, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def test_a_cache_past_4_gib():
    """The last pages of a cache whose codes pass 2^32 bytes (and 2^23 tokens)."""
    pages = 2 ** 32 // (64 * 512) + 9000
    cache = LatentCache(pages, 64, 512, 64, device=DEV)
    assert cache._c.numel() > 2 ** 32
    table = [[pages - 1, 3, pages - 2], [5, pages - 70000, 1]]
    lens, counts = [150, 129], [150, 129]
    c, r = randn(279, 512, seed=1), randn(279, 64, seed=2)
    batch = batch_of(table, lens, counts)
    cache.append(c, r, batch)
    used = sorted(sum(table, []))
    few = LatentCache(len(used), 64, 512, 64, device=DEV)               # the same pages alone
    small = [[used.index(p) for p in t] for t in table]
    few.append(c, r, batch_of(small, lens, counts))
    assert torch.equal(cache._c[used], few._c) and torch.equal(cache._r[used], few._r) and torch.equal(cache.scales[used], few.scales)
    rest = torch.ones(pages, dtype=torch.bool, device=DEV)
    rest[used] = False
    assert not cache.scales[rest].any() and int((cache._c.view(pages, -1)[:, ::4096] != 0).any(1).sum()) <= len(used)
    assert all(torch.equal(a, b) for a, b in zip(cache.read(batch, 279), few.read(batch_of(small, lens, counts), 279)))
    q = randn(2, 16, 576, seed=3)
    assert torch.equal(cache.attend(q, batch_of(table, lens), 0.1), few.attend(q, batch_of(small, lens), 0.1))


def test_pages_that_were_never_written():
    """Codes and scales of zero: every token scores 0 and adds 0."""
    cache = LatentCache(9, 64, 200, 24, device=DEV)
    table, lens = [[0, 1, 2], [3, 4, 5], [6, 7, 8]], [130, 1, 64]
    q = randn(3, 16, 224)
    out, lse = cache.attend(q, batch_of(table, lens), 0.1, return_lse=True)
    assert not out.any()
    assert torch.allclose(lse.cpu(), torch.tensor(lens).float().log()[:, None].expand(3, 16), rtol=0, atol=200 * U + 8 * U * 5)
    cache.append(randn(1, 200, seed=1), randn(1, 24, seed=2), LatentBatch(ints([[0, 1, 2]]), ints([130])))     # the last page alone
    check_attend(cache, q, table, lens, None, 0.1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_values_that_are_not_finite_do_not_count(dtype):
    """One by one and among finite ones, in a page's first tokens and later ones."""
    cache, table = filled([40] * 4, 16, 32, 8, seed=3)
    ref = R.Cache(cache)
    bad = [float("inf"), float("nan"), -float("inf"), 1.0]
    for step, lens in enumerate(([3] * 4, [20, 17, 16, 33])):
        counts = [3, 3, 2, 1] if step == 0 else [17, 14, 14, 30]
        T = sum(counts)
        c, r = randn(T, 32, seed=step, dtype=dtype), randn(T, 8, seed=step + 9, dtype=dtype)
        for i in range(0, T, 2):
            c[i, i % 32], r[i, (3 * i) % 8] = bad[i // 2 % 4], bad[(i // 2 + 1) % 4]
        cache.append(c, r, batch_of(table, lens, counts))
        ref.append((f64(c), f64(r)), table, lens, counts)
        same(cache, ref)


def step(cache, rope, c, r, q, batch, positions, **kw):
    """What a layer calls: turn, write, attend, read."""
    cache.append(c, rope(r, positions, **kw), batch, **kw)
    rope(q[..., 512:], positions, out=q[..., 512:], **kw)
    return cache.attend(q, batch, 0.1, **kw), *cache.read(batch, len(r), **kw)


def test_streams_that_a_captured_graph_forks_and_joins():
    lens = [90, 200, 31]
    cache, table = filled([n + 4 for n in lens], 64, 512, 64, seed=4)
    other, _ = filled([n + 4 for n in lens], 64, 512, 64, seed=4)
    rope, batch, positions = Rope.yarn(64, device=DEV), batch_of(table, lens), ints(lens) - 1
    c, r, q = randn(3, 512, seed=5), randn(3, 64, seed=6), randn(3, 16, 576, seed=7)
    qa, qb = q.clone(), q.clone()
    for each in (cache, other):                      # (one history: a page's scale keeps what it has grown to)
        step(each, rope, c, r, q.clone(), batch, positions)
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        qa.copy_(q)
        a = step(cache, rope, c, r, qa, batch, positions, stream=here)
        with torch.cuda.stream(side):
            qb.copy_(q)
        b = step(other, rope, c, r, qb, batch, positions, stream=side)
        here.wait_stream(side)
        both = [x + y for x, y in zip(a, b)]
    for seed in range(3):
        c.copy_(randn(3, 512, seed=seed + 20))
        q.copy_(randn(3, 16, 576, seed=seed + 30))
        graph.replay()
        torch.cuda.synchronize()
        want = step(cache, rope, c, r, q.clone(), batch, positions)
        assert all(torch.equal(x, w) and torch.equal(y, w) and torch.equal(s, w + w) for x, y, s, w in zip(a, b, both, want))


@pytest.mark.parametrize("raw", [False, True])
def test_tensors_dropped_while_the_stream_is_busy(raw):
    lens = [90, 200, 31]
    cache, table = filled([n + 4 for n in lens], 64, 512, 64, seed=8)
    rope = Rope.yarn(64, device=DEV)
    make = lambda: (randn(3, 512, seed=5), randn(3, 64, seed=6), randn(3, 16, 576, seed=7), batch_of(table, lens), ints(lens) - 1)  # noqa: E731
    want = step(cache, rope, *make())
    side, tensors = torch.cuda.Stream(), make()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)                # about 10 ms
    got = step(cache, rope, *tensors, stream=side.cuda_stream if raw else side)
    shapes = [(t.shape, t.dtype) for t in tensors if isinstance(t, torch.Tensor)] + [((3, 4), torch.int32), ((3,), torch.int32)] * 4
    del tensors
    again = [torch.full(s, 1, dtype=d, device=DEV) for s, d in shapes for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for g, w in zip(got, want)) and again


def test_calls_one_after_another_read_what_the_last_one_wrote():
    """Launches that start early wait all the same: a chain of appends and attentions, against the chain with a wait between."""
    lens = [60, 127, 5]
    a, table = filled([n + 50 for n in lens], 64, 512, 64, seed=9)
    b, _ = filled([n + 50 for n in lens], 64, 512, 64, seed=9)
    rope = Rope.yarn(64, device=DEV)
    qs = [randn(3, 16, 576, seed=10), randn(3, 16, 576, seed=10)]
    for _ in range(50):
        outs = []
        for cache, q in zip((a, b), qs):
            batch, positions = batch_of(table, lens), ints(lens) - 1
            torch.cuda.synchronize()
            for i in range(3):
                out = cache.attend(q, batch, 0.05)
                if cache is b:
                    torch.cuda.synchronize()
                cache.append(out[:, i], q[:, i, 512:], batch)
                if cache is b:
                    torch.cuda.synchronize()
                rope(q[..., 512:], positions, out=q[..., 512:])
                if cache is b:
                    torch.cuda.synchronize()
            outs.append(cache.attend(q, batch, 0.05))
        assert torch.equal(*outs) and torch.equal(*qs)
        lens = [n + 1 for n in lens]
    assert torch.equal(a._c, b._c) and torch.equal(a.scales, b.scales)


def test_refused_on_the_gpu():
    cache, table = filled([70, 3], 64, 512, 64)
    batch, rows = batch_of(table, [70, 3]), batch_of(table, [70, 3], [4, 2])
    c, r, q = randn(2, 512), randn(2, 64), randn(2, 16, 576)
    big = torch.zeros(2, 16, 2000, dtype=torch.bfloat16, device=DEV)
    cpu = LatentBatch(torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
    bad = ValueError
    for call in (
            lambda: cache.append(c.float(), r, batch), lambda: cache.append(c, r.half(), batch), lambda: cache.append(c[:1], r, batch),
            lambda: cache.append(c[:, :511], r, batch), lambda: cache.append(c.T.contiguous().T, r, batch), lambda: cache.append(c, r, cpu),
            lambda: cache.append(c[:1], r[:1], batch), lambda: cache.append(c.cpu(), r, batch), lambda: cache.append(c[0], r, batch),
            lambda: cache.read(batch, 3), lambda: cache.read(rows, 6, out=(c, r)), lambda: cache.read(batch, 2, out=(c, r.half())),
            lambda: cache.read(batch, 2, out=(c[:1].expand(2, 512), r)), lambda: cache.read(batch, 2, out=(big[:, 0, :512], big[:, 0, 500:564])),
            lambda: cache.attend(q[..., :575], batch, 1.0), lambda: cache.attend(q.float(), batch, 1.0), lambda: cache.attend(q[0], batch, 1.0),
            lambda: cache.attend(q[:1], batch, 1.0), lambda: cache.attend(q, cpu, 1.0), lambda: cache.attend(q.cpu(), batch, 1.0),
            lambda: cache.attend(q, batch, 1.0, out=q[..., :512]), lambda: cache.attend(q, batch, 1.0, out=big[..., :500]),
            lambda: cache.attend(q, batch, 1.0, out=big[:1, :, :512].expand(2, 16, 512)), lambda: cache.attend(q, batch, 1.0, out=big[..., :512].half()),
            lambda: cache.attend(q, batch, 1.0, out=cache._c.view(torch.bfloat16).view(-1)[:2 * 16 * 512].view(2, 16, 512))):
        with pytest.raises(bad):
            call()
    with pytest.raises(TypeError):
        cache.read(batch, 2, dtype=torch.float32)
    rope, pos = Rope.yarn(64, device=DEV), ints([1, 2])
    x = randn(2, 4, 192)
    for call in (lambda: rope(x, pos, 129), lambda: rope(x, pos, -1), lambda: rope(x[..., :63], pos), lambda: rope(x, pos[:1]), lambda: rope(x, ints([[1, 2]])),
                 lambda: rope(x, ints([1, 0, 2])[::2]), lambda: rope(x.transpose(1, 2), pos), lambda: rope(x.cpu(), pos), lambda: rope(x, pos.cpu()),
                 lambda: rope(x, pos, out=x[:, :3]), lambda: rope(x, pos, out=x.half()), lambda: rope(x[:, :2], pos, out=x[:, 1:3]),
                 lambda: rope(x, pos, out=x[:, :1].expand(2, 4, 192)), lambda: rope(x[:, 0], pos, out=x)):
        with pytest.raises(ValueError):
            call()
    for x in (x.float(), x.double()):
        with pytest.raises(TypeError):
            rope(x, pos)
    with pytest.raises(TypeError):
        rope(randn(2, 4, 64), pos.short())
    # nothing of it was written
    assert not big.any() and np.array_equal(c.float().cpu().numpy(), randn(2, 512).float().cpu().numpy())
