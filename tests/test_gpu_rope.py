"""Rope on the GPU against rotary positions in 64 bits.

An angle is off by at most 2 pi x (2^-25 of the turn's rounding to FP32 and, at positions up to 2^30, 2^-24 of the
product's two roundings in 64 bits), sincospif by 2 units of 2^-24, the scale and the two products and their sum by
3 x 2^-24: together below 2^-20 (|a| + |b|) scale; the output's own rounding is half a step."""
import numpy as np
import pytest
import torch

import latent_ref as R
from fleet.capture import YARN, rope_tables
from fleet.rope import Rope

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def inv_freq(dim):
    return torch.tensor(10000.0 ** -(np.arange(0, dim, 2) / dim), dtype=torch.float64, device=DEV)


def expect(x, positions, rope, start):
    f = lambda v: v.double().cpu().numpy()  # noqa: E731
    y, size = R.rope(f(x), positions.tolist(), rope.inv_freq.cpu().numpy(), rope.scale, rope.layout, start)
    return torch.tensor(y), torch.tensor(size)


def close(got, want, size):
    got, eps = got.double().cpu(), torch.finfo(got.dtype).eps
    assert got.shape == want.shape
    bound = eps / 2 * want.abs() + (1 + eps) * 2.0 ** -20 * size
    assert ((got - want).abs() <= bound).all(), ((got - want).abs() - bound).max()
    assert torch.equal(got[size == 0], want[size == 0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["half", "interleaved", "pairs_to_half"])
@pytest.mark.parametrize("T,H,W,dim,start", [(1, 16, 64, 64, 0), (5, 3, 192, 64, 128), (7, 1, 2, 2, 0), (3, 5, 96, 80, 8), (4, 2, 33, 30, 1),
                                             (2, 3, 512, 512, 0), (2, 2, 600, 400, 40), (1, 70, 16, 16, 0), (130, 4, 24, 16, 8), (3, 2, 300, 258, 42)])
def test_layouts(T, H, W, dim, start, layout, dtype):
    g = torch.Generator(device=DEV).manual_seed(T + W)
    x = torch.randn(T, H, W, generator=g, device=DEV).to(dtype)
    pos = torch.randint(0, 1 << 20, (T,), generator=g, device=DEV)
    rope = Rope(inv_freq(dim), 1.25, layout)
    want, size = expect(x, pos, rope, start)
    keep = x.clone()
    close(rope(x, pos, start), want, size)
    close(rope(x, pos.int(), start), want, size)
    assert torch.equal(x, keep)
    out = torch.empty_like(x)
    assert rope(x, pos, start, out=out) is out
    close(out, want, size)
    rope(x, pos, start, out=x)                   # in place
    assert torch.equal(x, out)


@pytest.mark.parametrize("layout", ["half", "interleaved", "pairs_to_half"])
def test_strides_and_parts_of_wider_tensors(layout):
    g = torch.Generator(device=DEV).manual_seed(3)
    pos = torch.randint(0, 5000, (9,), generator=g, device=DEV)
    rope = Rope(inv_freq(64), 1.0, layout)
    for off in (0, 8, 3):                         # 16-byte rows, and rows of any alignment
        base = torch.randn(9, 4 * 200 + 40, generator=g, device=DEV).bfloat16()
        x = base[:, off:off + 800].view(9, 4, 200)[..., 128:192] if off == 0 else base[:, off:off + 800].unflatten(1, (4, 200))[..., 128:192]
        big = torch.zeros(4, 9, 576, dtype=torch.bfloat16, device=DEV)
        out = big.transpose(0, 1)[..., 512:]
        want, size = expect(x, pos, rope, 0)
        rope(x, pos, out=out)
        close(out, want, size)
        assert not big[..., :512].any()
        before = base.clone()
        rope(x, pos, out=x)
        close(x, want, size)
        x.copy_(out)
        mask = torch.ones_like(base, dtype=torch.bool)
        mask[:, off:off + 800].unflatten(1, (4, 200))[..., 128:192] = False
        assert torch.equal(base[mask], before[mask])
    row = torch.randn(1, 1, 64, generator=g, device=DEV).half().expand(9, 4, 64)      # one row for all
    want, size = expect(row, pos, rope, 0)
    close(rope(row, pos), want, size)
    flat = torch.randn(9, 64, generator=g, device=DEV).bfloat16()                     # no heads
    want, size = expect(flat[:, None], pos, rope, 0)
    close(rope(flat, pos), want[:, 0], size[:, 0])
    out = torch.empty_like(flat)
    assert rope(flat, pos, out=out) is out
    close(out, want[:, 0], size[:, 0])


def test_far_and_negative_positions():
    rope = Rope(inv_freq(64), layout="half")
    x = torch.randn(6, 2, 64, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).half()
    pos = torch.tensor([0, 1, 2 ** 24 + 1, 2 ** 30, 2 ** 30 - 1, 123456789], device=DEV)
    want, size = expect(x, pos, rope, 0)
    close(rope(x, pos), want, size)
    assert torch.equal(rope(x, pos)[0], x[0])
    out = torch.full_like(x, 7)
    skip = pos.clone()
    skip[[1, 4]] = -1
    rope(x, skip, out=out)
    close(out[[0, 2, 3, 5]], want[[0, 2, 3, 5]], size[[0, 2, 3, 5]])
    assert (out[[1, 4]] == 7).all()


def test_no_tokens_and_many():
    rope = Rope(inv_freq(16), layout="interleaved")
    assert rope(torch.empty(0, 4, 16, device=DEV).half(), torch.empty(0, dtype=torch.int32, device=DEV)).shape == (0, 4, 16)
    assert rope(torch.empty(3, 0, 16, device=DEV).half(), torch.zeros(3, dtype=torch.int32, device=DEV)).shape == (3, 0, 16)
    x = torch.randn(70001, 1, 16, device=DEV).half()
    pos = torch.arange(70001, device=DEV, dtype=torch.int32)
    got = rope(x, pos)
    some = torch.tensor([0, 1, 255, 256, 65535, 65536, 70000], device=DEV)
    want, size = expect(x[some], pos[some], rope, 0)
    close(got[some], want, size)
    assert torch.equal(got[some], rope(x[some], pos[some]))


def test_infinities_stay_in_their_pair():
    rope = Rope(inv_freq(64), layout="half")
    x = torch.randn(2, 2, 64, device=DEV).bfloat16()
    pos = torch.tensor([5, 6], device=DEV)
    want = rope(x, pos)
    x[1, 0, 3], x[0, 1, 40] = float("inf"), float("nan")
    got = rope(x, pos)
    hit = torch.zeros_like(x, dtype=torch.bool)
    hit[1, 0, [3, 35]] = hit[0, 1, [8, 40]] = True
    assert torch.equal(got[~hit], want[~hit]) and not got[hit].isfinite().any()


def test_the_models_tables():
    """Rope.yarn is the table of the decode graph, less its rounding to BF16 and of the angle to FP32."""
    rope = Rope.yarn(64, device=DEV)
    cos, sin = rope_tables(64, 4096)
    pos = torch.tensor([0, 1, 17, 1000, 4095], device=DEV)
    x = torch.zeros(5, 32, 64, device=DEV).bfloat16()
    x[:, torch.arange(32), 2 * torch.arange(32)] = 1       # head i: pair i is (1, 0)
    y = rope(x, pos).float().cpu()
    at = torch.arange(32)
    # BF16 twice, and 4096 x 2^-24 of an FP32 angle
    assert ((y[:, at, at] - cos[pos.cpu(), :32].float()).abs() <= 2 * 2.0 ** -8 * 1.0 + 2.0 ** -11).all()
    assert ((y[:, at, at + 32] - sin[pos.cpu(), :32].float()).abs() <= 2 * 2.0 ** -8 * 1.0 + 2.0 ** -11).all()
    assert rope.scale == 1.0 and YARN["factor"] == 40.0


def test_streams_and_a_captured_graph():
    rope = Rope(inv_freq(64), layout="half")
    x = torch.randn(33, 16, 192, device=DEV).bfloat16()
    pos = torch.arange(33, device=DEV)
    want = rope(x, pos, 128)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for s in (side, side.cuda_stream):
        got = rope(x, pos, 128, stream=s)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    graph, static = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        out = rope(static, pos, 128)
    for shift in (0, 9):
        pos.add_(shift)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, rope(x, pos, 128))
