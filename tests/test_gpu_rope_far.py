"""Rope at far positions against turns in exact rationals, and heads so wide that a loop of its own copies them.

A turn is off by at most its size x (2^-54 of 1 / 2 pi, and 2^-53 for each of two products), 2.5 x 2^-53 x 2^29 < 2^-22.6 at
positions up to 2^31 and frequencies up to 1, and by 2^-26 from its rest's rounding to FP32: an angle by less than 2 pi x 2^-22.4
< 2^-19.7. sincospif is within 2 units of 2^-24, the scale, the two products and their sum add 3 x 2^-24: together within 2^-19.5
(|a| + |b|) scale, and the output's own rounding is half a step."""
import math
from fractions import Fraction

import pytest
import torch

from fleet.rope import Rope

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# 2 pi to 100 bits: pi = 16 atan(1/5) - 4 atan(1/239) as sums of fractions
atan = lambda n: sum(Fraction((-1) ** k, (2 * k + 1) * n ** (2 * k + 1)) for k in range(40))  # noqa: E731
TURN = 2 * (16 * atan(5) - 4 * atan(239))


def angle(position, inv_freq):
    turns = Fraction(position) * Fraction(inv_freq) / TURN
    return float((turns - round(turns)) * TURN)


def expect(x, positions, rope, start):
    """(values, the size of each turned one) of halves or neighbours in 64 bits, angles from exact turns."""
    n = rope.dim
    t = torch.tensor([[angle(p, f) for f in rope.inv_freq.tolist()] for p in positions.tolist()], dtype=torch.float64)[:, None]
    c, s = rope.scale * t.cos(), rope.scale * t.sin()
    y, size = x.double().cpu(), torch.zeros(x.shape, dtype=torch.float64)
    part = y[..., start:start + n]
    a, b = (part[..., :n // 2], part[..., n // 2:]) if rope.layout == "half" else (part[..., ::2], part[..., 1::2])
    w = abs(rope.scale) * (a.abs() + b.abs())
    lo, hi = a * c - b * s, b * c + a * s
    both = (lambda u, v: torch.stack([u, v], -1).flatten(-2)) if rope.layout == "interleaved" else (lambda u, v: torch.cat([u, v], -1))
    y[..., start:start + n], size[..., start:start + n] = both(lo, hi), both(w, w)
    return y, size


def close(got, want, size):
    eps = torch.finfo(got.dtype).eps
    off = (got.double().cpu() - want).abs()
    bound = eps / 2 * want.abs() + (1 + eps) * 2.0 ** -19.5 * size
    assert (off <= bound).all(), (off - bound).max()
    assert torch.equal(got.double().cpu()[size == 0], want[size == 0])


def test_the_reference_itself():
    assert abs(float(TURN) - 2 * math.pi) <= 2 ** -51 and abs(angle(7, 1.0) - math.remainder(7.0, 2 * math.pi)) < 1e-14


@pytest.mark.parametrize("layout", ["half", "interleaved", "pairs_to_half"])
def test_positions_up_to_32_bits(layout):
    inv = torch.tensor([1.0, 0.7, 0.1, 1e-3, 1 / 3, 0.999, 1e-5, 0.5], dtype=torch.float64, device=DEV)
    rope = Rope(inv, 1.25, layout)
    pos = torch.tensor([2 ** 31 - 1, 2 ** 31 - 2, 2 ** 30 + 1, 2 ** 28 + 12345, 2 ** 24 + 1, 0, 1, 1987654321], device=DEV)
    x = torch.randn(8, 3, 16, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).half()
    want = expect(x, pos, rope, 0)
    close(rope(x, pos), *want)
    close(rope(x, pos.int()), *want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["half", "interleaved", "pairs_to_half"])
@pytest.mark.parametrize("T,H,W,dim,start", [(3, 2, 1300, 30, 700), (2, 3, 1055, 2, 0), (3, 2, 4400, 64, 2048), (400, 1, 4176, 16, 4160), (2, 5, 9000, 512, 8)])
def test_heads_wider_than_a_blocks_registers(T, H, W, dim, start, layout, dtype):
    """More values beside the turned ones than a block's threads hold at once: 1024 one by one, 4096 eight at a time."""
    g = torch.Generator(device=DEV).manual_seed(W)
    x = torch.randn(T, H, W, generator=g, device=DEV).to(dtype)
    pos = torch.randint(0, 1 << 16, (T,), generator=g, device=DEV)
    rope = Rope(torch.tensor([10000.0 ** -(2 * i / dim) for i in range(dim // 2)], dtype=torch.float64, device=DEV), 1.0, layout)
    want, size = expect(x, pos, rope, start)
    close(rope(x, pos, start), want, size)
    pos[1] = -1
    out = torch.full((T, H + 1, W), 7.0, device=DEV).to(dtype)
    rope(x, pos, start, out=out[:, :H])
    live = torch.arange(T) != 1
    close(out[:, :H][live.to(DEV)], want[live], size[live])
    assert (out[1] == 7).all() and (out[:, H] == 7).all()
    keep = x.clone()
    rope(x, pos, start, out=x)                   # in place: only the part moves
    close(x[live.to(DEV)], want[live], size[live])
    assert torch.equal(x[1], keep[1])
