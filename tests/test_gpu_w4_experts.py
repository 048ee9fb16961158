"""W4Experts where its intermediate, the order of its sums and its forms can go wrong, against 64 bits.

The bounds are those of a computation in FP32 that rounds once, at the end. The intermediate a = silu(g) u goes
to the down projection as two BF16 values: the second holds the first one's remainder to 8 significant
bits, so a is off by at most 2^-16 of itself. An MMA rounds or truncates its sum by at most 2^-23 of the terms'
magnitudes; a group has at most 8 of them for the gate and up rows and 16 for the down projection (8 for
each value), each with two such roundings, then one for the scale and one for the sum per group and 18
across the warps, the residual and the result, as for the linear."""
import pytest
import torch

from fleet.pack_weights import dequantize_w4
from fleet.w4 import W4Experts, W4Linear

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U16 = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a step of 8 and 11 significant bits
SUBNORMAL = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}   # half a step below the normal range
U = 2.0 ** -24


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def weight_of(g, shape, k, group, zeros, dtype, scale=0.01):
    n = -(-k // group)
    codes = torch.randint(0, 256, (*shape, (k + 1) // 2), generator=g, device=DEV, dtype=torch.uint8)
    scales = (torch.rand(*shape, n, generator=g, device=DEV) * scale + scale / 10).to(dtype)
    return codes, scales, torch.randint(0, 16, (*shape, n), generator=g, device=DEV, dtype=torch.uint8) if zeros else None


def reference(x, ids, weights, w13, w2, H, I, group, res, dtype):
    """(want, bound) in 64 bits; empty slots are ids outside the experts."""
    E = w13[0].shape[0]
    sums = lambda mmas, k: (2 * mmas + 2 * -(-k // group) + 18) * 2 * U  # noqa: E731
    want = torch.zeros(x.shape[0], H, dtype=torch.float64, device=DEV) if res is None else res.double().clone()
    err, mag = torch.zeros_like(want), want.abs()
    part = lambda w, e: [None if v is None else v[e] for v in w]  # noqa: E731
    for e in ids.unique().tolist():
        if not 0 <= e < E:
            continue
        W13, W2 = dequantize_w4(*part(w13, e), H, group).double(), dequantize_w4(*part(w2, e), I, group).double()
        t, s = (ids == e).nonzero(as_tuple=True)
        xe = x[t].double()
        gu, m = xe @ W13.T, (xe.abs() @ W13.abs().T) * sums(8, H)
        gt, up = gu[:, 0::2], gu[:, 1::2]
        silu = gt * torch.sigmoid(gt)
        a = silu * up
        # |silu'| <= 1.1; expf, the addition, the division and the product round by at most 6 units
        ea = 1.1 * m[:, 0::2] * (up.abs() + m[:, 1::2]) + silu.abs() * m[:, 1::2] + a.abs() * (2.0 ** -16 + 6 * U)
        ey = ea @ W2.abs().T + ((a.abs() + ea) @ W2.abs().T) * sums(16, I)
        f, y = weights[t, s].double()[:, None], a @ W2.T
        want.index_add_(0, t, f * y)
        err.index_add_(0, t, f.abs() * ey)
        mag.index_add_(0, t, f.abs() * (y.abs() + ey))
    err = err + mag * (ids.shape[1] + 2) * 2 * U
    return want, err + (want.abs() + err) * U16[dtype] + SUBNORMAL[dtype]


def routed(g, T, E, S):
    ids = torch.rand(T, E, generator=g, device=DEV).argsort(1)[:, :S].to(torch.int32).contiguous()
    return ids, torch.rand(T, S, generator=g, device=DEV)


def check(T, H, I, E, S, group, zeros, residual, dtype, scale=0.01, x_scale=1.0, w2_scale=None):
    g = gen(T * 37 + H)
    w13 = weight_of(g, (E, 2 * I), H, group, zeros, dtype, scale)
    w2 = weight_of(g, (E, H), I, group, zeros, dtype, w2_scale or scale)
    x = (torch.randn(T, H, generator=g, device=DEV) * x_scale).to(dtype)
    ids, weights = routed(g, T, E, S)
    res = torch.randn(T, H, generator=g, device=DEV).to(dtype) if residual else None
    op = W4Experts(w13, w2, group=group, inter=I)
    got = op(x, ids, weights, residual=res)
    want, bound = reference(x, ids, weights, w13, w2, H, I, group, res, dtype)
    assert ((got.double() - want).abs() <= bound).all()
    return op, x, ids, weights, res, got, want


DTYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])


@DTYPES
@pytest.mark.parametrize("T,H,I,E,S,group,zeros,residual", [
    (1, 256, 512, 4, 4, 128, False, False), (6, 512, 640, 8, 3, 32, True, True), (8, 192, 330, 16, 8, 64, True, False),
    (24, 256, 512, 6, 3, 64, False, False), (50, 384, 523, 4, 2, 32, True, True), (30, 9500, 48, 3, 2, 64, False, True),
])
def test_one_rounding(T, H, I, E, S, group, zeros, residual, dtype):
    """No rounding to 16 bits but the result's: the bound has none, and where the result does not cancel the
    errors are those of one rounding."""
    got, want = check(T, H, I, E, S, group, zeros, residual, dtype)[-2:]
    once = (want.to(dtype).double() - want).norm()
    assert (got.double() - want).norm() <= 1.05 * once


@pytest.mark.parametrize("T", [1, 5, 20])
def test_fp16_intermediate_past_its_types_range(T):
    """silu(g) u past 65504 with results inside FP16's range."""
    op, x, ids, weights, res, got, want = check(T, 64, 96, 4, 2, 32, True, True, torch.float16, scale=0.5, x_scale=40.0,
                                                w2_scale=2e-6)
    g = gen(T * 37 + 64)
    w13 = weight_of(g, (4, 192), 64, 32, True, torch.float16, 0.5)
    gu = torch.einsum("tk,enk->ten", x.float(), dequantize_w4(*w13, 64, 32))
    assert (torch.nn.functional.silu(gu[..., 0::2]) * gu[..., 1::2]).abs().max() > 4 * 65504
    assert want.abs().max() < 65504 and got.isfinite().all()


@DTYPES
@pytest.mark.parametrize("T", [1, 9])
def test_rows_of_the_down_projection_too_long_to_stage(T, dtype):
    check(T, 64, 50011, 2, 1, 64, False, True, dtype)


@DTYPES
@pytest.mark.parametrize("T,S,E,H,I", [(64, 8, 66, 512, 200), (256, 2, 4, 512, 512), (1000, 4, 8, 1024, 256), (300, 1, 1, 256, 300)])
def test_experts_of_several_items_are_the_same_on_every_run(T, S, E, H, I, dtype):
    """More slots an expert than an item has columns: which of them share an item must not depend on timing."""
    op, x, ids, weights, res, got, want = check(T, H, I, E, S, 64, True, False, dtype)
    for _ in range(30):
        assert torch.equal(op(x, ids, weights), got)


@pytest.mark.parametrize("T,S,E", [(9, 1, 1024), (2000, 16, 1024), (3000, 32, 700), (5000, 2, 321), (40, 8, 320), (20000, 3, 5)])
def test_every_slot_has_its_place(T, S, E):
    """Empty slots between the others, an expert's slots spread over all warps of the plan, repeated slots, more
    experts than all of its warps can count."""
    g = gen(T + E)
    H, I = 32, 16
    w13 = torch.randint(0, 256, (E, 2 * I, H // 2), generator=g, device=DEV, dtype=torch.uint8)
    w2 = torch.randint(0, 256, (E, H, I // 2), generator=g, device=DEV, dtype=torch.uint8)
    one = torch.ones(E, 2 * I, 1, device=DEV, dtype=torch.bfloat16)
    op = W4Experts((w13, one / 64, None), (w2, one[:, :H], None), group=32, inter=I)
    x = torch.randn(T, H, generator=g, device=DEV).bfloat16()
    ids = torch.randint(0, E, (T, S), generator=g, device=DEV, dtype=torch.int32)
    ids[torch.rand(T, S, generator=g, device=DEV) < 0.2] = -1
    weights = torch.randint(-2, 3, (T, S), generator=g, device=DEV).float()
    got = op(x, ids, weights)
    want, bound = reference(x, ids, weights, (w13, one / 64, None), (w2, one[:, :H], None), H, I, 32, None, torch.bfloat16)
    assert ((got.double() - want).abs() <= bound).all()
    assert torch.equal(op(x, ids, weights), got)


def test_more_tokens_than_a_grid_has_rows():
    check(70000, 16, 8, 3, 1, 32, False, True, torch.bfloat16)


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("T", [5, 8, 20])
def test_scales_that_are_not_finite_stay_with_their_expert(T, bad):
    """Tokens that do not select the expert have the results they have without its scales."""
    g = gen(T)
    H, I, E = 96, 200, 6
    for k in (0, 1):
        ws = [weight_of(g, (E, 2 * I), H, 32, True, torch.bfloat16), weight_of(g, (E, H), I, 32, True, torch.bfloat16)]
        x = torch.randn(T, H, generator=g, device=DEV).bfloat16()
        ids, weights = routed(g, T, E, 2)
        ids[0] = torch.tensor([1, 4])
        weights[0, 1] = 0.0                      # expert 4 with weight 0: 0 x an infinity is NaN
        clean = W4Experts(*ws, group=32, inter=I)(x, ids, weights)
        ws[k][1][4] = bad
        got = W4Experts(*ws, group=32, inter=I)(x, ids, weights)
        selects = (ids == 4).any(1)
        assert 0 < selects.sum() < T and torch.equal(got[~selects], clean[~selects])
        assert got[0].isnan().any()


def test_linear_of_more_tokens_than_a_launch_counts():
    """Two launches of one call: the rows on either side of where they part, and the last ones (small integers, exact)."""
    g, T, N, K, group = gen(6), 16 * 10715 + 300, 16000, 12800, 64
    codes = torch.randint(0, 256, (N, K // 2), generator=g, device=DEV, dtype=torch.uint8)
    scales = (2.0 ** torch.randint(-1, 1, (N, K // group), generator=g, device=DEV).float()).bfloat16()
    x = torch.randint(-1, 2, (8 * T + K,), generator=g, device=DEV).bfloat16().as_strided((T, K), (8, 1))   # a row every 8 values
    got = W4Linear(codes, scales, group=group)(x)
    W = dequantize_w4(codes, scales, None, K, group)
    for rows in (slice(0, 20), slice(16 * 10715 - 20, 16 * 10715 + 20), slice(T - 20, T)):
        want = x[rows].double() @ W.double().T
        assert want.abs().max() * 2 < 2 ** 24 and torch.equal(got[rows], want.bfloat16())


@DTYPES
@pytest.mark.parametrize("T,H,I,E,S,group,zeros,residual", [
    # odd values and rows: the last store of an intermediate, its padding, results in single stores
    (1, 131, 51, 4, 2, 32, True, True), (3, 131, 51, 5, 3, 64, False, False), (8, 33, 1, 3, 2, 128, True, True),
    (7, 1, 77, 4, 4, 32, False, True), (2, 255, 129, 6, 2, 128, True, False), (20, 131, 51, 5, 3, 32, True, True),
    (33, 65, 127, 3, 1, 64, False, False),
    # plans near their limits: 256 slots of a small batch, more slots than lanes, many experts
    (8, 64, 24, 40, 32, 32, False, True), (5, 48, 40, 60, 50, 64, True, False), (1, 32, 16, 300, 256, 32, False, True),
    (8, 32, 16, 1024, 32, 32, True, False), (9, 32, 16, 1024, 40, 32, False, True),
])
def test_odd_sizes_and_plans_near_their_limits(T, H, I, E, S, group, zeros, residual, dtype):
    op, x, ids, weights, res, got, want = check(T, H, I, E, S, group, zeros, residual, dtype)
    assert torch.equal(op(x, ids, weights, residual=res), got)


@pytest.mark.parametrize("T", [1, 5, 20])
@pytest.mark.parametrize("H", [96, 97])
def test_strides_and_alignment(T, H):
    """x, residual and out at odd places of wider rows; nothing outside the results is written."""
    g = gen(T + H)
    I, E, dtype = 40, 6, torch.bfloat16
    w13, w2 = weight_of(g, (E, 2 * I), H, 32, True, dtype), weight_of(g, (E, H), I, 32, True, dtype)
    op, (ids, weights) = W4Experts(w13, w2, group=32, inter=I), routed(g, T, E, 2)
    wide = torch.randn(T + 1, H + 13, generator=g, device=DEV).to(dtype)
    wide_res = torch.randn(T, H + 7, generator=g, device=DEV).to(dtype)
    for x0, r0, o0, extra in ((0, 0, 0, 8), (3, 1, 5, 9), (8, 2, 4, 10), (1, 7, 3, 6)):
        x, res = wide[1:, x0:x0 + H], wide_res[:, r0:r0 + H]
        out = torch.full((T, H + extra), 7.0, device=DEV, dtype=dtype)
        view = out[:, o0:o0 + H]
        assert op(x, ids, weights, residual=res, out=view) is view
        want, bound = reference(x, ids, weights, w13, w2, H, I, 32, res, dtype)
        assert ((view.double() - want).abs() <= bound).all()
        assert (out[:, :o0] == 7).all() and (out[:, o0 + H:] == 7).all()
        first = op(x, ids, weights, residual=res)
        assert torch.equal(first, view)
        assert op(x, ids, weights, residual=res, out=res) is res and torch.equal(res, first)     # in place
    one = wide[:1, 2:H + 2].expand(T, H)                                                         # one row for every token
    want, bound = reference(one, ids, weights, w13, w2, H, I, 32, None, dtype)
    assert ((op(one, ids, weights).double() - want).abs() <= bound).all()
