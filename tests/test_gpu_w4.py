"""W4Linear and W4Experts on the GPU against the same formulas in 64 bits.

Two kinds of checks. Exact ones: integer activations and power-of-two scales, so that every product
and sum is a small integer and the FP32 result has to be the exact one whatever the order (one wrong
code, column or group shows). Bounded ones: random values against 64 bits, the bound being the sum of
the roundings the kernels do. u16 is the unit roundoff of the 16-bit type, and every FP32 rounding or
truncation of a partial sum is at most 2^-23 of S, the sum of the terms' magnitudes: a row has at most 16
of them within a group (8 MMAs that round their products and their sum), one per group when the
group is scaled, one when it is added, and 16 + 2 across the warps, the residual and the result."""
import pytest
import torch

from fleet.pack_weights import dequantize_w4, quantize_w4
from fleet.w4 import W4Experts, W4Linear

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U16 = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a step of 8 and 11 significant bits


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def sum_bound(groups):
    return (16 + 2 * groups + 18) * 2.0 ** -23


def codes_of(g, shape, k, group, zeros, dtype, scale=None):
    """Random codes (every value), zero points and power-of-two scales (or random ones)."""
    G = -(-k // group)
    codes = torch.randint(0, 256, (*shape, (k + 1) // 2), generator=g, device=DEV, dtype=torch.uint8)
    if scale == "exact":
        s = 2.0 ** torch.randint(-2, 2, (*shape, G), generator=g, device=DEV).float()
    else:
        s = torch.rand(*shape, G, generator=g, device=DEV) * 0.01 + 0.001
    z = torch.randint(0, 16, (*shape, G), generator=g, device=DEV, dtype=torch.uint8) if zeros else None
    return codes, s.to(dtype), z


SHAPES = [  # T, N, K, group, zeros
    (1, 16, 64, 32, False), (1, 1, 1, 32, True), (1, 2048, 2048, 128, False), (2, 17, 33, 32, True),
    (3, 100, 95, 64, True), (5, 48, 1408, 128, False), (8, 31, 96, 32, False), (9, 250, 160, 128, True),
    (16, 64, 2048, 64, False), (17, 33, 130, 64, True), (31, 40, 1350, 32, True), (32, 80, 512, 128, False),
    (33, 20, 200, 32, False), (70, 24, 129, 128, True), (4, 5000, 192, 64, False), (12, 16, 10944, 64, False),
    (1, 32, 20000, 32, True), (1, 2400, 64, 32, False),
    # rows for two tiles a warp, and with rows too long for staged activations
    (1, 9601, 160, 128, False), (7, 9500, 300, 32, True), (16, 9477, 129, 64, False), (32, 9472, 64, 32, True),
    (8, 9500, 12000, 64, False), (8, 40, 24008, 128, True),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("T,N,K,group,zeros", SHAPES)
def test_linear_exact(T, N, K, group, zeros, dtype):
    g = gen(T * 7919 + N)
    w = codes_of(g, (N,), K, group, zeros, dtype, "exact")
    x = torch.randint(-3, 4, (T, K), generator=g, device=DEV).to(dtype)
    res = torch.randint(-8, 9, (T, N), generator=g, device=DEV).to(dtype)
    want = x.double() @ dequantize_w4(*w, K, group).double().T + res.double()
    assert want.abs().max() * 4 < 2 ** 24                       # quarters, exact in FP32
    lin = W4Linear(*w, k=K, group=group)
    assert torch.equal(lin(x, residual=res, out_dtype=torch.float32).double(), want)
    assert torch.equal(lin(x, residual=res), want.to(dtype))    # rounded once
    assert torch.equal(lin(x), (want - res.double()).to(dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("T,N,K,group,zeros", SHAPES)
def test_linear_bounded(T, N, K, group, zeros, dtype):
    g = gen(T * 104729 + K)
    w = codes_of(g, (N,), K, group, zeros, dtype)
    x = torch.randn(T, K, generator=g, device=DEV).to(dtype)
    W = dequantize_w4(*w, K, group).double()
    want = x.double() @ W.T
    bound = (x.double().abs() @ W.abs().T) * sum_bound(-(-K // group))
    lin = W4Linear(*w, k=K, group=group)
    got = lin(x, out_dtype=torch.float32)
    assert ((got.double() - want).abs() <= bound).all()
    assert torch.equal(lin(x), got.to(dtype))                   # the 16-bit result is the FP32 one rounded
    assert torch.equal(lin(x, out_dtype=torch.float32), got)    # and the same on every run


def test_linear_strides_and_alignment():
    g = gen(5)
    T, N, K = 6, 70, 200
    w = codes_of(g, (N,), K, 64, True, torch.bfloat16, "exact")
    W = dequantize_w4(*w, K, 64).double()
    lin = W4Linear(*w, k=K, group=64)
    big = torch.randint(-3, 4, (T + 1, K + 13), generator=g, device=DEV).to(torch.bfloat16)
    out = torch.full((T, N + 9), 7.0, device=DEV, dtype=torch.bfloat16)
    for x in (big[:T, :K], big[1:, 3:K + 3], big[:T, 8:K + 8], big[1:2, 5:K + 5].expand(T, K)):   # odd starts, odd rows, one row
        view = out[:, 3:N + 3]
        assert lin(x, out=view) is view
        assert torch.equal(view.double(), (x.double() @ W.T).to(torch.bfloat16).double())
        assert (out[:, :3] == 7).all() and (out[:, N + 3:] == 7).all()
    res = out[:, 3:N + 3]
    want = (big[:T, :K].double() @ W.T + res.double()).to(torch.bfloat16)
    lin(big[:T, :K], out=res, residual=res)                      # in place
    assert torch.equal(res, want)


def test_linear_long_rows_without_alignment():
    """Rows too long to be staged for all tokens and not 16-byte aligned: fewer tokens at a time."""
    g = gen(8)
    w = codes_of(g, (24,), 10949, 64, True, torch.bfloat16, "exact")
    big = torch.randint(-3, 4, (13, 10952), generator=g, device=DEV).to(torch.bfloat16)
    x = big[:, 1:10950]
    want = x.double() @ dequantize_w4(*w, 10949, 64).double().T
    assert torch.equal(W4Linear(*w, k=10949, group=64)(x, out_dtype=torch.float32).double(), want)


def test_linear_weight_past_4_gib():
    """Codes of 4.6 GiB: the last rows, whose bytes lie past 32 bits."""
    g, N, K = gen(3), 300032, 32768
    w = codes_of(g, (N,), K, 128, False, torch.bfloat16, "exact")
    x = torch.randint(-3, 4, (2, K), generator=g, device=DEV).to(torch.bfloat16)
    got = W4Linear(*w, k=K, group=128)(x, out_dtype=torch.float32)
    assert w[0].numel() > 2 ** 32
    for rows in (slice(0, 40), slice(N - 100, N)):
        want = x.double() @ dequantize_w4(w[0][rows], w[1][rows], None, K, 128).double().T
        assert torch.equal(got[:, rows].double(), want)


def test_linear_many_tokens():
    g = gen(4)
    w = codes_of(g, (50,), 100, 32, True, torch.float16, "exact")
    x = torch.randint(-3, 4, (3001, 100), generator=g, device=DEV).half()
    assert torch.equal(W4Linear(*w, k=100, group=32)(x, out_dtype=torch.float32).double(),
                       x.double() @ dequantize_w4(*w, 100, 32).double().T)


def test_linear_no_tokens_and_refusals():
    w = quantize_w4(torch.randn(32, 64, generator=gen(0), device=DEV).to(torch.bfloat16), 32)
    lin = W4Linear(*w, k=64, group=32)
    x = torch.zeros(2, 64, device=DEV, dtype=torch.bfloat16)
    assert lin(x[:0]).shape == (0, 32)
    for bad in (lambda: lin(x.half()), lambda: lin(x[:, :63]), lambda: lin(x.t()), lambda: lin(x[0]), lambda: lin(x.cpu()),
                lambda: lin(x, out_dtype=torch.float16), lambda: lin(x, residual=x[:, :32].float()),
                lambda: lin(x, out=torch.empty(2, 31, device=DEV, dtype=torch.bfloat16)), lambda: lin(x, out=x[:, :32])):
        with pytest.raises(ValueError):
            bad()


def test_linear_infinities_stay_in_their_token():
    g = gen(9)
    w = quantize_w4(torch.randn(48, 256, generator=g, device=DEV).to(torch.bfloat16), 64)
    lin = W4Linear(*w, k=256, group=64)
    x = torch.randn(5, 256, generator=g, device=DEV).to(torch.bfloat16)
    clean = lin(x)
    x[1, 17] = float("nan")
    x[3, 200] = float("inf")
    got = lin(x)
    assert torch.equal(got[[0, 2, 4]], clean[[0, 2, 4]])
    assert got[1].isnan().all()
    code = dequantize_w4(*w, 256, 64)[:, 200]
    want = torch.where(code == 0, float("nan"), torch.where(code > 0, float("inf"), -float("inf")))
    assert torch.equal(got[3].float().nan_to_num(nan=1.0), want.nan_to_num(nan=1.0))


def experts_reference(x, ids, weights, w13, w2, H, I, group, res, dtype):
    """(want, bound) in 64 bits: the activations' rounding (u16 of each) and FP32 sums through the products."""
    W13, W2 = dequantize_w4(*w13, H, group).double(), dequantize_w4(*w2, I, group).double()
    e13, e2 = sum_bound(-(-H // group)), sum_bound(-(-I // group))
    T, S = ids.shape
    want = torch.zeros(T, H, dtype=torch.float64, device=DEV) if res is None else res.double().clone()
    err, mag = torch.zeros_like(want), want.abs()
    for e in ids.unique().tolist():
        if not 0 <= e < W13.shape[0]:
            continue
        t, s = (ids == e).nonzero(as_tuple=True)
        xe = x[t].double()
        gu, m = xe @ W13[e].T, (xe.abs() @ W13[e].abs().T) * e13
        gt, up = gu[:, 0::2], gu[:, 1::2]
        silu = gt * torch.sigmoid(gt)
        a = silu * up
        # |silu'| <= 1.1; expf, the addition, the division and the product round by at most 6 units of 2^-24
        ea = 1.1 * m[:, 0::2] * (up.abs() + m[:, 1::2]) + silu.abs() * m[:, 1::2] + a.abs() * (U16[dtype] + 6 * 2.0 ** -24)
        # an FP16 activation under the normal range is off by half a step of 2^-24
        ea = ea + (2.0 ** -25 if dtype == torch.float16 else 0.0)
        y = a @ W2[e].T
        ey = ea @ W2[e].abs().T + ((a.abs() + ea) @ W2[e].abs().T) * e2
        f = weights[t, s].double()[:, None]
        want.index_add_(0, t, f * y)
        err.index_add_(0, t, f.abs() * ey)
        mag.index_add_(0, t, f.abs() * (y.abs() + ey))
    return want, err + mag * (S + 2) * 2.0 ** -23 + (want.abs() + err) * U16[dtype]


EXPERTS = [  # T, H, I, E, S, group, zeros, residual
    (1, 64, 64, 4, 2, 32, False, True), (1, 2048, 1408, 10, 8, 128, False, True), (2, 72, 40, 3, 3, 32, True, False),
    (7, 130, 50, 9, 4, 64, True, True), (8, 256, 96, 66, 8, 64, True, True), (16, 200, 174, 20, 5, 32, True, False),
    (17, 96, 33, 5, 1, 128, False, True), (40, 500, 174, 6, 3, 32, True, False), (33, 128, 72, 2, 2, 64, False, True),
    (64, 64, 200, 80, 8, 32, False, True), (150, 48, 16, 7, 4, 32, True, True),
    (5, 9500, 40, 3, 2, 64, False, True), (12, 9500, 33, 2, 2, 32, True, False), (20, 4800, 24, 6, 2, 128, False, True),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("T,H,I,E,S,group,zeros,residual", EXPERTS)
def test_experts(T, H, I, E, S, group, zeros, residual, dtype):
    g = gen(T * 31 + H)
    w13 = codes_of(g, (E, 2 * I), H, group, zeros, dtype)
    w2 = codes_of(g, (E, H), I, group, zeros, dtype)
    x = torch.randn(T, H, generator=g, device=DEV).to(dtype)
    ids = torch.rand(T, E, generator=g, device=DEV).argsort(1)[:, :S].to(torch.int32).contiguous()
    weights = torch.rand(T, S, generator=g, device=DEV)
    res = torch.randn(T, H, generator=g, device=DEV).to(dtype) if residual else None
    op = W4Experts(w13, w2, group=group, inter=I)
    got = op(x, ids, weights, residual=res)
    want, bound = experts_reference(x, ids, weights, w13, w2, H, I, group, res, dtype)
    assert ((got.double() - want).abs() <= bound).all()
    for _ in range(3):
        assert torch.equal(op(x, ids, weights, residual=res), got)      # the same on every run
    if residual:
        out = res.clone()
        assert op(x, ids, weights, residual=out, out=out) is out and torch.equal(out, got)


def small_experts(T=6, H=64, I=48, E=5, S=3, dtype=torch.bfloat16, seed=2):
    g = gen(seed)
    w13, w2 = codes_of(g, (E, 2 * I), H, 32, True, dtype), codes_of(g, (E, H), I, 32, True, dtype)
    x = torch.randn(T, H, generator=g, device=DEV).to(dtype)
    ids = torch.rand(T, E, generator=g, device=DEV).argsort(1)[:, :S].to(torch.int32).contiguous()
    return g, w13, w2, x, ids, torch.rand(T, S, generator=g, device=DEV), W4Experts(w13, w2, group=32, inter=I)


@pytest.mark.parametrize("T", [3, 6, 40])
def test_experts_empty_and_repeated_slots(T):
    g, w13, w2, x, ids, weights, op = small_experts(T)
    ids[0] = -1                          # a padding token
    ids[1] = torch.tensor([4, 4, 4])     # one expert three times
    ids[2] = torch.tensor([5, 1, 2 ** 31 - 1])   # ids past the experts
    weights[0, 0] = float("nan")         # the weight of an empty slot is not read
    want, bound = experts_reference(x, ids, torch.nan_to_num(weights), w13, w2, 64, 48, 32, None, torch.bfloat16)
    got = op(x, ids, weights)
    assert (got[0] == 0).all()
    assert ((got.double() - want).abs() <= bound).all()
    ids.fill_(-1)
    assert (op(x, ids, weights) == 0).all() and torch.equal(op(x, ids, weights, residual=x), x)


@pytest.mark.parametrize("T", [4, 40])
def test_experts_all_tokens_on_one_expert(T):
    g, w13, w2, x, ids, weights, op = small_experts(T, S=1)
    ids.fill_(3)
    want, bound = experts_reference(x, ids, weights, w13, w2, 64, 48, 32, None, torch.bfloat16)
    assert ((op(x, ids, weights).double() - want).abs() <= bound).all()


def test_experts_nan_stays_in_its_token():
    g, w13, w2, x, ids, weights, op = small_experts()
    clean = op(x, ids, weights)
    x[2, 5] = float("nan")
    got = op(x, ids, weights)
    others = [0, 1, 3, 4, 5]
    assert torch.equal(got[others], clean[others]) and got[2].isnan().all()


def test_experts_no_tokens_no_slots_and_refusals():
    g, w13, w2, x, ids, weights, op = small_experts()
    assert op(x[:0], ids[:0], weights[:0]).shape == (0, 64)
    assert torch.equal(op(x, ids[:, :0].contiguous(), weights[:, :0].contiguous(), residual=x), x)
    for bad in (lambda: op(x, ids.long(), weights), lambda: op(x, ids[:5], weights[:5]), lambda: op(x, ids, weights[:, :2]),
                lambda: op(x, ids.t().contiguous().t(), weights), lambda: op(x, ids, weights.half()), lambda: op(x.half(), ids, weights),
                lambda: op(x, ids.cpu(), weights), lambda: op(x, ids, weights, out=x),
                lambda: op(x, ids, weights, residual=x[:5])):
        with pytest.raises(ValueError):
            bad()


def test_streams_and_graphs():
    """Calls on other streams and in a captured graph give the default stream's results."""
    from fleet.routing import route_experts
    g, w13, w2, x, ids, weights, op = small_experts(T=20)
    lin = W4Linear(*codes_of(g, (96,), 64, 32, False, torch.bfloat16), k=64, group=32)
    logits = torch.randn(20, 5, generator=g, device=DEV)

    def layer(x, **kw):
        i, w = route_experts(logits, 3, **kw)
        return lin(op(x, i, w, residual=x, **kw), **kw)
    want = layer(x)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(20):
        outs.append(layer(x, stream=a))
        outs.append(layer(x, stream=b.cuda_stream))
        with torch.cuda.stream(b):
            outs.append(layer(x))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    static, graph = x.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(static)
    static.copy_(x.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    # the routing is by row, so the flipped tokens meet other experts: compare with a plain call
    assert torch.equal(out, layer(x.flip(0)))
