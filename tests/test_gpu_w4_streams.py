"""Calls on a stream of their own: what the allocator may do with their tensors meanwhile, and inputs that change
from call to call in one workspace."""
import pytest
import torch

from fleet.pack_weights import quantize_w4
from fleet.routing import route_experts
from fleet.w4 import W4Experts, W4Linear

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def later(make, call):
    """call(*tensors, stream) on a stream that is busy until after the tensors of make() have been dropped and their
    memory has been used again; its result."""
    side = torch.cuda.Stream()
    tensors = make()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)                # about 10 ms
    result = call(*tensors, side)
    sizes = [(t.shape, t.dtype) for t in tensors]
    del tensors
    again = [torch.zeros(shape, dtype=dtype, device=DEV) for shape, dtype in sizes for _ in range(3)]
    torch.cuda.synchronize()
    del again
    return result


@pytest.mark.parametrize("raw", [False, True])
def test_inputs_dropped_while_the_stream_is_busy(raw):
    handle = lambda s: s.cuda_stream if raw else s  # noqa: E731
    g = lambda: torch.Generator(device=DEV).manual_seed(1)  # noqa: E731
    w = lambda *s: torch.randn(*s, generator=g(), device=DEV).bfloat16()  # noqa: E731
    lin = W4Linear(*quantize_w4(w(256, 512), 64), group=64)
    make = lambda: [w(9, 512), w(9, 256)]  # noqa: E731
    want = lin(*make()[:1], residual=make()[1])
    assert torch.equal(later(make, lambda x, r, s: lin(x, residual=r, stream=handle(s))), want)

    experts = W4Experts(quantize_w4(w(4, 256, 512), 64), quantize_w4(w(4, 512, 128), 64), group=64)

    def make():
        ids = torch.rand(9, 4, generator=g(), device=DEV).argsort(1)[:, :2].int().contiguous()
        return w(9, 512), ids, torch.rand(9, 2, generator=g(), device=DEV), w(9, 512) + 1
    x, ids, weights, res = make()
    want = experts(x, ids, weights, residual=res)
    assert torch.equal(later(make, lambda x, i, v, r, s: experts(x, i, v, residual=r, stream=handle(s))), want)

    make = lambda: [torch.randn(50, 64, generator=g(), device=DEV), torch.rand(64, generator=g(), device=DEV)]  # noqa: E731
    logits, bias = make()
    want = route_experts(logits, 6, bias=bias)
    got = later(make, lambda l, b, s: route_experts(l, 6, bias=b, stream=handle(s)))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_weights_dropped_while_the_stream_is_busy():
    g = torch.Generator(device=DEV).manual_seed(2)
    codes = quantize_w4(torch.randn(256, 512, generator=g, device=DEV).bfloat16(), 64, True)
    x = torch.randn(3, 512, generator=g, device=DEV).bfloat16()
    want = W4Linear(*codes, group=64)(x)
    side, lin = torch.cuda.Stream(), W4Linear(*codes, group=64)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
    got = lin(x, stream=side)
    shapes = [(t.shape, t.dtype) for t in (lin.w.codes, lin.w.scales, lin.w.zeros)]
    del lin
    again = [torch.zeros(s, dtype=d, device=DEV) for s, d in shapes for _ in range(3)]
    torch.cuda.synchronize()
    assert torch.equal(got, want) and again


@pytest.mark.parametrize("T", [1, 3, 8, 9, 30])
def test_inputs_change_from_call_to_call(T):
    """Every launch of a call reads what this call's earlier launches wrote, not the last call's values."""
    g = torch.Generator(device=DEV).manual_seed(T)
    E, H, I = 12, 512, 200
    experts = W4Experts(quantize_w4(torch.randn(E, 2 * I, H, generator=g, device=DEV).bfloat16(), 64),
                        quantize_w4(torch.randn(E, H, I, generator=g, device=DEV).bfloat16(), 64), group=64, inter=I)
    sets = []
    for _ in range(8):
        ids = torch.rand(T, E, generator=g, device=DEV).argsort(1)[:, :4].int().contiguous()
        sets.append((torch.randn(T, H, generator=g, device=DEV).bfloat16(), ids, torch.rand(T, 4, generator=g, device=DEV)))
    want = []
    for s in sets:
        want.append(experts(*s))
        torch.cuda.synchronize()
    for i in range(1, len(want)):
        assert not torch.equal(want[0], want[i])
    got = [experts(*sets[i % 8]) for i in range(400)]
    assert all(torch.equal(v, want[i % 8]) for i, v in enumerate(got))


@pytest.mark.parametrize("T", [4, 20])
def test_calls_on_a_stream_in_a_captured_graph(T):
    """stream= while a graph is captured: the capturing stream itself, and one that it forks to and joins."""
    g = torch.Generator(device=DEV).manual_seed(T)
    w = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()  # noqa: E731
    lin = W4Linear(*quantize_w4(w(256, 512), 64), group=64)
    experts = W4Experts(quantize_w4(w(4, 256, 512), 64), quantize_w4(w(4, 512, 128), 64), group=64)
    static, logits = w(T, 512), torch.randn(T, 4, generator=g, device=DEV)

    def step(x, **kw):
        ids, weights = route_experts(logits, 2, **kw)
        return lin(experts(x, ids, weights, residual=x, **kw), **kw)
    inputs = [w(T, 512) for _ in range(3)]
    want = [step(x) for x in inputs]
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        here = torch.cuda.current_stream()
        a = step(static, stream=here)
        side.wait_stream(here)
        b = step(static, stream=side)
        here.wait_stream(side)
    for x, v in zip(inputs, want):
        static.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, v) and torch.equal(b, v)
