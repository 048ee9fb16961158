"""4-bit weights and routing without a GPU: the quantiser, the laid-out order, the struct layouts and
every refusal (the library checks its arguments before it touches the device)."""
import ctypes

import numpy as np
import pytest
import torch

from fleet import mk, w4
from fleet.pack_weights import dequantize_w4, quantize_w4

needs_lib = pytest.mark.skipif(not mk.LIB_PATH.exists(), reason="library not built")


@pytest.mark.parametrize("shape,group,zero_point", [((5, 64), 32, False), ((2, 3, 100), 64, True), ((7, 129), 128, True),
                                                    ((4, 31), 32, False), ((1, 1), 32, True)])
def test_quantize_is_within_half_a_step(shape, group, zero_point):
    w = torch.randn(*shape, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    codes, scales, zeros = quantize_w4(w, group, zero_point)
    K, g = shape[-1], -(-shape[-1] // group)
    assert codes.shape == (*shape[:-1], (K + 1) // 2) and scales.shape == (*shape[:-1], g)
    back = dequantize_w4(codes, scales, zeros, K, group)
    step = scales.float().repeat_interleave(group, -1)[..., :K]
    # half a step from rounding; the scale's own BF16 rounding moves the range's ends by 8 / 2^9 steps
    # (a step more with a zero point, which is rounded too)
    assert ((back - w.float()).abs() <= step * (0.5 + 16 / 512 + (0.5 if zero_point else 0.0))).all()


def test_quantize_zero_group_decodes_to_zero():
    w = torch.zeros(2, 64, dtype=torch.bfloat16)
    for zero_point in (False, True):
        codes, scales, zeros = quantize_w4(w, 32, zero_point)
        assert (scales == 0).all() and (dequantize_w4(codes, scales, zeros, 64, 32) == 0).all()


def test_quantize_past_the_scale_range_saturates():
    w = torch.tensor([[3e6, -1e6] + [0.0] * 30])
    codes, scales, zeros = quantize_w4(w, 32, dtype=torch.float16)
    back = dequantize_w4(codes, scales, zeros, 32, 32)
    assert scales.item() == 65504 and back.isfinite().all() and back[0, 0] == 7 * 65504


def decode_layout(q, s, z, N, k, group, gate_up):
    """W [E, N, k] from the laid-out tensors, word by word as csrc/mk_w4.cuh states the order."""
    q, s = q.numpy(), s.float().numpy()
    z = np.full_like(s, 8) if z is None else z.numpy().astype(np.float32)
    E, strips, units, _ = q.shape
    words = q.reshape(E, strips, units, 2, 2, 32, 16).view(np.uint32)        # [.., tile, chunk, lane, word]
    w = np.zeros((E, strips * 32, units * 128), np.float32)
    for tile, chunk, lane, h, j, i, half in np.ndindex(2, 2, 32, 2, 2, 4, 2):
        g, t = lane >> 2, lane & 3
        code = (words[:, :, :, tile, chunk, lane, 2 * h + j] >> (4 * i + 16 * half)) & 15
        kk = 64 * chunk + 32 * h + 8 * t + 4 * j + 2 * (i >> 1) + half
        sc, ze = (v[:, :, :, tile, g, kk // group, i & 1] for v in (s, z))
        row = 16 * tile + (2 * g + (i & 1) if gate_up else g + 8 * (i & 1))
        w[:, row::32, kk::128] = sc * (code.astype(np.float32) - ze)
    return w[:, :N, :k], w


@pytest.mark.parametrize("E,N,K,group,zp,gate_up", [(1, 16, 64, 64, False, False), (2, 40, 200, 32, True, False),
                                                    (1, 5, 33, 128, True, False), (3, 22, 70, 64, True, True),
                                                    (1, 48, 96, 32, False, True), (2, 17, 1, 32, True, False)])
def test_laid_out_order(E, N, K, group, zp, gate_up):
    gen = torch.Generator().manual_seed(N)
    codes, scales, zeros = quantize_w4(torch.randn(E, N, K, generator=gen).to(torch.bfloat16), group, zp)
    q, s, z = w4.lay_out(codes, scales, zeros, K, group, gate_up)
    got, padded = decode_layout(q, s, z, N, K, group, gate_up)
    assert np.array_equal(got, dequantize_w4(codes, scales, zeros, K, group).numpy())
    assert (padded[:, N:] == 0).all()                 # rows past the end weigh nothing
    assert (z is None) == (not zp)


def test_odd_k_ignores_the_spare_nibble():
    codes, scales, zeros = quantize_w4(torch.randn(4, 7, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16), 32)
    spare = codes.clone()
    spare[:, -1] |= 0xF0
    a = w4.lay_out(codes[None], scales[None], None, 7, 32)[0]
    b = w4.lay_out(spare[None], scales[None], None, 7, 32)[0]
    assert torch.equal(a, b)


def test_struct_layouts():
    assert ctypes.sizeof(mk.MkW4) == 3 * 8 + 6 * 4
    assert ctypes.sizeof(mk.MkRoute) == 10 * 4


def weight(N=32, K=64, group=32, E=None, zeros=False, dtype=torch.bfloat16):
    shape = (N, K) if E is None else (E, N, K)
    return quantize_w4(torch.ones(*shape).to(dtype), group, zeros)


@pytest.mark.parametrize("make", [
    lambda: w4.W4Linear(*weight(), k=64, group=16),
    lambda: w4.W4Linear(*weight(), k=66, group=32),
    lambda: w4.W4Linear(weight()[0].int(), weight()[1], k=64, group=32),
    lambda: w4.W4Linear(weight()[0], weight()[1].float(), k=64, group=32),
    lambda: w4.W4Linear(weight()[0], weight()[1][:, :1], k=64, group=32),
    lambda: w4.W4Linear(weight()[0], weight()[1], torch.zeros(32, 1, dtype=torch.uint8), k=64, group=32),
    lambda: w4.W4Linear(*weight(E=2), k=64, group=32),
    lambda: w4.W4Experts(weight(E=2, N=64, K=32), weight(E=3, N=32, K=32), group=32),
    lambda: w4.W4Experts(weight(E=2, N=64, K=32), weight(E=2, N=32, K=64), group=32, inter=64),
    lambda: w4.W4Experts(weight(E=2, N=64, K=32), weight(E=2, N=32, K=32, dtype=torch.float16), group=32, inter=32),
])
def test_constructors_refuse(make):
    with pytest.raises(ValueError):
        make()


def test_calls_on_cpu_tensors_are_refused():
    from fleet.routing import route_experts
    lin = w4.W4Linear(*weight(), k=64, group=32)
    with pytest.raises(mk.MkError):
        lin(torch.zeros(1, 64, dtype=torch.bfloat16))
    with pytest.raises(mk.MkError):
        route_experts(torch.zeros(1, 8), 2)


@pytest.mark.parametrize("kw", [dict(score="tanh"), dict(group_score="mean")])
def test_route_refuses_unknown_names(kw):
    from fleet.routing import route_experts
    with pytest.raises(ValueError):
        route_experts(torch.zeros(1, 8), 2, **kw)


ROUTE = dict(experts=64, topk=6, n_forced=0, n_group=1, topk_group=1, group_top2=0, score=0, renormalize=0,
             logits_dtype=0, scaling=1.0)


@needs_lib
@pytest.mark.parametrize("change", [dict(experts=0), dict(experts=513), dict(topk=0), dict(topk=33), dict(experts=4),
                                    dict(n_group=5), dict(n_group=0), dict(topk_group=2), dict(n_group=64, topk_group=8),
                                    dict(n_group=16, topk_group=1), dict(n_forced=-1), dict(n_forced=33), dict(score=2),
                                    dict(logits_dtype=2)])
def test_route_refuses_parameters(change):
    r = mk.MkRoute(**{**ROUTE, **change})
    assert mk.lib().mk_route(ctypes.addressof(r), 256, 64, 1, None, 256, 256, None) == mk.MK_EINVAL
    assert mk.lib().mk_last_error()


@needs_lib
def test_route_refuses_arguments():
    r = mk.MkRoute(**ROUTE)
    p = ctypes.addressof(r)
    call = mk.lib().mk_route
    assert call(p, 256, 64, -1, None, 256, 256, None) == mk.MK_EINVAL
    assert call(p, None, 64, 1, None, 256, 256, None) == mk.MK_EINVAL
    assert call(p, 256, 64, 1, None, None, 256, None) == mk.MK_EINVAL
    assert call(p, 257, 64, 1, None, 256, 256, None) == mk.MK_EINVAL
    assert call(None, 256, 64, 1, None, 256, 256, None) == mk.MK_EINVAL
    assert call(p, None, 64, 0, None, None, None, None) == mk.MK_OK        # no tokens: nothing to do


def c_weight(n=32, k=64, group=32, dtype=0, experts=1, codes=4096):
    return mk.MkW4(codes, 4096, None, n, k, group, dtype, experts, 0)


@needs_lib
@pytest.mark.parametrize("w", [dict(n=0), dict(k=0), dict(group=48), dict(dtype=2), dict(experts=0), dict(experts=2),
                               dict(codes=8), dict(codes=None), dict(k=1 << 20)])
def test_linear_refuses_weights(w):
    c = c_weight(**w)
    assert mk.lib().mk_w4_linear(ctypes.addressof(c), 4096, 64, 1, None, 0, 4096, 32, 0, None) in (mk.MK_EINVAL, mk.MK_ECUDA)
    if w != dict(k=1 << 20):          # too long a row is found after the device's size is asked for
        assert mk.lib().mk_w4_linear(ctypes.addressof(c), 4096, 64, 1, None, 0, 4096, 32, 0, None) == mk.MK_EINVAL


@needs_lib
def test_linear_refuses_arguments():
    c = c_weight()
    p = ctypes.addressof(c)
    call = mk.lib().mk_w4_linear
    assert call(p, 4096, 64, -1, None, 0, 4096, 32, 0, None) == mk.MK_EINVAL
    assert call(p, None, 64, 1, None, 0, 4096, 32, 0, None) == mk.MK_EINVAL
    assert call(p, 4097, 64, 1, None, 0, 4096, 32, 0, None) == mk.MK_EINVAL
    assert call(p, 4096, 64, 1, None, 0, 4098, 32, 1, None) == mk.MK_EINVAL    # FP32 output at a 2-byte boundary
    assert call(None, 4096, 64, 1, None, 0, 4096, 32, 0, None) == mk.MK_EINVAL
    assert call(p, None, 64, 0, None, 0, None, 32, 0, None) == mk.MK_OK


@needs_lib
def test_experts_refuse():
    a, b = c_weight(n=2 * 96, k=64, experts=4), c_weight(n=64, k=96, experts=4)
    pa, pb = ctypes.addressof(a), ctypes.addressof(b)
    need = ctypes.c_int64()
    size = lambda p, q, t, s: mk.lib().mk_w4_experts_workspace(p, q, t, s, ctypes.byref(need))  # noqa: E731
    assert size(pa, pb, 3, 2) == mk.MK_OK and need.value > 3 * 2 * 96 * 2
    assert size(pa, pa, 3, 2) == mk.MK_EINVAL
    assert size(pa, pb, -1, 2) == mk.MK_EINVAL and size(pa, pb, 1, -2) == mk.MK_EINVAL
    assert size(pa, pb, 1 << 20, 64) == mk.MK_EINVAL
    for other in (c_weight(n=64, k=95, experts=4), c_weight(n=63, k=96, experts=4), c_weight(n=64, k=96, experts=5),
                  c_weight(n=64, k=96, experts=4, dtype=1)):
        assert size(pa, ctypes.addressof(other), 3, 2) == mk.MK_EINVAL
    many = c_weight(n=192, k=64, experts=1025), c_weight(n=64, k=96, experts=1025)
    assert size(*map(ctypes.addressof, many), 1, 1) == mk.MK_EINVAL
    call = mk.lib().mk_w4_experts
    size(pa, pb, 3, 2)
    ok = [pa, pb, 4096, 64, 4096, 4096, 3, 2, None, 0, 8192, 64, 1 << 20, need.value, None]

    def with_(i, v):
        return [v if j == i else u for j, u in enumerate(ok)]
    for i, v in ((2, None), (2, 4097), (4, None), (5, None), (10, None), (12, None), (12, (1 << 20) + 16), (13, need.value - 1)):
        assert call(*with_(i, v)) == mk.MK_EINVAL, (i, v)
    assert call(*with_(6, 0)) == mk.MK_OK


def test_output_rules():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    base = torch.zeros(4, 128, dtype=torch.bfloat16)
    shape, dts = (4, 32), (torch.bfloat16, torch.float32)
    assert w4._out(base[:, 32:64], shape, dts, x.device, x, None) == 128
    assert w4._out(base[:, :32], shape, dts, x.device, x, base[:, :32]) == 128          # the residual itself
    for out, xx, res in [(base[:, :32], base[:, 64:], None),                            # spans x's rows
                         (base[:, 0:32], x, base[:, 16:48]),                            # half the residual
                         (base[:, :64:2], x, None), (base[:1, :32].expand(4, 32), x, None), (base[:, :31], x, None)]:
        with pytest.raises(ValueError):
            w4._out(out, shape, dts, x.device, xx, res)
