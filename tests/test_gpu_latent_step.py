"""harness/run_w4.py --context: the projections, rotary positions, the cache and the attention over it run together with
the rest of the layers, against the same step in FP32 over the dequantised weights and the cached latents.

Either side rounds the attention's half of a layer to BF16 (2^-8 each at most) at the norm, the projections, the rotary
parts, the absorbed query, the attention's output, the value projection and the residual: 7, of which the
first 4 reach the scores, whose terms' sizes sum up to S: a weight is off by at most 2 x 4 x 2^-8 S of itself. So a layer
parts by at most 2 x (7 + 8 S) 2^-8 and its other half, as in the step without attention, by 2 x 3 x 2^-8."""
import pytest

pytestmark = pytest.mark.gpu

SMALL = "H=256,NH=4,D_N=32,D_R=16,D_V=32,D_C=64,V=1000,L=3,I_DENSE=384,I_MOE=72,E=16,TOPK=4,N_SHARED=2"


@pytest.mark.parametrize("tokens,context,zero_point,std", [(1, 1, False, 0.02), (5, 200, True, 0.02), (24, 700, False, 0.02), (9, 333, False, 0.04)])
def test_step_with_attention_equals_fp32(tokens, context, zero_point, std):
    from harness import run_w4
    out = run_w4.main(["--dims", SMALL, "--tokens", str(tokens), "--context", str(context), "--group", "32", "--steps", "2", "--std", str(std),
                       "--check"] + (["--zero-point"] if zero_point else []))
    assert len(out["ids"]) == tokens
    layer = 2 * (7 + 8 * out["score_terms"] + 3) * 2.0 ** -8
    assert max(out["residual_distance"]) <= 2 * layer < 1
    assert out["logits_distance"] <= 2 * layer + 2 * 2.0 ** -8


def test_attention_outweighs_a_small_residual():
    """A residual of 2^-10: the norm undoes it, and what comes out is the attention itself."""
    import torch
    from fleet.pack_weights import Dims, synthetic_packed
    from harness import run_w4
    d = Dims(**{k: int(v) for k, v in (f.split("=") for f in SMALL.split(","))})
    packed = synthetic_packed(d, layers=2, head=True, seed=3, device="cuda", std=0.06)
    lens = [1, 64, 65, 200, 7]
    attention = run_w4.W4Attention(packed, d, 1, lens, group=32)
    x = (torch.randn(5, d.H, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda") * 2.0 ** -10).bfloat16()
    got = attention(x)
    want, terms = attention.plain(x)
    assert x.norm() < 0.02 * want.norm() and 2 * (7 + 8 * terms) * 2.0 ** -8 < 1
    for g, w in zip(got.float(), want.float()):
        assert (g - w).norm() <= 2 * (7 + 8 * terms) * 2.0 ** -8 * w.norm()
    assert run_w4.distance(got, want) < 0.05 < run_w4.distance(got.flip(0), want)


def test_step_repeats_its_bits():
    from harness import run_w4
    args = ["--dims", SMALL, "--tokens", "6", "--context", "300", "--group", "64", "--steps", "1"]
    assert run_w4.main(args) == {**run_w4.main(args), "ms_per_step": pytest.approx(0, abs=1e9)}
