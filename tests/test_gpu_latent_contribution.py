"""What the attention adds to a step of harness/run_w4.py, against FP32 over the same weights, where it is most of what comes out:
a residual of 2^-10, which the norms undo. The bound is test_gpu_latent_step.py's, with S the largest sum of a score's terms:
2 x (7 + 8 S + 3) 2^-8 a layer. That it sees the attention is shown by steps that lack it, or attend to another's tokens."""
import pytest
import torch

pytestmark = pytest.mark.gpu

SMALL = "H=256,NH=4,D_N=32,D_R=16,D_V=32,D_C=64,V=1000,L=3,I_DENSE=384,I_MOE=72,E=16,TOPK=4,N_SHARED=2"


def model_of(packed, dims, lens):
    from harness import run_w4
    return run_w4.W4Layers(packed, dims, range(1, 3), 32, False, lens)


@pytest.mark.parametrize("lens", [[1, 2, 3, 4, 5], [1, 64, 65, 200, 7], [3, 90] * 12])
def test_the_attention_in_a_step(lens):
    from fleet.pack_weights import Dims, synthetic_packed
    from harness import run_w4
    d = Dims(**{k: int(v) for k, v in (f.split("=") for f in SMALL.split(","))})
    packed = synthetic_packed(d, layers=3, head=True, seed=3, device="cuda", std=0.02)
    x = (torch.randn(len(lens), d.H, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda") * 2.0 ** -10).bfloat16()
    model = model_of(packed, d, lens)
    ids, logits, residuals, routes = model.step(x)
    want, want_logits, terms = model.plain_and_terms(x, routes)
    layer = 2 * (7 + 8 * terms + 3) * 2.0 ** -8
    assert 2 * layer + 2 * 2.0 ** -8 < 0.75
    assert max(run_w4.distance(r, w) for r, w in zip(residuals, want)) <= 2 * layer
    assert run_w4.distance(logits, want_logits) <= 2 * layer + 2 * 2.0 ** -8
    first = model.attention[0]
    y, p = first(x), first.plain(x)[0]
    assert run_w4.distance(y.float() - x.float(), p.float() - x.float()) <= layer
    # without it, and with each sequence's tokens another's
    lacking = model_of(packed, d, None).step(x)[2]
    assert min(run_w4.distance(r, w) for r, w in zip(lacking, want)) > 2 * layer
    if len(set(lens)) == len(lens):
        shifted = torch.cat([y[1:], y[:1]])
        assert run_w4.distance(shifted.float() - x.float(), p.float() - x.float()) > layer


def test_plain_is_a_pair():
    """(residuals, logits), with the attention and without."""
    from fleet.pack_weights import Dims, synthetic_packed
    d = Dims(**{k: int(v) for k, v in (f.split("=") for f in SMALL.split(","))})
    packed = synthetic_packed(d, layers=3, head=True, seed=3, device="cuda", std=0.02)
    x = torch.randn(2, d.H, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").bfloat16()
    for lens in (None, [5, 9]):
        model = model_of(packed, d, lens)
        residuals, logits = model.plain(x, model.step(x)[3])
        again, same, terms = model.plain_and_terms(x, model.step(x)[3])
        assert len(residuals) == 2 and logits.shape == (2, d.V) and len(again) == 2 and same.shape == logits.shape
        assert (terms > 0) == (lens is not None)
