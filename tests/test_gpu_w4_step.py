"""harness/run_w4.py: the router, the experts and the head in 4 bits run together, against the same step in
FP32 over the dequantised weights. Each layer rounds to BF16 three times on either side (the norm, the
experts' activation, the residual; 2^-8 each at most), so two layers part by at most 2 x 3 x 2 x 2^-8, and the
logits by one norm's rounding on either side more. The weights' spread makes the experts' share of
the residual as large as the residual, so that a wrong expert, slot or weight is far outside that."""
import pytest

pytestmark = pytest.mark.gpu

SMALL = "H=256,NH=4,D_N=32,D_R=16,D_V=32,D_C=64,V=1000,L=3,I_DENSE=384,I_MOE=72,E=16,TOPK=4,N_SHARED=2"


@pytest.mark.parametrize("tokens,group,zero_point", [(1, 128, False), (5, 32, True), (24, 64, False)])
def test_step_equals_fp32_over_the_same_codes(tokens, group, zero_point):
    from harness import run_w4
    out = run_w4.main(["--dims", SMALL, "--tokens", str(tokens), "--group", str(group), "--steps", "2", "--std", "0.1", "--check"] +
                      (["--zero-point"] if zero_point else []))
    assert len(out["ids"]) == tokens
    assert max(out["residual_distance"]) <= 2 * 3 * 2 * 2.0 ** -8
    assert out["logits_distance"] <= (2 * 3 * 2 + 2) * 2.0 ** -8
