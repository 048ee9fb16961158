"""Arguments of the 4-bit products that are refused, or accepted, without a GPU."""
import pytest
import torch

from fleet import w4
from fleet.pack_weights import quantize_w4


def test_zero_points_past_15_are_refused():
    """A BF16 operand's mantissa holds a code or a zero point of up to 127; the format's end at 15."""
    codes, scales, zeros = quantize_w4(torch.randn(8, 64, generator=torch.Generator().manual_seed(1)).bfloat16(), 32, True)
    w4.W4Linear(codes, scales, zeros, group=32)
    zeros[3, 1] = 16
    with pytest.raises(ValueError):
        w4.W4Linear(codes, scales, zeros, group=32)
    with pytest.raises(ValueError):
        w4.W4Experts((codes[None], scales[None], zeros[None]), (torch.zeros(1, 64, 2, dtype=torch.uint8), torch.ones(1, 64, 1).bfloat16(), None),
                     group=32, inter=4)
