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


def test_one_row_in_place_whatever_its_row_stride_says():
    """The stride of a single row names no memory: the last token of a sequence and a row of its own are one place."""
    x, h = torch.zeros(1, 64, dtype=torch.bfloat16), torch.zeros(1, 5, 32, dtype=torch.bfloat16)
    shape, dtypes = (1, 32), (torch.bfloat16,)
    out, residual = h[:, -1], h.view(-1, 32)[-1:]
    assert out.stride(0) != residual.stride(0) and out.data_ptr() == residual.data_ptr()
    w4._out(out, shape, dtypes, x.device, x, residual)
    with pytest.raises(ValueError):
        w4._out(h.view(-1)[16:48].view(1, 32), shape, dtypes, x.device, x, h.view(-1)[:32].view(1, 32))
