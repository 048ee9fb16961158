"""Rotary positions of a batch of tokens (mk_rope, csrc/mk_rope.cu).

The persistent kernel turns the rotary part of its one token by the model's tables; this turns any part
of the heads of a batch at any positions, in the three layouts that checkpoints have, with angles
counted in 64 bits: positions far beyond a table's end cost no precision.
"""
import ctypes
import math

import torch

from fleet import capture, mk

LAYOUTS = {"half": 0, "interleaved": 1, "pairs_to_half": 2}
DTYPES = {torch.bfloat16: 0, torch.float16: 1}
POSITIONS = {torch.int32: 0, torch.int64: 1}
MOST = 2 ** 31 - 1       # what the library counts tokens, heads and their values with has 32 bits


def _apart(shape, strides):
    """Whether the heads of a tensor [T, heads, width] of these strides are apart from one another."""
    (T, H, W), (t, h, _) = shape, strides
    return ((H <= 1 or h >= W) and (T <= 1 or t >= (max(H, 1) - 1) * h + W)) or \
        ((T <= 1 or t >= W) and (H <= 1 or h >= (max(T, 1) - 1) * t + W))


def _span(t):
    """[first byte, past the last byte) of a tensor."""
    if t.numel() == 0:
        return t.data_ptr(), t.data_ptr()
    n = sum((s - 1) * d for s, d in zip(t.shape, t.stride())) + 1
    return t.data_ptr(), t.data_ptr() + n * t.element_size()


def overlap(a, b):
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a0 < b1 and b0 < a1


class Rope:
    """rope(x, positions) turns pairs of values of x [T, heads, width] (or [T, width]) at the tokens'
    positions [T] (int32 or int64): pair i, (a, b), becomes (a cos t - b sin t, b cos t + a sin t)
    times `scale`, t = position x inv_freq[i]. `inv_freq` [dim / 2] are radians a position, float64 or
    float32 (taken as they are). The pairs of a head's values [start, start + dim) are

    * "half": i and i + dim / 2,
    * "interleaved": 2 i and 2 i + 1,
    * "pairs_to_half": read at 2 i and 2 i + 1, written to i and i + dim / 2: the layout of this
      model's checkpoints, and of the rotary keys in its cache.

    Values are bfloat16 or float16, computed in FP32 and rounded once. The values of a head outside
    the part are copied. `out` may be x itself (in place) or a tensor apart from it; a token at a
    negative position is left out, its output stays as it was (without `out`, undefined). Heads need
    unit stride along their values; tokens and heads may have any. Runs on `stream` (default: the
    current stream of the tensors' device)."""

    def __init__(self, inv_freq, scale=1.0, layout="half"):
        if layout not in LAYOUTS:
            raise ValueError(f"layout {layout!r} is one of {list(LAYOUTS)}")
        if inv_freq.dim() != 1 or not 1 <= inv_freq.shape[0] <= 256 or inv_freq.dtype not in (torch.float32, torch.float64):
            raise ValueError(f"inv_freq [dim / 2] float64 or float32, dim from 2 to 512, expected, got {inv_freq.dtype} {tuple(inv_freq.shape)}")
        if not math.isfinite(scale):
            raise ValueError(f"scale {scale} is not finite")
        self.inv_freq = inv_freq.detach().to(torch.float64, copy=True).contiguous()
        self.dim, self.layout, self.scale = 2 * inv_freq.shape[0], layout, float(scale)
        self.device = inv_freq.device
        self.index = -1 if inv_freq.device.index is None else inv_freq.device.index
        self._c, self._structs = {}, []        # (dtype, dtype of the positions) -> a struct's address

    @classmethod
    def yarn(cls, dim, layout="pairs_to_half", device="cuda", **parameters):
        """The model's rotary positions (fleet.capture.YARN, or `parameters` in their place): its stretched
        frequencies, and the ratio of its magnitudes as the scale."""
        y = dict(capture.YARN, **parameters)
        inv = capture.yarn_inv_freq(dim, y["base"], y["factor"], y["original_max_position_embeddings"], y["beta_fast"], y["beta_slow"])
        scale = capture.yarn_get_mscale(y["factor"], y["mscale"]) / capture.yarn_get_mscale(y["factor"], y["mscale_all_dim"])
        return cls(inv.to(device), scale, layout)

    def _params(self, dtype, positions):
        if dtype not in DTYPES or positions not in POSITIONS:
            raise TypeError(f"x is bfloat16 or float16 and positions are int32 or int64, not {dtype} and {positions}")
        c = mk.MkRope(self.inv_freq.data_ptr(), self.dim, LAYOUTS[self.layout], DTYPES[dtype], POSITIONS[positions], self.scale, 0)
        self._structs.append(c)
        p = self._c[(dtype, positions)] = ctypes.addressof(c)
        return p

    def __call__(self, x, positions, start=0, out=None, stream=None):
        if stream is not None:
            with mk.on_stream(x, stream, positions, out, self.inv_freq):
                return self(x, positions, start, out)
        call, device, current_stream, context = mk.entry("mk_rope")
        index = self.index
        if index < 0 or device() != index:
            return mk.off_device("mk_rope", index, context, lambda: self(x, positions, start, out))
        if x.dim() == 2:
            if out is not None and out.dim() != 2:
                raise ValueError(f"out: {x.dtype} {tuple(x.shape)} expected, got {out.dtype} {tuple(out.shape)}")
            y = self(x[:, None], positions, start, None if out is None else out[:, None])
            return y[:, 0] if out is None else out
        if x.dim() != 3 or x.get_device() != index or (x.stride(2) != 1 and x.shape[2] > 1):
            raise ValueError(f"x [T, heads, width] with unit stride along width on {self.device} expected, got "
                             f"{tuple(x.shape)}, strides {x.stride()} on {x.device}")
        T, H, W = x.shape
        xt, xh, _ = x.stride()
        if T > MOST or H > MOST or W > MOST:
            raise ValueError(f"x: fewer than 2^31 tokens, heads and values of a head expected, got {tuple(x.shape)}")
        if positions.dim() != 1 or positions.shape[0] != T or positions.get_device() != index or (T > 1 and positions.stride(0) != 1):
            raise ValueError(f"positions: contiguous [{T}] on {self.device} expected, got {tuple(positions.shape)} on {positions.device}")
        if not 0 <= start <= W - self.dim:
            raise ValueError(f"the {self.dim} rotary values from {start} on do not lie within a head of {W}")
        params = self._c.get((x.dtype, positions.dtype)) or self._params(x.dtype, positions.dtype)
        if out is None:
            out = torch.empty_strided((T, H, W), (H * W, W, 1), dtype=x.dtype, device=x.device)
            ot, oh = H * W, W
        else:
            if out.shape != x.shape or out.dtype != x.dtype or out.get_device() != index or (W > 1 and out.stride(2) != 1):
                raise ValueError(f"out: {x.dtype} {tuple(x.shape)} with unit stride along width on {self.device} expected, got "
                                 f"{out.dtype} {tuple(out.shape)}, strides {out.stride()} on {out.device}")
            ot, oh, _ = out.stride()
            if not _apart((T, H, W), out.stride()):
                raise ValueError(f"out: heads overlap (strides {out.stride()}, {W} values)")
            same = out.data_ptr() == x.data_ptr() and (T <= 1 or ot == xt) and (H <= 1 or oh == xh)
            if not same and overlap(x, out):
                raise ValueError("out is x itself or apart from it")
            if overlap(positions, out):
                raise ValueError("out overlaps the positions")
            if same:
                xt, xh = ot, oh
        rc = call(params, positions.data_ptr(), T, x.data_ptr(), xt, xh, H, W, start, out.data_ptr(), ot, oh, current_stream(index))
        if rc:
            mk._check(rc, "mk_rope")
        return out
