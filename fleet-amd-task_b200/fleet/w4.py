"""4-bit weights for a batch of sequences: W4Linear (one weight) and W4Experts (a layer's routed
experts), over mk_w4_linear / mk_w4_experts (csrc/mk_w4.cu).

A 4-bit weight W [..., N, K] is

* ``codes`` [..., N, ceil(K / 2)] uint8, the even k in the low nibble,
* ``scales`` [..., N, ceil(K / group)] of the activations' type (bfloat16 or float16),
* ``zeros`` [..., N, ceil(K / group)] uint8 in 0..15, or None (8 everywhere),

with W[n, k] = scales[n, k // group] * (code[n, k] - zeros[n, k // group]) and group 32, 64 or 128
(pack_weights.quantize_w4 makes one from a BF16 weight). The constructors lay the codes out once in
the order the kernels stream them (csrc/mk_w4.cuh) and keep only that form.

A call repeated gives the same bits. A token's sums are split by where its block of tokens or its expert's slots
lie, so its last bits may differ between batches of other sizes or routing.
"""
import ctypes

import torch

from fleet import mk

DTYPES = {torch.bfloat16: 0, torch.float16: 1}
GROUPS = (32, 64, 128)


def lay_out(codes, scales, zeros, k, group, gate_up=False):
    """(codes, scales, zeros) of weights [E, N, K] in the kernels' order (csrc/mk_w4.cuh): codes
    [E, strips, units, 2048] uint8, scales and zeros [E, strips, units, 2, 8, 128 / group, 2]. gate_up:
    rows 2i / 2i + 1 are gate / up row i (pack_weights.interleave_gate_up) and a tile takes 8 gate
    rows, then their 8 up rows."""
    E, N = codes.shape[:2]
    strips, units = -(-N // 32), -(-k // 128)

    def rows(v, fill):
        """[E, N, m] -> [E, strips, 2 (tile), 2 (row g, row g + 8), 8 (g), m]"""
        v = torch.nn.functional.pad(v, (0, 0, 0, strips * 32 - N), value=fill)
        if gate_up:
            return v.view(E, strips, 2, 8, 2, -1).transpose(3, 4)
        return v.view(E, strips, 2, 2, 8, -1)

    q = torch.full((E, N, units * 128), 8, dtype=torch.uint8, device=codes.device)
    q[..., 0:k:2] = codes[..., :(k + 1) // 2] & 15
    q[..., 1:k:2] = codes[..., :k // 2] >> 4
    # k = 128 unit + 64 chunk + 32 h + 8 t + 4 j + 2 p + half; a word's bytes: (half, p), its nibbles: the two rows
    q = rows(q, 8)
    q = (q[:, :, :, 0] | (q[:, :, :, 1] << 4)).view(E, strips, 2, 8, units, 2, 2, 4, 2, 2, 2)
    # e, strip, tile, g, unit, chunk, h, t, j, p, half -> e, strip, unit, tile, chunk, g, t, h, j, half, p
    q = q.permute(0, 1, 4, 2, 5, 3, 7, 6, 8, 10, 9).contiguous().view(E, strips, units, 2048)

    def grouped(v, fill):
        v = torch.nn.functional.pad(v, (0, units * 128 // group - v.shape[-1]), value=fill)
        v = rows(v, fill).view(E, strips, 2, 2, 8, units, 128 // group)
        # e, strip, tile, row half, g, unit, group -> e, strip, unit, tile, g, group, row half
        return v.permute(0, 1, 5, 2, 4, 6, 3).contiguous().view(E, strips, units, 2, 8, 128 // group, 2)

    return q, grouped(scales, 0), None if zeros is None else grouped(zeros, 8)


class W4Weight:
    """A laid-out weight [E, N, K] (or [N, K]) and the struct the library reads."""

    def __init__(self, codes, scales, zeros=None, k=None, group=128, gate_up=False):
        if codes.dim() == 2:
            codes, scales, zeros = codes[None], scales[None], None if zeros is None else zeros[None]
        k = 2 * codes.shape[-1] if k is None else k
        if group not in GROUPS:
            raise ValueError(f"group {group} is one of {GROUPS}")
        E, N = codes.shape[0], codes.shape[1] if codes.dim() == 3 else 0
        want = (E, N, -(-k // group))
        if codes.dim() != 3 or codes.dtype != torch.uint8 or k < 1 or codes.shape[2] != (k + 1) // 2 or N < 1 or E < 1:
            raise ValueError(f"codes [N, {(k + 1) // 2}] uint8 expected for k = {k}, got {codes.dtype} {tuple(codes.shape)}")
        if scales.dtype not in DTYPES or tuple(scales.shape) != want:
            raise ValueError(f"scales {want} bfloat16 or float16 expected, got {scales.dtype} {tuple(scales.shape)}")
        if zeros is not None and (zeros.dtype != torch.uint8 or tuple(zeros.shape) != want):
            raise ValueError(f"zeros {want} uint8 expected, got {zeros.dtype} {tuple(zeros.shape)}")
        if gate_up and N % 2:
            raise ValueError(f"gate and up rows come in pairs, got {N} rows")
        if any(v is not None and v.device != codes.device for v in (scales, zeros)):
            raise ValueError("codes, scales and zeros are on one device")
        if zeros is not None and int(zeros.max()) > 15:
            raise ValueError("zero points are in 0..15")
        self.n, self.k, self.group, self.experts, self.dtype, self.device = N, k, group, E, scales.dtype, codes.device
        self.index = -1 if codes.device.index is None else codes.device.index
        self.codes, self.scales, self.zeros = lay_out(codes, scales, zeros, k, group, gate_up)
        self.c = mk.MkW4(self.codes.data_ptr(), self.scales.data_ptr(), mk._ptr(self.zeros), N, k, group,
                         DTYPES[scales.dtype], E, 0)
        self.ptr = ctypes.addressof(self.c)
        self.tensors = self.codes, self.scales, self.zeros


def _fits(t, shape, dtype, index):
    """The row stride of t if it is `shape` of dtype on CUDA device `index` (-1: the CPU) with unit column
    stride, or None."""
    if t.dtype is not dtype or t.shape != shape or t.get_device() != index:
        return None
    rows, cols = t.stride()
    return rows if cols == 1 or shape[1] == 1 else None


def _refuse(t, shape, dtypes, device, name):
    raise ValueError(f"{name}: {' or '.join(map(str, dtypes))} {shape} with unit stride along its rows on {device} "
                     f"expected, got {t.dtype} {tuple(t.shape)}, strides {t.stride()} on {t.device}")


def _span(t):
    """[first byte, past the last byte) of a 2-D tensor of unit column stride."""
    n = ((t.shape[0] - 1) * t.stride(0) + t.shape[1]) * t.element_size() if t.numel() else 0
    return t.data_ptr(), t.data_ptr() + n


def _out(out, shape, dtypes, device, x, residual):
    """The row stride of a caller's output: rows apart from one another and from x, and the residual's
    own rows or none of them."""
    ld = _fits(out, shape, out.dtype, -1 if device.index is None else device.index)
    if ld is None or out.dtype not in dtypes:
        _refuse(out, shape, dtypes, device, "out")
    if shape[0] > 1 and ld < shape[1]:
        raise ValueError(f"out: rows overlap (stride {ld}, {shape[1]} values)")
    lo, hi = _span(out)
    apart = lambda t: _span(t)[1] <= lo or hi <= _span(t)[0]  # noqa: E731
    if not apart(x):
        raise ValueError("out overlaps x")
    if residual is not None and not apart(residual) and not (
            residual.data_ptr() == lo and (shape[0] == 1 or residual.stride(0) == ld) and residual.dtype == out.dtype):
        raise ValueError("out is the residual itself or apart from it")
    return ld


class W4Linear:
    """out [T, N] = x [T, K] W^T (+ residual [T, N]) with a 4-bit W, for the tokens of a decode or
    verification step. x in the scales' type with any row stride; products and sums are FP32 and rounded
    once, to the type of x or not at all (out_dtype / out float32). Runs on `stream` (default: the
    current stream of the weight's device)."""

    def __init__(self, codes, scales, zeros=None, k=None, group=128):
        if codes.dim() != 2:
            raise ValueError(f"codes [N, ceil(K / 2)] expected, got {tuple(codes.shape)}")
        self.w = W4Weight(codes, scales, zeros, k, group)

    def __call__(self, x, out=None, residual=None, out_dtype=None, stream=None):
        if stream is not None:
            with mk.on_stream(x, stream, out, residual, *self.w.tensors):
                return self(x, out, residual, out_dtype)
        w = self.w
        call, device, current_stream, context = mk.entry("mk_w4_linear")
        n, index, dtype = w.n, w.index, w.dtype
        if index < 0 or device() != index:
            return mk.off_device("mk_w4_linear", index, context, lambda: self(x, out, residual, out_dtype))
        T = x.shape[0] if x.dim() == 2 else -1
        ldx = _fits(x, (T, w.k), dtype, index)
        if ldx is None:
            _refuse(x, ("T", w.k), (dtype,), w.device, "x")
        shape = (T, n)
        res = ldr = 0
        if residual is not None:
            ldr = _fits(residual, shape, dtype, index)
            if ldr is None:
                _refuse(residual, shape, (dtype,), w.device, "residual")
            res = residual.data_ptr()
        if out is None:
            if out_dtype is None:
                out_dtype = dtype
            elif out_dtype is not dtype and out_dtype is not torch.float32:
                raise ValueError(f"out_dtype is {dtype} or float32, not {out_dtype}")
            out, ldo = torch.empty_strided(shape, (n, 1), dtype=out_dtype, device=w.device), n
        else:
            if out_dtype is not None and out_dtype != out.dtype:
                raise ValueError(f"out is {out.dtype}, out_dtype {out_dtype}")
            ldo, out_dtype = _out(out, shape, (dtype, torch.float32), w.device, x, residual), out.dtype
        rc = call(w.ptr, x.data_ptr(), ldx, T, res, ldr, out.data_ptr(), ldo, out_dtype is torch.float32, current_stream(index))
        if rc:
            mk._check(rc, "mk_w4_linear")
        return out


class W4Experts:
    """The routed experts of a layer with 4-bit weights: out [T, H] = (residual [T, H] +) the sum over a
    token's slots of weights[t, s] W2[e] (silu(g) u), (g, u) = W13[e] x[t], e = ids[t, s].

    w13, w2: (codes, scales, zeros or None) of W13 [E, 2 I, H] (gate/up rows interleaved as
    pack_weights packs them) and W2 [E, H, I] (`inter` = I). ids [T, S] int32 and weights [T, S] float32 as
    route_experts returns them; a slot whose id is outside [0, E) is empty. The intermediate
    silu(g) u is held to 16 significant bits in FP32's range, all sums are FP32, rounded once. Runs on
    `stream` (default: the current stream); the workspace comes from torch's allocator for each call,
    so calls on several streams do not share one."""

    def __init__(self, w13, w2, group=128, inter=None):
        hidden = w2[0].shape[1] if w2[0].dim() == 3 else -1
        if w13[0].dim() != 3 or w2[0].dim() != 3 or w13[0].shape[0] != w2[0].shape[0]:
            raise ValueError(f"w13 [E, 2 I, H / 2] and w2 [E, H, I / 2] codes expected, got {tuple(w13[0].shape)} and {tuple(w2[0].shape)}")
        inter = w13[0].shape[1] // 2 if inter is None else inter
        self.w13 = W4Weight(*w13, k=hidden, group=group, gate_up=True)
        self.w2 = W4Weight(*w2, k=inter, group=group)
        if self.w13.n != 2 * inter or self.w13.dtype != self.w2.dtype or self.w13.device != self.w2.device:
            raise ValueError(f"w13 has {self.w13.n} rows, {self.w13.dtype}, {self.w13.device}; w2 has rows of {inter}, {self.w2.dtype}, {self.w2.device}")
        self.hidden = hidden
        self._need = {}            # (T, S) -> workspace bytes

    def workspace_bytes(self, T, S):
        got = self._need.get((T, S))
        if got is None:
            n = ctypes.c_int64()
            mk._check(mk.lib().mk_w4_experts_workspace(self.w13.ptr, self.w2.ptr, T, S, ctypes.byref(n)),
                      "mk_w4_experts_workspace")
            if len(self._need) > 4096:
                self._need.clear()
            got = self._need[(T, S)] = n.value
        return got

    def __call__(self, x, ids, weights, residual=None, out=None, stream=None):
        if stream is not None:
            with mk.on_stream(x, stream, ids, weights, residual, out, *self.w13.tensors, *self.w2.tensors):
                return self(x, ids, weights, residual, out)
        w = self.w13
        call, device, current_stream, context = mk.entry("mk_w4_experts")
        H, index, dtype = self.hidden, w.index, w.dtype
        if index < 0 or device() != index:
            return mk.off_device("mk_w4_experts", index, context, lambda: self(x, ids, weights, residual, out))
        T = x.shape[0] if x.dim() == 2 else -1
        shape = (T, H)
        ldx = _fits(x, shape, dtype, index)
        if ldx is None:
            _refuse(x, ("T", H), (dtype,), w.device, "x")
        slots = (T, ids.shape[1] if ids.dim() == 2 else -1)
        if _fits(ids, slots, torch.int32, index) is None or not ids.is_contiguous():
            raise ValueError(f"ids: contiguous int32 [{T}, S] on {w.device} expected, got {ids.dtype} {tuple(ids.shape)} on {ids.device}")
        if _fits(weights, slots, torch.float32, index) is None or not weights.is_contiguous():
            raise ValueError(f"weights: contiguous float32 {slots} on {w.device} expected, got {weights.dtype} "
                             f"{tuple(weights.shape)} on {weights.device}")
        res = ldr = 0
        if residual is not None:
            ldr = _fits(residual, shape, dtype, index)
            if ldr is None:
                _refuse(residual, shape, (dtype,), w.device, "residual")
            res = residual.data_ptr()
        if out is None:
            out, ldo = torch.empty_strided(shape, (H, 1), dtype=dtype, device=w.device), H
        else:
            ldo = _out(out, shape, (dtype,), w.device, x, residual)
        nbytes = self._need.get(slots) or self.workspace_bytes(*slots)
        ws = torch.empty_strided((nbytes,), (1,), dtype=torch.uint8, device=w.device)
        rc = call(w.ptr, self.w2.ptr, x.data_ptr(), ldx, ids.data_ptr(), weights.data_ptr(), T, slots[1], res, ldr,
                  out.data_ptr(), ldo, ws.data_ptr(), nbytes, current_stream(index))
        if rc:
            mk._check(rc, "mk_w4_experts")
        return out
