#!/usr/bin/env python3
"""One decode step of a batch through a MoE layer and the head in 4 bits: RMSNorm, the FP32 router,
route_experts, W4Experts with the residual, then the final norm and a W4Linear head with greedy ids.

    python harness/run_w4.py [--tokens 8] [--layers 2] [--group 128] [--zero-point] [--steps 20] [--check]

The weights are the benchmark's seeded synthetic BF16 ones (pack_weights.synthetic_packed) quantised
by pack_weights.quantize_w4; the layers' routers and norms stay as they are. Prints the time of a
step, and with --check the distance of its residuals and logits from the same step in FP32 over the
dequantised weights (the routing is taken from the 4-bit step, so a near-tie cannot part the two)."""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
from fleet import w4  # noqa: E402
from fleet.graph_plan import RMS_EPS  # noqa: E402
from fleet.pack_weights import Dims, dequantize_w4, quantize_w4, synthetic_packed  # noqa: E402
from fleet.routing import route_experts  # noqa: E402


def rms_norm(x, w):
    f = x.float()
    return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + RMS_EPS) * w.float()).to(x.dtype)


class W4Layers:
    """The MoE layers (after their attention) and the head of a packed model, experts and head in 4 bits."""

    def __init__(self, packed, dims: Dims, layers, group=128, zero_point=False):
        self.dims, self.group = dims, group
        quantize = lambda w: quantize_w4(w, group, zero_point)  # noqa: E731
        self.codes = [(quantize(packed[f"W13_{l}"]), quantize(packed[f"W2_{l}"])) for l in layers]
        self.experts = [w4.W4Experts(w13, w2, group=group, inter=dims.I_MOE) for w13, w2 in self.codes]
        self.gates = [packed[f"W_gate_{l}"].float() for l in layers]
        self.norms = [packed[f"w_norm2_{l}"] for l in layers]
        self.final_norm = packed["w_final_norm"]
        self.head_codes = quantize(packed["W_lm"])
        self.head = w4.W4Linear(*self.head_codes, k=dims.H, group=group)

    def step(self, x):
        """(ids [T], logits [T, V], residuals after each layer, (ids, weights) of each layer's routing)."""
        d, residuals, routes = self.dims, [], []
        for norm, gate, experts in zip(self.norms, self.gates, self.experts):
            h = rms_norm(x, norm)
            ids, weights = route_experts(h.float() @ gate.T, d.TOPK, n_forced=d.N_SHARED)
            x = experts(h, ids, weights, residual=x)
            residuals.append(x)
            routes.append((ids, weights))
        logits = self.head(rms_norm(x, self.final_norm), out_dtype=torch.float32)
        return logits.argmax(-1), logits, residuals, routes

    def plain(self, x, routes):
        """The residuals and logits of step(x) in FP32 over the dequantised weights, with step's routing."""
        d, residuals = self.dims, []
        for norm, (w13, w2), (ids, weights) in zip(self.norms, self.codes, routes):
            h, out = rms_norm(x, norm).float(), x.float()
            for e in ids.unique().tolist():
                t, s = (ids == e).nonzero(as_tuple=True)
                part = lambda w: [None if v is None else v[e] for v in w]  # noqa: E731, B023
                gu = h[t] @ dequantize_w4(*part(w13), d.H, self.group).T
                y = (torch.nn.functional.silu(gu[:, 0::2]) * gu[:, 1::2]) @ dequantize_w4(*part(w2), d.I_MOE, self.group).T
                out.index_add_(0, t, y * weights[t, s][:, None])
            x = out.to(x.dtype)
            residuals.append(x)
        return residuals, rms_norm(x, self.final_norm).float() @ dequantize_w4(*self.head_codes, d.H, self.group).T


def distance(a, b):
    return ((a.float() - b.float()).norm() / b.float().norm()).item()


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=8)
    ap.add_argument("--layers", type=int, default=2, help="MoE layers (1, 2, ...; layer 0 is dense)")
    ap.add_argument("--group", type=int, default=128, choices=w4.GROUPS)
    ap.add_argument("--zero-point", action="store_true")
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--check", action="store_true")
    ap.add_argument("--std", type=float, default=0.02, help="spread of the synthetic weights")
    ap.add_argument("--dims", default=None, help="Dims fields as name=value,... (default: the real model's)")
    a = ap.parse_args(argv)
    from fleet.pack_weights import REAL_DIMS
    dims = REAL_DIMS if a.dims is None else Dims(**{k: int(v) for k, v in (f.split("=") for f in a.dims.split(","))})
    layers = range(1, a.layers + 1)
    packed = synthetic_packed(dims, layers=a.layers + 1, head=True, seed=0, device="cuda", std=a.std)
    model = W4Layers(packed, dims, layers, a.group, a.zero_point)
    x = torch.randn(a.tokens, dims.H, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(torch.bfloat16)
    for _ in range(3):
        ids, logits, residuals, routes = model.step(x)
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    for _ in range(a.steps):
        model.step(x)
    end.record()
    torch.cuda.synchronize()
    out = {"tokens": a.tokens, "layers": a.layers, "ms_per_step": begin.elapsed_time(end) / a.steps, "ids": ids.tolist()}
    if a.check:
        want, want_logits = model.plain(x, routes)
        out["residual_distance"] = [distance(r, p) for r, p in zip(residuals, want)]
        out["logits_distance"] = distance(logits, want_logits)
    print(out)
    return out


if __name__ == "__main__":
    main()
