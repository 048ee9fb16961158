#!/usr/bin/env python3
"""One decode step of a batch through a MoE layer and the head in 4 bits: RMSNorm, the FP32 router,
route_experts, W4Experts with the residual, then the final norm and a W4Linear head with greedy ids.

    python harness/run_w4.py [--tokens 8] [--layers 2] [--group 128] [--zero-point] [--steps 20] [--check] [--context 1024]

With --context each layer begins with its attention: RMSNorm, W4Linear for queries and latents, the latent's norm,
Rope on the rotary parts, LatentCache.append and attend over sequences of up to that many tokens (a random cache of
latents in 8 bits stands for what came before), the value projection and a W4Linear with the residual.

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
from fleet.capture import softmax_scale  # noqa: E402
from fleet.graph_plan import RMS_EPS  # noqa: E402
from fleet.latent import LatentBatch, LatentCache  # noqa: E402
from fleet.pack_weights import Dims, dequantize_w4, quantize_w4, synthetic_packed  # noqa: E402
from fleet.rope import Rope  # noqa: E402
from fleet.routing import route_experts  # noqa: E402


def rms_norm(x, w):
    f = x.float()
    return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + RMS_EPS) * w.float()).to(x.dtype)


class W4Attention:
    """A layer's attention for a token of each sequence: projections in 4 bits, latents in an 8-bit cache. lens [T] are the
    sequences' tokens, the step's own included."""

    PAGE = 64

    def __init__(self, packed, dims: Dims, l, lens, group=128, zero_point=False):
        d = self.dims = dims
        self.group, self.scale, self.lens = group, softmax_scale(d.D_N, d.D_R), lens
        self.codes = [quantize_w4(packed[f"{w}_{l}"], group, zero_point) for w in ("W_qkva", "W_o")]
        self.qkva, self.o = (w4.W4Linear(*c, k=k, group=group) for c, k in zip(self.codes, (d.H, d.NH * d.D_V)))
        self.norm, self.kv_norm = packed[f"w_norm1_{l}"], packed[f"w_kv_norm_{l}"]
        self.uk, self.uv = packed[f"W_ukT_{l}"], packed[f"W_uv_{l}"]
        self.rope = Rope.yarn(d.D_R, device=self.uk.device)
        used = [-(-n // self.PAGE) for n in lens]
        g = torch.Generator(device=self.uk.device).manual_seed(l)
        order = torch.randperm(sum(used), generator=g, device=self.uk.device).int()
        table = torch.zeros(len(lens), max(used), dtype=torch.int32, device=self.uk.device)
        for b, n in enumerate(used):
            table[b, :n] = order[sum(used[:b]):sum(used[:b + 1])]
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device=self.uk.device)  # noqa: E731
        self.cache = LatentCache(sum(used), self.PAGE, d.D_C, d.D_R, device=self.uk.device)
        self.batch = LatentBatch(table, ints(lens))
        self.whole = LatentBatch(table, ints(lens), ints([sum(lens[:b]) for b in range(len(lens) + 1)]))
        self.positions = ints(lens) - 1
        random = lambda *s: torch.randn(*s, generator=g, device=self.uk.device).bfloat16()  # noqa: E731
        self.cache.append(random(sum(lens), d.D_C), random(sum(lens), d.D_R), self.whole)
        self.q = torch.empty(len(lens), d.NH, d.D_C + d.D_R, dtype=torch.bfloat16, device=self.uk.device)

    def __call__(self, x):
        d = self.dims
        y = self.qkva(rms_norm(x, self.norm))
        q, latent, k_pe = y[:, :d.Q_OUT].unflatten(1, (d.NH, d.D_N + d.D_R)), y[:, d.Q_OUT:d.Q_OUT + d.D_C], y[:, d.Q_OUT + d.D_C:]
        self.cache.append(rms_norm(latent, self.kv_norm), self.rope(k_pe, self.positions), self.batch)
        self.q[..., :d.D_C] = torch.bmm(q[..., :d.D_N].transpose(0, 1), self.uk.transpose(1, 2)).transpose(0, 1)
        self.rope(q[..., d.D_N:], self.positions, out=self.q[..., d.D_C:])
        out = self.cache.attend(self.q, self.batch, self.scale)
        attn = torch.bmm(out.transpose(0, 1), self.uv.transpose(1, 2)).transpose(0, 1).reshape(len(self.lens), -1)
        return self.o(attn, residual=x)

    def plain(self, x):
        """(what __call__ returns, the largest sum of a score's terms) in FP32 over the dequantised weights and the
        cache as __call__ left it."""
        d = self.dims
        qkva, o = (dequantize_w4(*c, k, self.group) for c, k in zip(self.codes, (d.H, d.NH * d.D_V)))
        y = rms_norm(x, self.norm).float() @ qkva.T
        q = y[:, :d.Q_OUT].unflatten(1, (d.NH, d.D_N + d.D_R))
        angle = self.positions.double()[:, None] * self.rope.inv_freq
        cos, sin = angle.cos().float()[:, None] * self.rope.scale, angle.sin().float()[:, None] * self.rope.scale
        a, b = q[..., d.D_N::2], q[..., d.D_N + 1::2]
        q = torch.cat([torch.einsum("thn,hcn->thc", q[..., :d.D_N], self.uk.float()), a * cos - b * sin, b * cos + a * sin], -1)
        latents, keys = self.cache.read(self.whole, sum(self.lens))
        attn, spread, at = [], 0.0, 0
        for row, n in zip(q, self.lens):
            k = torch.cat([latents[at:at + n], keys[at:at + n]], 1).float()
            out = torch.softmax(row @ k.T * self.scale, 1) @ k[:, :d.D_C]
            spread = max(spread, (row.abs() @ k.abs().T * self.scale).max().item())
            attn.append(torch.einsum("hc,hvc->hv", out, self.uv.float()).flatten())
            at += n
        return (torch.stack(attn) @ o.T + x.float()).to(x.dtype), spread


class W4Layers:
    """The MoE layers (after their attention, or with it: `lens`, the sequences' tokens) and the head of a packed model,
    experts, projections and head in 4 bits."""

    def __init__(self, packed, dims: Dims, layers, group=128, zero_point=False, lens=None):
        self.dims, self.group = dims, group
        self.attention = [None if lens is None else W4Attention(packed, dims, l, lens, group, zero_point) for l in layers]
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
        for attention, norm, gate, experts in zip(self.attention, self.norms, self.gates, self.experts):
            if attention is not None:
                x = attention(x)
            h = rms_norm(x, norm)
            ids, weights = route_experts(h.float() @ gate.T, d.TOPK, n_forced=d.N_SHARED)
            x = experts(h, ids, weights, residual=x)
            residuals.append(x)
            routes.append((ids, weights))
        logits = self.head(rms_norm(x, self.final_norm), out_dtype=torch.float32)
        return logits.argmax(-1), logits, residuals, routes

    def plain(self, x, routes):
        """The residuals and logits of step(x) in FP32 over the dequantised weights, with step's routing (and cached latents)."""
        return self.plain_and_terms(x, routes)[:2]

    def plain_and_terms(self, x, routes):
        """plain(x, routes), and the largest sum of a score's terms in the attention (0 without it)."""
        d, residuals, spread = self.dims, [], 0.0
        for attention, norm, (w13, w2), (ids, weights) in zip(self.attention, self.norms, self.codes, routes):
            if attention is not None:
                x, terms = attention.plain(x)
                spread = max(spread, terms)
            h, out = rms_norm(x, norm).float(), x.float()
            for e in ids.unique().tolist():
                t, s = (ids == e).nonzero(as_tuple=True)
                part = lambda w: [None if v is None else v[e] for v in w]  # noqa: E731, B023
                gu = h[t] @ dequantize_w4(*part(w13), d.H, self.group).T
                y = (torch.nn.functional.silu(gu[:, 0::2]) * gu[:, 1::2]) @ dequantize_w4(*part(w2), d.I_MOE, self.group).T
                out.index_add_(0, t, y * weights[t, s][:, None])
            x = out.to(x.dtype)
            residuals.append(x)
        return residuals, rms_norm(x, self.final_norm).float() @ dequantize_w4(*self.head_codes, d.H, self.group).T, spread


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
    ap.add_argument("--context", type=int, default=0, help="tokens of the longest sequence: each layer's attention too")
    ap.add_argument("--std", type=float, default=0.02, help="spread of the synthetic weights")
    ap.add_argument("--dims", default=None, help="Dims fields as name=value,... (default: the real model's)")
    a = ap.parse_args(argv)
    from fleet.pack_weights import REAL_DIMS
    dims = REAL_DIMS if a.dims is None else Dims(**{k: int(v) for k, v in (f.split("=") for f in a.dims.split(","))})
    layers = range(1, a.layers + 1)
    packed = synthetic_packed(dims, layers=a.layers + 1, head=True, seed=0, device="cuda", std=a.std)
    # sequences from the whole context down to a tenth of it
    lens = None if a.context < 1 else [max(1, a.context - b * a.context * 9 // (10 * a.tokens)) for b in range(a.tokens)]
    model = W4Layers(packed, dims, layers, a.group, a.zero_point, lens)
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
        want, want_logits, spread = model.plain_and_terms(x, routes)
        out["residual_distance"] = [distance(r, p) for r, p in zip(residuals, want)]
        out["logits_distance"] = distance(logits, want_logits)
        if lens is not None:
            out["score_terms"] = spread
    print(out)
    return out


if __name__ == "__main__":
    main()
