"""Trains a recurrent model of temporal neighbourhoods on a synthetic stream.

Two blocks walk every query's neighbours from the oldest to the newest:
``gated_scan`` carries a state along the tokens that ``DataPipeline.prepare``
masked, and ``residual_norm`` adds what a block gives to what runs past it and
norms the sum for the next one.  ``clip_grad_norm_`` takes the gradients' norm, and
``AdamW`` clips them by it as it steps, with 8-bit averages for the node table.

    python examples/train_scan.py [--steps 200] [--dtype bf16] [--bits 8]
"""
from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from tgengine_amd import DataPipeline, GatherSpec, NeighborSpec, RawBatch, TemporalGraph, ops  # noqa: E402


class TemporalScan(torch.nn.Module):
    """One vector per query node from its own learned row and the states that its
    neighbours' tokens (learned row, edge features, time encoding) leave."""

    def __init__(self, nodes: int, edge_dim: int, time_dim: int, dim: int = 64, dtype: torch.dtype = torch.float32):
        super().__init__()
        self.scale = dim ** 0.5
        new = dict(device="cuda", dtype=dtype)
        self.table = torch.nn.Parameter(torch.randn(nodes, dim, **new) / dim)
        self.token = torch.nn.Linear(dim + edge_dim + time_dim, dim, **new)
        self.mix = torch.nn.ModuleList(torch.nn.Linear(dim, 2 * dim, **new) for _ in range(2))
        self.out = torch.nn.ModuleList(torch.nn.Linear(dim, dim, **new) for _ in range(2))
        self.gate = torch.nn.Linear(dim, dim, **new)
        self.norm = torch.nn.ParameterList(torch.ones(dim, **new) for _ in range(3))
        self.bias = torch.nn.Parameter(torch.zeros(dim, **new))
        self.step = torch.nn.Parameter(torch.full((dim,), 0.5, **new))

    def scan(self, i: int, tokens, mask):
        x, gate = self.mix[i](tokens).unflatten(-1, (2, -1)).unbind(-2)  # read in place, side by side
        return ops.gated_scan(x, gate, mask=mask)

    def forward(self, nodes, neighbors):
        own = ops.embed(self.table, nodes, scale=self.scale)
        near = ops.embed(self.table, neighbors.neighbor_ids, scale=self.scale)
        tokens = torch.cat([near, neighbors.edge_feats.to(near.dtype), neighbors.time_enc.to(near.dtype)], -1)
        tokens = self.token(tokens)
        states, _ = self.scan(0, tokens, neighbors.mask)
        tokens, _ = ops.residual_norm(self.out[0](states), tokens, self.norm[0], self.bias, scale=self.step)
        _, last = self.scan(1, tokens, neighbors.mask)
        seen = self.out[1](last.to(own.dtype))
        y, _ = ops.residual_norm(seen, own, self.norm[1], gate=self.gate(own), post_weight=self.norm[2], center=False)
        return y


def train(steps: int = 200, batch: int = 400, nodes: int = 2_000, edge_dim: int = 16, dtype: torch.dtype = torch.float32,
          bits: int = 8, seed: int = 0, log=print):
    """The loss of every step, as floats."""
    torch.manual_seed(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    graph = TemporalGraph(nodes, edge_feat_dim=edge_dim, device="cuda", buffer_size=16)
    pipe = DataPipeline(GatherSpec(neighbors=NeighborSpec(k=16), time_encoding=20), graph)
    model = TemporalScan(nodes, edge_dim, 20, dtype=dtype)
    params = list(model.parameters())
    adam = ops.AdamW(params, lr=3e-3, bits=bits)
    losses, t0 = [], 2.0 * batch
    began = time.perf_counter()
    for step in range(steps):
        # sources meet destinations of their own residue class: something to learn
        src = torch.randint(0, nodes, (batch,), generator=gen, device="cuda")
        dst = (src + 7 * torch.randint(0, nodes // 7, (batch,), generator=gen, device="cuda")) % nodes
        neg = torch.randint(0, nodes, (batch,), generator=gen, device="cuda")
        at = t0 + torch.arange(batch, device="cuda", dtype=torch.float64)
        t0 += batch
        feat = torch.randn(batch, edge_dim, generator=gen, device="cuda")
        pb = pipe.prepare(RawBatch(src, dst, at, feat, neg=neg))
        hs, hd, hn = (model(n, nb) for n, nb in ((src, pb.src_neighbors), (dst, pb.dst_neighbors),
                                                 (neg, pb.neg_neighbors)))
        score = torch.cat([(hs * hd).mean(-1), -(hs * hn).mean(-1)]).float()
        loss = torch.nn.functional.softplus(-score).mean()
        adam.zero_grad(set_to_none=True)
        loss.backward()
        norm = ops.clip_grad_norm_(params, float("inf"))  # the norm; the step scales by it
        adam.step(grad_norm=norm, max_norm=1.0)
        graph.advance(src, dst, at, feat)
        losses.append(loss.detach())
        if log and (step % 50 == 0 or step == steps - 1):
            log(f"step {step}: loss {float(loss.detach()):.4f}, gradient norm {float(norm):.3f}")
    torch.cuda.synchronize()
    if log:
        log(f"{steps} steps of {batch} events, {(time.perf_counter() - began) / steps * 1e3:.2f} ms each")
    return [float(x) for x in losses]


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--dtype", choices=("f32", "bf16"), default="f32")
    ap.add_argument("--bits", type=int, choices=(8, 32), default=8)
    a = ap.parse_args()
    train(a.steps, dtype=torch.float32 if a.dtype == "f32" else torch.bfloat16, bits=a.bits)
