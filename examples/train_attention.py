"""Trains one layer of temporal attention on a synthetic stream.

Every step takes a batch through the pipeline and the operators as a model does:
``DataPipeline.prepare`` gathers neighbours, masks and time encodings; ``embed``
looks up the learned rows of queries and neighbours; ``layer_norm`` and
``cross_attention`` turn them into one vector per query; a dot product scores
the batch's edges against its negatives; ``clip_grad_norm_`` bounds the
gradients; ``TemporalGraph.advance`` takes the events in.

    python examples/train_attention.py [--steps 200] [--dtype bf16]
"""
from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from tgengine_amd import DataPipeline, GatherSpec, NeighborSpec, RawBatch, TemporalGraph, ops  # noqa: E402


class TemporalAttention(torch.nn.Module):
    """One vector per query node from its own learned row and its neighbours' tokens
    (learned row, edge features, time encoding)."""

    def __init__(self, nodes: int, edge_dim: int, time_dim: int, dim: int = 64, heads: int = 2,
                 dtype: torch.dtype = torch.float32):
        super().__init__()
        self.heads, self.scale = heads, dim ** 0.5
        new = dict(device="cuda", dtype=dtype)
        self.table = torch.nn.Parameter(torch.randn(nodes, dim, **new) / dim)
        self.token = torch.nn.Linear(dim + edge_dim + time_dim, dim, **new)
        self.norm_w = torch.nn.Parameter(torch.ones(dim, **new))
        self.norm_b = torch.nn.Parameter(torch.zeros(dim, **new))
        self.query = torch.nn.Linear(dim, dim, **new)
        self.keys = torch.nn.Linear(dim, 2 * dim, **new)
        self.out = torch.nn.Linear(2 * dim, dim, **new)

    def forward(self, nodes, neighbors):
        b, k = neighbors.neighbor_ids.shape
        own = ops.embed(self.table, nodes, scale=self.scale)
        near = ops.embed(self.table, neighbors.neighbor_ids, scale=self.scale)
        tokens = torch.cat([near, neighbors.edge_feats.to(near.dtype), neighbors.time_enc.to(near.dtype)], -1)
        tokens = ops.layer_norm(self.token(tokens), self.norm_w, self.norm_b)
        q = self.query(own).view(b, 1, self.heads, -1)
        kv = self.keys(tokens).view(b, k, 2, self.heads, -1)  # read in place, side by side
        seen = ops.cross_attention(q, kv[:, :, 0], kv[:, :, 1], mask=neighbors.mask)
        return self.out(torch.cat([own, seen.reshape(b, -1)], -1))


def train(steps: int = 200, batch: int = 400, nodes: int = 2_000, edge_dim: int = 16, dtype: torch.dtype = torch.float32,
          seed: int = 0, log=print):
    """The loss of every step, as floats."""
    torch.manual_seed(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    graph = TemporalGraph(nodes, edge_feat_dim=edge_dim, device="cuda", buffer_size=16)
    pipe = DataPipeline(GatherSpec(neighbors=NeighborSpec(k=16), time_encoding=20), graph)
    model = TemporalAttention(nodes, edge_dim, 20, dtype=dtype)
    params = list(model.parameters())
    adam = torch.optim.AdamW(params, lr=3e-3)
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
        score = torch.cat([(hs * hd).sum(-1), -(hs * hn).sum(-1)]).float()
        loss = torch.nn.functional.softplus(-score).mean()
        adam.zero_grad(set_to_none=True)
        loss.backward()
        norm = ops.clip_grad_norm_(params, 1.0)
        adam.step()
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
    a = ap.parse_args()
    train(a.steps, dtype=torch.float32 if a.dtype == "f32" else torch.bfloat16)
