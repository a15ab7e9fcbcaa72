"""The operators together, as examples/train_scan.py runs them: on prepared batches of a
stream, against the same model in torch operations, stepped, and captured as a whole."""
import importlib.util
from pathlib import Path

import pytest
import torch

from tgengine_amd import DataPipeline, GatherSpec, NeighborSpec, RawBatch, TemporalGraph, ops

pytestmark = pytest.mark.gpu

_spec = importlib.util.spec_from_file_location(
    "train_scan", Path(__file__).resolve().parent.parent / "examples" / "train_scan.py")
example = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(example)


class _Plain:
    """The operators of the model in torch operations, 64 bits."""

    @staticmethod
    def embed(table, ids, scale=1.0):
        ok = (ids >= 0) & (ids.long() < table.shape[0])
        return torch.where(ok[..., None], table[torch.where(ok, ids.long(), 0)] * scale, 0.0)

    @staticmethod
    def gated_scan(x, gate, mask=None, state=None):
        h = torch.zeros_like(x[:, 0]) if state is None else state
        out = []
        for t in range(x.shape[1]):
            f = torch.sigmoid(gate[:, t])
            h = torch.where(mask[:, t, None], f * h + (1 - f) * x[:, t], h)
            out.append(h)
        return torch.stack(out, 1), h

    @staticmethod
    def residual_norm(x, residual, weight, bias=None, *, gate=None, scale=None, post_weight=None, center=True, eps=1e-5):
        def norm(v):
            v = v - v.mean(-1, keepdim=True) if center else v
            return v * (v.square().mean(-1, keepdim=True) + eps).rsqrt()

        n = x if post_weight is None else norm(x) * post_weight
        n = n if gate is None else n * torch.sigmoid(gate)
        s = residual + (n if scale is None else n * scale)
        y = norm(s) * weight
        return (y if bias is None else y + bias), s


def _batches(steps, nodes=150, b=60, de=8, seed=3):
    torch.manual_seed(seed)
    g = TemporalGraph(nodes, edge_feat_dim=de, device="cuda", buffer_size=12)
    pipe = DataPipeline(GatherSpec(neighbors=NeighborSpec(k=12), time_encoding=10), g)
    for step in range(steps):
        src, dst = (torch.randint(0, nodes, (b,), device="cuda") for _ in range(2))
        t = 500.0 + b * step + torch.arange(b, device="cuda", dtype=torch.float64)
        feat = torch.randn(b, de, device="cuda")
        yield src, pipe.prepare(RawBatch(src, dst, t, feat, neg=dst)).src_neighbors
        g.advance(src, dst, t, feat)


def test_model_and_gradients_on_prepared_batches(monkeypatch):
    """Outputs and every parameter's gradient on batches whose first queries have no neighbour
    at all, whose tables follow each other through steps of the optimizer.  The model's products
    and sums are of at most 100 terms in 32 bits, some deep, and its norms divide by
    deviations down to a tenth, so 1e-4 of the largest value holds them with room."""
    model = example.TemporalScan(150, 8, 10, dim=36)
    adam = ops.AdamW(model.parameters(), lr=1e-2, bits=8)
    for src, near in _batches(4):
        got = model(src, near)
        dout = torch.randn_like(got)
        params = list(model.parameters())
        grads = torch.autograd.grad(got, params, dout)
        with monkeypatch.context() as m:
            for name in ("embed", "gated_scan", "residual_norm"):
                m.setattr(ops, name, getattr(_Plain, name))
            wide = example.TemporalScan(150, 8, 10, dim=36, dtype=torch.float64)
            wide.load_state_dict(model.state_dict())
            want = wide(src, near)
            wgrads = torch.autograd.grad(want, list(wide.parameters()), dout.double())
        for x, y in zip((got, *grads), (want, *wgrads)):
            assert bool(((x.double() - y).abs() <= 1e-4 * y.abs().max()).all())
        for p, g in zip(params, grads):
            p.grad = g
        norm = ops.clip_grad_norm_(params, float("inf"))
        want = torch.cat([g.double().reshape(-1) for g in grads]).norm()
        assert abs(float(norm) - float(want)) <= 1e-5 * float(want)
        adam.step(grad_norm=norm, max_norm=1.0)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_runs(dtype, bits):
    losses = example.train(steps=40, dtype=dtype, bits=bits, log=None)
    assert len(losses) == 40 and all(0.0 < x < 10.0 for x in losses)
    again = example.train(steps=40, dtype=dtype, bits=bits, log=None)
    assert losses == again  # the same bits


def test_step_in_a_graph():
    """Forward, backward, norm and step captured once and replayed on new batches: the eager step's bits."""
    def new():
        torch.manual_seed(5)
        model = example.TemporalScan(150, 8, 10, dim=36)
        return model, ops.AdamW(model.parameters(), lr=1e-2, bits=8)

    def step(model, adam, src, near, dout):
        params = list(model.parameters())
        for p, g in zip(params, torch.autograd.grad(model(src, near), params, dout)):
            p.grad = g
        adam.step(grad_norm=ops.clip_grad_norm_(params, float("inf")), max_norm=1.0)

    batches = list(_batches(6))
    douts = [torch.randn(60, 36, device="cuda") for _ in batches]
    want, wadam = new()
    for (src, near), dout in zip(batches, douts):
        step(want, wadam, src, near, dout)
    model, adam = new()
    src, near, dout = batches[0][0].clone(), batches[0][1], douts[0].clone()
    names = ("neighbor_ids", "edge_feats", "time_enc", "mask")
    for n in names:
        setattr(near, n, getattr(near, n).clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(model, adam, src, near, dout)  # the averages' first step
    torch.cuda.current_stream().wait_stream(side)
    for p in model.parameters():
        p.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(model, adam, src, near, dout)
    for (s, nb), d in zip(batches[1:], douts[1:]):
        src.copy_(s)
        dout.copy_(d)
        for n in names:
            getattr(near, n).copy_(getattr(nb, n))
        graph.replay()
        torch.cuda.synchronize()
    for p, q in zip(model.parameters(), want.parameters()):
        assert torch.equal(p, q)
