"""The operators together, as examples/train_attention.py runs them: on prepared batches
of a stream, against the same layer in torch operations, and trained."""
import importlib.util
from pathlib import Path

import pytest
import torch

from tgengine_amd import DataPipeline, GatherSpec, NeighborSpec, RawBatch, TemporalGraph, ops

pytestmark = pytest.mark.gpu

_spec = importlib.util.spec_from_file_location(
    "train_attention", Path(__file__).resolve().parent.parent / "examples" / "train_attention.py")
example = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(example)


class _Plain:
    """The operators of the layer in torch operations, 64 bits."""

    @staticmethod
    def embed(table, ids, scale=1.0):
        ok = (ids >= 0) & (ids.long() < table.shape[0])
        return torch.where(ok[..., None], table[torch.where(ok, ids.long(), 0)] * scale, 0.0)

    @staticmethod
    def layer_norm(x, w, b):
        return torch.nn.functional.layer_norm(x, (x.shape[-1],), w, b)

    @staticmethod
    def cross_attention(q, k, v, mask):
        s = torch.einsum("bihc,bjhc->bhij", q, k) * q.shape[-1] ** -0.5
        s = s.masked_fill(~mask[:, None, None, :], -1e300)
        p = torch.softmax(s, -1) * mask[:, None, None, :]
        return torch.einsum("bhij,bjhc->bihc", p, v)


def test_layer_and_gradients_on_prepared_batches(monkeypatch):
    """Outputs and every parameter's gradient on batches whose first queries have no
    neighbour at all.  The layer's products and sums are of at most 100 terms in 32 bits,
    a few deep, so 1e-4 of the largest value holds them with room."""
    torch.manual_seed(3)
    nodes, b, de = 150, 60, 8
    g = TemporalGraph(nodes, edge_feat_dim=de, device="cuda", buffer_size=12)
    pipe = DataPipeline(GatherSpec(neighbors=NeighborSpec(k=12), time_encoding=10), g)
    model = example.TemporalAttention(nodes, de, 10, dim=36, heads=2)
    for step in range(4):
        src, dst = (torch.randint(0, nodes, (b,), device="cuda") for _ in range(2))
        t = 500.0 + b * step + torch.arange(b, device="cuda", dtype=torch.float64)
        feat = torch.randn(b, de, device="cuda")
        pb = pipe.prepare(RawBatch(src, dst, t, feat, neg=dst))
        assert step == 0 or pb.src_neighbors.mask.any()
        got = model(src, pb.src_neighbors)
        dout = torch.randn_like(got)
        grads = torch.autograd.grad(got, list(model.parameters()), dout)
        with monkeypatch.context() as m:
            for name in ("embed", "layer_norm", "cross_attention"):
                m.setattr(ops, name, getattr(_Plain, name))
            wide = example.TemporalAttention(nodes, de, 10, dim=36, heads=2, dtype=torch.float64)
            wide.load_state_dict(model.state_dict())
            want = wide(src, pb.src_neighbors)
            wgrads = torch.autograd.grad(want, list(wide.parameters()), dout.double())
        for x, y in zip((got, *grads), (want, *wgrads)):
            assert bool(((x.double() - y).abs() <= 1e-4 * y.abs().max()).all())
        g.advance(src, dst, t, feat)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_learns(dtype):
    losses = example.train(steps=120, dtype=dtype, log=None)
    assert all(x == x for x in losses)
    assert sum(losses[-20:]) / 20 < 0.9 * losses[0]
