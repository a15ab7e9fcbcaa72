"""cross_attention over many batch rows: the launches' limits, and the walks of few rows over
several tiles of keys that only many problems make.  Rows of a large batch have the bits of
the same rows alone where no range is cut, and stay within the bounds of 64 bits."""
import pytest
import torch

from test_gpu_attention import _exact, _inputs, _mask
from tgengine_amd import ops

pytestmark = pytest.mark.gpu


def _run(q, k, v, g, mask=None):
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    o = ops.cross_attention(*leaves, mask=mask)
    return (o.detach(), *torch.autograd.grad(o, leaves, g))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_8_600_000_problems(dtype):
    """More problems than 2^32 threads of 512 a workgroup, which no kernel here takes for 5 rows."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    b, lq, lk, h, d = 4_300_000, 5, 3, 2, 8
    q, k, v, g = (torch.randn(b, n, h, d, generator=gen, device="cuda", dtype=dtype) for n in (lq, lk, lk, lq))
    got = _run(q, k, v, g)
    for rows in (slice(0, 50), slice(b - 50, b)):
        want = _run(*(x[rows].contiguous() for x in (q, k, v, g)))
        assert all(torch.equal(x[rows], y) for x, y in zip(got, want))
    assert all(bool(torch.isfinite(x.sum(dtype=torch.float32))) for x in got)


def _bounds(q, k, v, g, mask, got):
    ref = _exact(q, k, v, g, mask, q.shape[-1] ** -0.5)
    for name, x in zip(("out", "dq", "dk", "dv"), got):
        y, e = ref[name]
        off = (x.double() - y).abs()
        assert bool((off <= e).all()), f"{name}: {float((off / e).max()):.3g} of the bound"


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lq,h,kv,d", [(1, 2, 2, 20), (1, 8, 2, 33), (2, 2, 1, 86), (1, 1, 1, 172)])
@pytest.mark.parametrize("lk,mask", [(65, "recent"), (130, "holes"), (200, "prefix")])
def test_one_wave_walks_several_tiles(lk, mask, lq, h, kv, d, dtype):
    """4,096 problems or more of at most 4 rows, not a multiple of the 4 waves of a workgroup: a wave takes a
    problem's tiles of 64 keys one after the other."""
    b = 4_099 // kv + 1 - (4_099 // kv) % 2  # an odd number of batch rows
    q, k, v, g = _inputs(b, lq, lk, h, kv, d, dtype, seed=lk)
    m = _mask(mask, b, lk, seed=lk + 1)
    _bounds(q, k, v, g, m, _run(q, k, v, g, m))


@pytest.mark.parametrize("mask", ["holes", None])
@pytest.mark.parametrize("b,lq,lk,h,kv,d", [(16, 300, 1_100, 4, 4, 24), (8, 260, 1_500, 4, 2, 100), (40, 70, 1_030, 4, 4, 140)])
def test_kept_scores_of_long_keys(b, lq, lk, h, kv, d, mask):
    """f32 with more than 1,024 keys and 128 row tiles or more: dq from score gradients that were kept."""
    q, k, v, g = _inputs(b, lq, lk, h, kv, d, "f32", seed=3)
    m = _mask(mask, b, lk, seed=4)
    _bounds(q, k, v, g, m, _run(q, k, v, g, m))
