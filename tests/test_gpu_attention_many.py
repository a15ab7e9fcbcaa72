"""cross_attention over many batch rows: the launches' limits, and the walks of few rows over
several tiles of keys that only many problems make.  Rows of a large batch have the bits of
the same rows alone where no range is cut, and stay within the bounds of 64 bits."""
import pytest
import torch

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
