"""Gradients that reach a state through masked tokens are sums of as many terms: how gated_scan adds them up.

u = 2^-24.  A masked token adds its gradient to what comes from the right and leaves it whole (a = 1).  In f32, n of
them added one by one to a large value c lose up to n u c, and all of themselves where each is below u c.  Added up in
groups of 8 first, the groups lose 7 u of their own sums and then u c a group."""
import pytest
import torch

from tgengine_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F, B = torch.float32, torch.bfloat16
SHAPES = [(300, 512, 172), (5, 511, 3), (2, 3001, 2), (3, 520, 40), (4, 17, 9)]


def _grads(x, gate, mask, state, gout, glast):
    leaves = [t.detach().requires_grad_() for t in (x, gate, state)]
    y = ops.gated_scan(leaves[0], leaves[1], mask, leaves[2])
    return torch.autograd.grad(y, leaves, (gout, glast))


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("shape", SHAPES)
def test_small_terms_join_a_large_one(shape, dtype):
    """All tokens masked, the last state's gradient 2^24, every output's 1: sums of 8 ones and their multiples up to
    2^24 are numbers of f32, and so is every 2^24 + 8 k below 2^25.  The tokens past the last whole span, fewer than 8,
    come first: where their number is odd, one rounding is off by u (2^24 + 7), which is 1 and a little, and where
    pieces of a long row are joined all sums are whole again."""
    b, n, d = shape
    x, gate = (torch.randn(shape, device="cuda").to(dtype) for _ in range(2))
    mask = torch.zeros(b, n, device="cuda", dtype=torch.bool)
    state = torch.randn(b, d, device="cuda")
    dx, dgate, dstate = _grads(x, gate, mask, state, torch.ones(shape, device="cuda", dtype=dtype),
                               torch.full((b, d), 2.0 ** 24, device="cuda"))
    assert not dx.any() and not dgate.any()
    assert bool(((dstate.double() - (2.0 ** 24 + n)).abs() <= (1 if n % 2 else 0)).all())


@pytest.mark.parametrize("shape", SHAPES)
def test_long_masked_heads(shape):
    """Rows whose tokens are all masked but the last one, as those of nodes with one neighbour: dstate = a_n (dlast +
    dout_n) + the sum of the others, and against that sum of n terms in 64 bits an f32 sum in groups of 8 is off by at
    most (7 + n / 8 + 2) u times the absolute sum, a piece's joint adding two more; the factor a by (2 |gate| + 6) u."""
    b, n, d = shape
    g = torch.Generator(device="cuda").manual_seed(n)
    x, gate, gout = (torch.randn(shape, generator=g, device="cuda") for _ in range(3))
    state, glast = (torch.randn(b, d, generator=g, device="cuda") for _ in range(2))
    mask = torch.arange(n, device="cuda").expand(b, n) == n - 1
    got = _grads(x, gate, mask, state, gout, glast)[2].double()
    a, last = torch.sigmoid(gate[:, -1].double()), glast.double() + gout[:, -1].double()
    want = a * last + gout[:, :-1].double().sum(1)
    size = (a * last).abs() + gout[:, :-1].double().abs().sum(1)
    pieces = 64  # at most, for these shapes
    bound = (9 + n / 8 + 2 * pieces * (n > 1000)) * U * size + (2 * gate[:, -1].double().abs() + 8) * U * (a * last).abs()
    assert bool(((got - want).abs() <= 1.01 * bound).all())
