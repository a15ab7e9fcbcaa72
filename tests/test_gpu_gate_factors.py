"""sigmoid(gate) and 1 - sigmoid(gate) as the kernels form them, read from calls whose other factors are 0 and 1.

u = 2^-24.  The smaller of the two is e / (1 + e) with e = 2^(-|gate| / ln 2).  Its argument is off by 1.3 u |gate|
relatively, in e: the constant by 0.22 u and the product by u, times |gate|.  The instructions for the power and the
reciprocal are off by a unit in the last place, 2 u, the sum and the product by u: (1.3 |gate| + 6) u together.  The
larger as a reciprocal: u + 2 u, and e's error times e / (1 + e), below 2 u: 5 u.  As 1 less the smaller: u, and
the smaller's error times its share, which is largest at 0, 6 u: 7 u."""
import pytest
import torch

from tgengine_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _gates():
    g = torch.cat([torch.linspace(-87, 87, 200_001), torch.randn(200_000, generator=torch.Generator().manual_seed(0)) * 3,
                   torch.tensor([0.0, -0.0, 2.0 ** -30, -2.0 ** -30, 1.0, -1.0])])
    return g[g.abs() <= 87].cuda()


def _off(got, g, larger):
    want, size = torch.sigmoid(g.double()), g.double().abs()
    bound = torch.where(g < 0, 1.3 * size + 6, torch.full_like(size, larger)) * U
    assert bool(((got.double() - want).abs() <= 1.001 * bound * want).all())


def test_of_the_scan():
    g = _gates()
    one, zero = torch.ones_like(g), torch.zeros_like(g)
    keep = ops.gated_scan(zero[None, None], g[None, None], state=one[None])[1][0]
    take = ops.gated_scan(one[None, None], g[None, None], state=zero[None])[1][0]
    _off(keep, g, 5.0)
    _off(take, -g, 5.0)


@pytest.mark.parametrize("rows", [1, 3])
def test_of_the_residual_norm(rows):
    """sum = 0 + sigmoid(gate) 1, and the gradient of scale sums that factor: one row's is the factor itself.  The
    backward pass forms the sum again, so its factor has to be the forward one's, bit by bit."""
    g = _gates()
    g = g[:g.numel() // (96 * rows) * 96 * rows].view(-1, rows, 96)
    for gate in g[:: max(1, len(g) // 500)]:
        x, scale = torch.ones_like(gate), torch.ones(96, device="cuda").requires_grad_()
        s = ops.residual_norm(x, torch.zeros_like(x), gate=gate, scale=scale)[1]
        _off(s.detach(), gate, 7.0)
        for row in range(rows):
            only = torch.zeros_like(x)
            only[row] = 1.0
            back, = torch.autograd.grad(s, scale, only, retain_graph=True)
            assert torch.equal(back, s[row].detach())
