"""clip_grad_norm_ against norms in 64 bits.

A thread sums at most 2^16 squares in 32 bits before the sums are joined in 64: the norm
is off by at most half of 2^16 u relatively, far less for these sizes; 2^10 u holds for
sums of up to 2,048 squares a thread.  A scaled value is two roundings off the exact
product (u each, and r of its type)."""
import math

import pytest
import torch

from tgengine_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _grads(sizes, dtypes, seed=0, scale=0.1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(n, generator=g, device="cuda") * scale).to(t) for n, t in zip(sizes, dtypes)]


def _check(grads, max_norm, out=None):
    before = [g.clone() for g in grads]
    exact = math.sqrt(sum(float(g.double().square().sum()) for g in before))
    norm = ops.clip_grad_norm_(grads, max_norm, out=out)
    assert norm.shape == () and norm.dtype == torch.float32
    assert abs(float(norm) - exact) <= 2 ** 10 * U * exact
    by = min(1.0, max_norm / (exact + 1e-6))
    for g, b, o in zip(grads, before, grads if out is None else out):
        r = U if o.dtype == torch.float32 else 2.0 ** -8
        want = b.double() * by
        assert bool(((o.double() - want).abs() <= want.abs() * (r + 2 ** 11 * U) + 1e-45).all())
        if by == 1.0 and o.dtype == b.dtype:
            assert torch.equal(o, b)
        if out is not None:
            assert torch.equal(g, b)
    return norm


F, B = torch.float32, torch.bfloat16


@pytest.mark.parametrize("sizes,dtypes", [
    ((1,), (F,)), ((7,), (B,)), ((20_000, 116, 1, 20_001), (F, F, F, F)), ((300_001, 5, 0, 77), (B, F, B, B)),
    (tuple(range(1, 60)), (F, B) * 30), ((3_000_003, 8_191, 8_193), (F, F, B)), ((64,) * 300, (F,) * 300),
    ((20_000_001, 3), (B, F)), ((0, 0, 5), (F, B, F))])
def test_clip(sizes, dtypes):
    for max_norm in (0.05, 1e6):
        _check(_grads(sizes, dtypes), max_norm)
        grads = _grads(sizes, dtypes, 1)
        _check(grads, max_norm, out=[torch.full_like(g, float("nan")) for g in grads])
    grads = _grads(sizes, dtypes, 2)
    _check(grads, 0.05, out=[torch.empty_like(g, dtype=F) for g in grads])
    _check(grads, 0.05, out=[torch.empty_like(g, dtype=B) for g in grads])


def test_shifted_and_shaped():
    base = _grads((50_003, 4_000), (B, F), 3)
    grads = [base[0][1:], base[1].view(40, 100)[3:]]
    _check(grads, 0.3, out=[torch.empty(50_005, device="cuda", dtype=B)[3:], torch.empty(37, 100, device="cuda")])
    _check(grads, 0.3)


def test_parameters():
    p = [torch.nn.Parameter(torch.randn(30, 4, device="cuda")), torch.nn.Parameter(torch.randn(9, device="cuda")),
         torch.nn.Parameter(torch.randn(5, device="cuda"))]
    (p[0].sum() * 3 + p[1].square().sum()).backward()
    want = torch.linalg.vector_norm(torch.cat([p[0].grad.reshape(-1), p[1].grad]).double())
    norm = ops.clip_grad_norm_(p, 1.0)
    assert abs(float(norm) - float(want)) <= 2 ** 10 * U * float(want) and p[2].grad is None
    after = torch.cat([p[0].grad.reshape(-1), p[1].grad]).double().norm()
    assert abs(float(after) - 1.0) < 1e-5


@pytest.mark.parametrize("x", [float("nan"), float("inf")])
def test_not_finite(x):
    """As the formula says: a NaN norm makes everything NaN, an infinite one zeros (and NaN of the infinity)."""
    grads = _grads((100, 50), (F, B), 4)
    grads[0][7] = x
    norm = ops.clip_grad_norm_(grads, 1.0)
    if math.isnan(x):
        assert norm.isnan() and all(g.isnan().all() for g in grads)
    else:
        assert norm.isinf() and grads[0][7].isnan() and not grads[1].any()


def test_zero_gradients():
    grads = [torch.zeros(100, device="cuda"), torch.zeros(3, device="cuda", dtype=B)]
    assert float(ops.clip_grad_norm_(grads, 1.0)) == 0 and not grads[0].any() and not grads[1].any()
    assert float(ops.clip_grad_norm_([torch.empty(0, device="cuda")], 1.0)) == 0


def test_autograd_sees_the_write():
    g = torch.randn(10, device="cuda")
    x = torch.randn(10, device="cuda", requires_grad=True)
    y = (x * g).sum()
    ops.clip_grad_norm_([g], 1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_graph_replays():
    grads = _grads((5_000, 700), (F, B), 5)
    out = [torch.empty_like(g) for g in grads]
    ops.clip_grad_norm_(grads, 0.5, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ops.clip_grad_norm_(grads, 0.5, out=out)
    for n in range(3):
        for g, x in zip(grads, _grads((5_000, 700), (F, B), 30 + n)):
            g.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        other = [torch.empty_like(g) for g in grads]
        assert torch.equal(ops.clip_grad_norm_(grads, 0.5, out=other), norm)
        assert all(torch.equal(a, b) for a, b in zip(out, other)), n


def test_refusals():
    g = torch.randn(4, 6, device="cuda")
    C = ops.clip_grad_norm_
    for args, kw, text in ((([],), {}, "no gradients"), (([g.t()],), {}, "contiguous"), (([g.half()],), {}, "float32 or bfloat16"),
                           (([g],), {"out": [g[0]]}, "shapes"), (([g],), {"out": [g, g]}, "one tensor per gradient"),
                           (([g],), {"out": [g.cpu()]}, "device")):
        with pytest.raises(ValueError, match=text):
            C(*args, 1.0, **kw)
    with pytest.raises(RuntimeError, match="on the GPU"):
        C([g.cpu()], 1.0)


def test_overlaps():
    """What would be written in no order is refused; gradients that are only read may be shared."""
    a, b = torch.randn(300, device="cuda"), torch.randn(300, device="cuda")
    keep = [a.clone(), b.clone()]
    tied = torch.nn.Parameter(torch.randn(40, device="cuda"))
    tied.grad = torch.randn(40, device="cuda")
    for grads, kw in (([a, b, a], {}), ([tied, torch.nn.Parameter(b), tied], {}), ([a, b], {"out": [b, a]}),
                      ([a, b], {"out": [keep[0], keep[0]]}), ([a[:200], a[199:]], {}), ([a[:200]], {"out": [a[50:250]]})):
        with pytest.raises(ValueError, match="overlap"):
            ops.clip_grad_norm_(grads, 1.0, **kw)
    assert torch.equal(a, keep[0]) and torch.equal(b, keep[1])
    _check([a, a], 1.0, out=[torch.empty_like(a), torch.empty_like(a)])
    _check([a[:200], a[200:], b], 1.0)


def test_leaves_are_parameters():
    """A plain leaf that requires a gradient is clipped by its gradient, as a Parameter is; no weight is scaled."""
    w, b, rest = (torch.randn(n, device="cuda", requires_grad=True) for n in (50, 7, 3))
    before = [x.detach().clone() for x in (w, b, rest)]
    ((w * 3).sum() + b.square().sum()).backward()
    want = torch.cat([w.grad, b.grad]).double().norm()
    norm = ops.clip_grad_norm_([w, b, rest], 1.0)
    assert abs(float(norm) - float(want)) <= 2 ** 10 * U * float(want) and rest.grad is None
    assert abs(float(torch.cat([w.grad, b.grad]).double().norm()) - 1.0) < 1e-5
    assert all(torch.equal(x, y) for x, y in zip((w, b, rest), before))
    with pytest.raises(ValueError, match="no gradients"):
        ops.clip_grad_norm_(rest, 1.0)
    g = torch.randn(7, device="cuda")
    with pytest.raises(ValueError, match="must not require a gradient"):
        ops.clip_grad_norm_([g], 1.0, out=[b])
    assert torch.equal(b, before[1])
    with torch.no_grad():  # as torch's own writes to a leaf
        ops.clip_grad_norm_([g], 1e6, out=[b])
    assert torch.equal(b, g)


@pytest.mark.parametrize("scale", [1e30, 1e19, 1e-30])
def test_squares_beyond_32_bits(scale):
    """Gradients whose squares pass what 32 bits hold, and whose norm does not."""
    _check(_grads((5_000, 3, 40_001), (F, B, F), 7, scale), 1.0)
    _check(_grads((200_003, 9), (B, F), 8, scale), scale * 10)
