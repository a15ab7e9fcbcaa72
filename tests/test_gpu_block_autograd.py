"""What the operators around attention refuse of torch's ways to follow a call, and what
autograd may do with them: forward-mode derivatives, traces and transforms; inputs changed
behind a saved graph; graphs kept and freed; inference mode."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from tgengine_amd import ops

pytestmark = pytest.mark.gpu


def _r(*shape):
    return torch.randn(*shape, device="cuda")


def _step(p, g):
    state = [torch.zeros_like(p), torch.zeros_like(p), torch.zeros((), dtype=torch.int64, device="cuda")]
    ops.adamw_([p], [g], *([s] for s in state))
    return p


CALLS = {
    "gated_scan": (lambda x, g, s: ops.gated_scan(x, g, state=s), [(2, 11, 8), (2, 11, 8), (2, 8)]),
    "residual_norm": (lambda x, r, w, b, g, s, p: ops.residual_norm(x, r, w, b, gate=g, scale=s, post_weight=p),
                      [(4, 8), (4, 8), (8,), (8,), (4, 8), (8,), (8,)]),
    "adamw_": (_step, [(4, 8), (4, 8)]),
}
DIFFERENTIABLE = ["gated_scan", "residual_norm"]


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode(name, grad):
    call, shapes = CALLS[name]
    for i in range(len(shapes)):
        args = [_r(*s) for s in shapes]
        if grad and name in DIFFERENTIABLE:
            args[i].requires_grad_()
        with fwd.dual_level():
            args[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(*args)
    with fwd.dual_level():  # no tangent: nothing to lose
        call(*[_r(*s) for s in shapes])


@pytest.mark.parametrize("name", CALLS)
def test_traces(name):
    call, shapes = CALLS[name]
    args = tuple(_r(*s) for s in shapes)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(call, args)
    call(*args)  # the next call is as before


@pytest.mark.parametrize("name", DIFFERENTIABLE)
def test_function_transforms(name):
    call, shapes = CALLS[name]
    args = tuple(_r(*s) for s in shapes)
    with pytest.raises(RuntimeError):
        torch.func.jvp(call, args, tuple(torch.ones_like(a) for a in args))


@pytest.mark.parametrize("name", DIFFERENTIABLE)
def test_graphs_kept_and_freed(name):
    """Twice through a kept graph: the same bits; through a freed one, or with an input changed: refused."""
    call, shapes = CALLS[name]
    args = [_r(*s).requires_grad_() for s in shapes]
    y = call(*args)
    g = [torch.ones_like(t) for t in y]
    one = torch.autograd.grad(y, args, g, retain_graph=True)
    two = torch.autograd.grad(y, args, g)
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, args, g)
    y = call(*args)
    with torch.no_grad():
        args[1].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(y, args, g)


@pytest.mark.parametrize("name", DIFFERENTIABLE)
def test_inference_mode(name):
    call, shapes = CALLS[name]
    args = [_r(*s).requires_grad_() for s in shapes]
    want = call(*args)
    with torch.inference_mode():
        got = call(*args)
    assert all(torch.equal(a, b) and not a.requires_grad for a, b in zip(got, want))


def test_accumulated_gradients():
    """Backward twice into .grad, and x and residual apart although one tensor was computed for both."""
    x, r, w = _r(6, 8).requires_grad_(), _r(6, 8).requires_grad_(), _r(8).requires_grad_()
    for _ in range(2):
        y, s = ops.residual_norm(x, r, w)
        (y.sum() + s.square().sum()).backward()
    one = torch.autograd.grad(sum(t.sum() if i == 0 else t.square().sum() for i, t in enumerate(ops.residual_norm(x, r, w))),
                              (x, r, w))
    for p, g in zip((x, r, w), one):
        assert torch.equal(p.grad, g * 2)
    x.grad.zero_()
    assert r.grad.any()


def test_unused_outputs_and_inputs():
    x, g = _r(2, 9, 8).requires_grad_(), _r(2, 9, 8)
    out, last = ops.gated_scan(x, g)
    assert out.requires_grad and last.requires_grad
    last.sum().backward()
    assert x.grad.shape == x.shape
    y, s = ops.residual_norm(_r(4, 8), _r(4, 8), _r(8))
    assert not y.requires_grad and not s.requires_grad
