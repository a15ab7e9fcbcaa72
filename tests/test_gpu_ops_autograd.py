"""What the operators refuse of torch's ways to follow a call: forward-mode derivatives, which
would come out as zeros, and traces, which would record outputs that nothing writes."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from tgengine_amd import ops

pytestmark = pytest.mark.gpu


def _r(*shape):
    return torch.randn(*shape, device="cuda")


IDS = [3, 0, -1]
CALLS = {
    "embed": (lambda t: ops.embed(t, torch.tensor(IDS, device="cuda")), [(5, 8)]),
    "layer_norm": (lambda x, w, b: ops.layer_norm(x, w, b), [(4, 8), (8,), (8,)]),
    "cross_attention": (lambda q, k, v: ops.cross_attention(q, k, v), [(2, 3, 2, 8), (2, 5, 2, 8), (2, 5, 2, 8)]),
    "clip_grad_norm_": (lambda g, h: ops.clip_grad_norm_([g, h], 1.0), [(4, 8), (3,)]),
}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode(name, grad):
    call, shapes = CALLS[name]
    for i in range(len(shapes)):
        args = [_r(*s) for s in shapes]
        if grad and name != "clip_grad_norm_":
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


@pytest.mark.parametrize("name", ["layer_norm", "cross_attention", "embed"])
def test_function_transforms(name):
    """torch.func's tensors have no memory to launch on."""
    call, shapes = CALLS[name]
    args = tuple(_r(*s) for s in shapes)
    with pytest.raises(RuntimeError):
        torch.func.jvp(call, args, tuple(torch.ones_like(a) for a in args))
