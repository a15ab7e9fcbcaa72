"""Tensors whose signs torch keeps apart from their memory, as those of the imaginary part of a conjugate: the
operators take the values, not the memory."""
import pytest
import torch

from tgengine_amd import ops

pytestmark = pytest.mark.gpu


def _parts(t):
    """t as the imaginary part of a conjugate: every second number of its memory."""
    out = torch.complex(torch.full_like(t, 7.0), -t).conj().imag
    assert out.is_neg() and torch.equal(out, t)
    return out


def _whole(t):
    """t over memory that holds -t, one value after the other."""
    out = torch._neg_view(-t)
    assert out.is_neg() and out.is_contiguous() and torch.equal(out, t)
    return out


def _r(*shape):
    return torch.randn(*shape, device="cuda")


CALLS = {
    "embed": (lambda t: ops.embed(t, torch.tensor([1, 0, -1, 2], device="cuda")), [(3, 1)]),
    "layer_norm": (lambda x, w, b: ops.layer_norm(x, w, b), [(5, 1), (1,), (1,)]),
    "cross_attention": (lambda q, k, v: ops.cross_attention(q, k, v, scale=1.0), [(2, 3, 2, 1), (2, 4, 2, 1), (2, 4, 2, 1)]),
    "gated_scan": (lambda x, g, s: ops.gated_scan(x, g, state=s), [(1, 3, 1), (1, 3, 1), (1, 1)]),
    "residual_norm": (lambda x, r, w, b, g, s, p: ops.residual_norm(x, r, w, b, gate=g, scale=s, post_weight=p, eps=0.5),
                      [(3, 1), (3, 1), (1,), (1,), (3, 1), (1,), (1,)]),
}


@pytest.mark.parametrize("turned", [_parts, _whole])
@pytest.mark.parametrize("width", [1, 6])
@pytest.mark.parametrize("name", CALLS)
def test_inputs_and_gradients(name, width, turned):
    call, shapes = CALLS[name]
    args = [_r(*s[:-1], s[-1] * width) for s in shapes]

    def run(args, turn):
        leaves = [a.detach().requires_grad_() for a in args]
        y = call(*(turned(a) if turn == "inputs" else a for a in leaves))
        y = y if isinstance(y, tuple) else (y,)
        with torch.no_grad():
            again = call(*(turned(a) if turn == "inputs" else a for a in args))
        g = [torch.arange(t.numel(), device="cuda").view(t.shape) * 0.5 - 1.25 for t in y]
        g = [turned(t) if turn == "gradients" else t for t in g]
        again = again if isinstance(again, tuple) else (again,)
        return [*y, *again, *torch.autograd.grad(y, leaves, g)]

    want = run(args, None)
    for turn in ("inputs", "gradients"):
        if turn == "gradients" and turned is _parts and width > 1:
            continue  # a copy either way
        for a, b in zip(run(args, turn), want):
            assert torch.equal(a, b), turn


@pytest.mark.parametrize("turned", [_parts, _whole])
def test_steps_and_clipping(turned):
    p, g = _r(1), _r(1)
    wide = _r(300)

    def step(g, h):
        ps = [p.clone(), wide.clone()]
        state = [[torch.zeros_like(x) for x in ps] for _ in range(2)]
        ops.adamw_(ps, [g, h], *state, [torch.zeros((), dtype=torch.int64, device="cuda") for _ in ps], lr=0.1)
        return [*ps, *state[0], *state[1]]

    for h in (wide * 0.1, turned(wide * 0.1).contiguous()):
        for a, b in zip(step(turned(g), h), step(g, wide * 0.1)):
            assert torch.equal(a, b)
    bad = turned(p.clone())
    for which in range(3):
        args = [[p.clone()], [torch.zeros_like(p)], [torch.zeros_like(p)]]
        args[which] = [bad]
        with pytest.raises(ValueError, match="turned signs"):
            ops.adamw_(args[0], [g], args[1], args[2], [torch.zeros((), dtype=torch.int64, device="cuda")])
    # scaled in place, and into tensors apart
    one, want = turned(g.clone()), g.clone()
    assert torch.equal(ops.clip_grad_norm_([one], 0.01), ops.clip_grad_norm_([want], 0.01)) and torch.equal(one, want)
    to, there = torch.empty_like(g), torch.empty_like(g)
    ops.clip_grad_norm_([turned(g)], 0.01, [to])
    ops.clip_grad_norm_([g], 0.01, [there])
    assert torch.equal(to, there)
    with pytest.raises(ValueError, match="turned signs"):
        ops.clip_grad_norm_([g], 0.01, [turned(g.clone())])
