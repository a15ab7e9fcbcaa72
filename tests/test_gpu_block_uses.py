"""The operators around attention under what torch puts around a model: saved tensors moved away, recomputation, halves of
a projection of any number of dimensions, schedulers, copies of the optimizer, hooks around its steps."""
import copy
import io

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from tgengine_amd import ops

pytestmark = pytest.mark.gpu
F, B = torch.float32, torch.bfloat16


def _r(*shape, dtype=F):
    return torch.randn(*shape, device="cuda").to(dtype)


def _block(tokens, w, mask, norm):
    x, gate = (tokens @ w).unflatten(-1, (2, -1)).unbind(-2)
    h, last = ops.gated_scan(x, gate, mask)
    y, s = ops.residual_norm(h, tokens, norm, gate=gate, scale=norm, post_weight=norm, center=False)
    return y, s, last


def _leaves(dtype):
    torch.manual_seed(0)
    return [_r(5, 37, 24, dtype=dtype).requires_grad_(), (_r(24, 48) * 0.2).to(dtype).requires_grad_(),
            torch.ones(24, device="cuda", dtype=dtype).requires_grad_()]


@pytest.mark.parametrize("dtype", [F, B])
def test_saved_tensors_and_recomputation(dtype):
    """Saved on the host, where they come back without their strides, or computed again: the same bits."""
    tokens, w, norm = leaves = _leaves(dtype)
    mask = torch.rand(5, 37, device="cuda") < 0.7
    wide = torch.zeros(5, 50, device="cuda", dtype=torch.bool)
    wide[:, 7:44] = mask
    grads = [_r(5, 37, 24, dtype=dtype), _r(5, 37, 24, dtype=dtype), _r(5, 24)]

    def run(f):
        y = f()
        return [*y, *torch.autograd.grad(y, leaves, grads)]

    want = run(lambda: _block(tokens, w, mask, norm))
    with torch.autograd.graph.save_on_cpu():
        got = run(lambda: _block(tokens, w, wide[:, 7:44], norm))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = run(lambda: checkpoint(_block, tokens, w, mask, norm, use_reentrant=False))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("lead", [(6,), (2, 3, 4), (3, 1, 5, 2)])
def test_halves_of_a_projection(lead, dtype):
    """x and gate side by side, in any number of dimensions, and flattened to rows: the bits of contiguous ones, and
    gradients that meet in the projection."""
    d = 20
    both, res, w = _r(*lead, 2 * d, dtype=dtype), _r(*lead, d, dtype=dtype), _r(d, dtype=dtype)
    grads = (_r(*lead, d, dtype=dtype), _r(*lead, d, dtype=dtype))

    def run(split):
        leaf = both.detach().requires_grad_()
        x, gate = split(leaf)
        y = ops.residual_norm(x, res.view(x.shape), w, gate=gate, scale=w, post_weight=w)
        g, = torch.autograd.grad(y, leaf, [t.view(x.shape) for t in grads])
        return [t.detach().reshape(*lead, d) for t in y] + [g]

    want = run(lambda t: (t[..., :d].contiguous(), t[..., d:].contiguous()))
    for split in (lambda t: t.chunk(2, -1), lambda t: t.unflatten(-1, (2, d)).unbind(-2), lambda t: t.flatten(0, -2).chunk(2, -1)):
        got = run(split)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("tensor", [False, True])
def test_schedulers(tensor):
    """Rates and betas that a scheduler changes, as numbers and as a tensor on the device, are those of the step: beside
    the same steps through adamw_ with numbers (lr rounded to 32 bits where the tensor holds it)."""
    n = 300
    p, q = torch.nn.Parameter(torch.ones(n, device="cuda")), torch.ones(n, device="cuda")
    adam = ops.AdamW([p], lr=torch.tensor(0.01, device="cuda") if tensor else 0.01)
    steps = torch.optim.lr_scheduler.OneCycleLR(adam, max_lr=0.1, total_steps=8)
    m, v, t = torch.zeros_like(q), torch.zeros_like(q), torch.zeros((), device="cuda", dtype=torch.int64)
    for k in range(6):
        g = torch.randn(n, generator=torch.Generator(device="cuda").manual_seed(k), device="cuda")
        p.grad = g.clone()
        group = adam.param_groups[0]
        lr, betas = float(group["lr"]), group["betas"]
        adam.step()
        steps.step()
        ops.adamw_([q], [g], [m], [v], [t], lr=lr, betas=betas)
        assert torch.equal(p.detach(), q), k
    assert torch.is_tensor(adam.param_groups[0]["lr"]) == tensor


def test_copies_and_hooks():
    params = [torch.nn.Parameter(_r(5000)), torch.nn.Parameter(_r(7))]
    adam = ops.AdamW([{"params": params[:1], "bits": 8}, {"params": params[1:], "lr": 0.1}], lr=0.01)
    seen = []
    adam.register_step_pre_hook(lambda o, args, kwargs: seen.append(sorted(kwargs)))
    adam.register_step_post_hook(lambda o, args, kwargs: seen.append(len(o.state)))
    for p in params:
        p.grad = torch.ones_like(p)
    norm = ops.clip_grad_norm_(params, float("inf"))
    adam.step(grad_norm=norm, max_norm=1.0)
    assert seen == [["grad_norm", "max_norm"], 2]
    held = io.BytesIO()
    torch.save(adam, held)
    held.seek(0)
    for other in (copy.deepcopy(adam), torch.load(held, weights_only=False)):  # what this test itself has written
        mine = [p for g in other.param_groups for p in g["params"]]
        for a, b in zip(mine, params):
            assert a is not b and torch.equal(a, b)
            assert {k: (t.dtype, t.shape) for k, t in other.state[a].items()} == {k: (t.dtype, t.shape) for k, t in adam.state[b].items()}
            a.grad = torch.ones_like(a)
        before = [p.detach().clone() for p in params]
        other.step()
        assert all(torch.equal(p, b) for p, b in zip(params, before)) and not torch.equal(mine[0], params[0])
    scaler = torch.amp.GradScaler("cuda", init_scale=4.0)
    loss = sum((p * 3).sum() for p in params)
    adam.zero_grad()
    scaler.scale(loss).backward()
    scaler.unscale_(adam)
    assert all(bool((p.grad == 3).all()) for p in params)
    steps = int(adam.state[params[0]]["step"])
    scaler.step(adam)
    scaler.update()
    assert int(adam.state[params[0]]["step"]) == steps + 1


def test_captured_groups_replay():
    """A step of two groups and both widths, captured: replays count, and give the eager steps' bits."""
    def new():
        torch.manual_seed(3)
        ps = [torch.nn.Parameter(torch.randn(n, device="cuda")) for n in (9000, 40, 4096)]
        o = ops.AdamW([{"params": ps[:2]}, {"params": ps[2:], "lr": 0.05, "weight_decay": 0.0}], lr=0.01, bits=8)
        for p in ps:
            p.grad = torch.full_like(p, 0.5)
        o.step()
        return ps, o

    a, one = new()
    b, two = new()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        two.step()
    for k in range(4):
        for p, q in zip(a, b):
            p.grad.normal_(generator=torch.Generator(device="cuda").manual_seed(k))
            q.grad.copy_(p.grad)
        one.step()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(a, b):
            assert torch.equal(p, q)
            assert all(torch.equal(s.float(), t.float()) for s, t in zip(one.state[p].values(), two.state[q].values()))


def test_two_streams_at_once():
    """The same calls on two streams, whose workspaces are their own: each gives what it gives alone."""
    cases = []
    for seed in range(2):
        torch.manual_seed(seed)
        cases.append([_r(2, 3000, 8), _r(2, 3000, 8), _r(2, 8), (_r(2, 3000, 8), _r(2, 8))])

    def run(c):
        x, gate, state = (t.detach().requires_grad_() for t in c[:3])
        y = ops.gated_scan(x, gate, state=state)
        return [*y, *torch.autograd.grad(y, (x, gate, state), c[3])]

    want = [run(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(cases[i]))
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        assert all(torch.equal(a, b) for r in runs for a, b in zip(r, w))
