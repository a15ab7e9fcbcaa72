"""layer_norm against the definition in 64 bits.

Sums run over at most N = 160 terms one after the other and then pairwise, so a mean is
off by at most N u mean |x| (u = 2^-24), a normed value h by that times rstd plus
2 N u |h| for the variance and the products; dx, dw and db are sums of such terms.
Outputs are rounded once (r = u in f32, 2^-8 in bf16)."""
import pytest
import torch

from tgengine_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
N = 160


def _case(shape, dtype, wdtype=None, seed=0, shift=0.3):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=g, device="cuda")

    dim = shape[-1]
    return ((r(*shape) * 1.5 + shift).to(dtype), (r(dim) * 0.2 + 1).to(wdtype or dtype), r(dim).to(wdtype or dtype),
            r(*shape).to(dtype))


def _exact(x, w, b, g, eps):
    """{name: (value, bound)} of y, dx, dw, db."""
    def unit(t):
        return U if t.dtype == torch.float32 else 2.0 ** -8

    dim = x.shape[-1]
    X, G = x.double().reshape(-1, dim), g.double().reshape(-1, dim)
    W = torch.ones(dim, device="cuda", dtype=torch.float64) if w is None else w.double()
    B = torch.zeros_like(W) if b is None else b.double()
    m = X.mean(1, keepdim=True)
    s = ((X - m).square().mean(1, keepdim=True) + eps).rsqrt()
    H = (X - m) * s
    em = N * U * X.abs().mean(1, keepdim=True) + U * X.abs()
    eh = em * s + H.abs() * (2 * N * U + em * s)
    Y = H * W + B
    gw = G * W
    a1, a2 = gw.mean(1, keepdim=True), (gw * H).mean(1, keepdim=True)
    dx = s * (gw - a1 - H * a2)
    abs1, abs2 = gw.abs().mean(1, keepdim=True), (gw * H).abs().mean(1, keepdim=True)
    edx = s * (4 * U * (gw.abs() + abs1 + (H * a2).abs()) + N * U * (abs1 + H.abs() * abs2)
               + eh * a2.abs() + H.abs() * (gw.abs() * eh).mean(1, keepdim=True)) + dx.abs() * (3 * N * U + eh.amax(1, keepdim=True))
    rows = X.shape[0]
    n = (rows + 64) * U
    out = {"y": (Y, eh * W.abs() + 3 * U * ((H * W).abs() + B.abs()) + Y.abs() * unit(x)),
           "dx": (dx, edx + dx.abs() * unit(x))}
    if w is not None:
        dw = (G * H).sum(0)
        out["dw"] = (dw, (G.abs() * eh).sum(0) + n * (G * H).abs().sum(0) + dw.abs() * unit(w))
    if b is not None:
        db = G.sum(0)
        out["db"] = (db, n * G.abs().sum(0) + db.abs() * unit(b))
    return out


def _run(x, w, b, g, eps=1e-5):
    leaves = {"dx": x.detach().requires_grad_()}
    if w is not None:
        leaves["dw"] = w.detach().requires_grad_()
    if b is not None:
        leaves["db"] = b.detach().requires_grad_()
    y = ops.layer_norm(leaves["dx"], leaves.get("dw"), leaves.get("db"), eps=eps)
    return {"y": y, **dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), g)))}


def _check(x, w, b, g, eps=1e-5):
    got = _run(x, w, b, g, eps)
    for name, (y, e) in _exact(x, w, b, g, eps).items():
        t = got[name]
        off = (t.double().reshape(y.shape) - y).abs()
        assert bool((off <= e + 1e-30).all()), f"{name}: {float((off / (e + 1e-30)).max()):.3g} of the bound"
    assert got["y"].shape == x.shape and got["dx"].shape == x.shape and got["y"].dtype == x.dtype == got["dx"].dtype
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x, w, b, eps=eps), got["y"])
    again = _run(x, w, b, g, eps)
    assert all(torch.equal(again[n], got[n]) for n in got)
    return got


@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, None), (torch.bfloat16, None), (torch.bfloat16, torch.float32),
                                          (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("shape", [(1, 1), (7, 2), (3, 5, 3), (240, 172), (1000, 8), (33, 100), (65, 64), (5, 129),
                                   (300, 255), (17, 257), (12, 513), (9, 1000), (40, 2047), (3, 4099), (2, 8192),
                                   (2, 16384), (9, 16383), (5000, 50), (70_001, 12), (1, 777)])
def test_against_64_bits(shape, dtype, wdtype):
    _check(*_case(shape, dtype, wdtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_without_weight_or_bias(dtype):
    x, w, b, g = _case((50, 172), dtype)
    _check(x, None, None, g)
    _check(x, w, None, g)
    _check(x, None, b, g)
    _check(x, w, b, g, eps=0.7)


@pytest.mark.parametrize("dim", [12, 172, 1500])
def test_far_from_zero_and_constant_rows(dim):
    """A mean of 1,000 deviations; rows of one value, whose variance is zero."""
    x, w, b, g = _case((64, dim), torch.float32, shift=1500.0)
    _check(x, w, b, g)
    x[5] = 3.25
    x[6] = 0.0
    y = ops.layer_norm(x, w, b)
    assert torch.equal(y[5], b) and torch.equal(y[6], b)


def test_many_rows():
    """More rows than the workgroups of the backward pass take at once."""
    _check(*_case((200_003, 24), torch.bfloat16))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [5, 50, 172, 600])
def test_layouts(dim, dtype):
    """Strided rows, shifted starts and non-contiguous gradients give the bits of contiguous ones."""
    x, w, b, g = _case((90, dim), dtype)
    want = _run(x, w, b, g)
    wide = torch.randn(90, dim + 11, device="cuda").to(dtype)
    wide[:, 3:3 + dim] = x
    odd = torch.empty(90 * dim + 1, device="cuda", dtype=dtype)[1:].view(90, dim)
    odd.copy_(x)
    for t in (wide[:, 3:3 + dim], odd, x.t().contiguous().t()):
        got = _run(t, w, b, torch.stack([g, g], -1)[..., 0])
        assert all(torch.equal(got[n], want[n]) for n in want)
    one = x[:1].expand(90, dim)  # one row for all
    got, full = _run(one, w, b, g), _run(one.contiguous(), w, b, g)
    assert all(torch.equal(got[n], full[n]) for n in full)


def test_partial_gradients():
    x, w, b, g = _case((40, 172), torch.bfloat16)
    want = _run(x, w, b, g)
    for ask in (("dx",), ("dw",), ("db",), ("dw", "db"), ("dx", "db")):
        leaves = {"dx": x.detach(), "dw": w.detach(), "db": b.detach()}
        for n in ask:
            leaves[n].requires_grad_()
        y = ops.layer_norm(*leaves.values())
        for n, d in zip(ask, torch.autograd.grad(y, [leaves[n] for n in ask], g)):
            assert torch.equal(d, want[n]), (ask, n)


def test_not_finite_rows_stay_apart():
    """NaN and infinity in one row reach no other row's outputs."""
    x, w, b, g = _case((20, 100), torch.float32)
    want = _run(x, w, b, g)
    x[3, 7], x[11, 0] = float("nan"), float("inf")
    got = _run(x, w, b, g)
    rest = [i for i in range(20) if i not in (3, 11)]
    assert torch.equal(got["y"][rest], want["y"][rest]) and torch.equal(got["dx"][rest], want["dx"][rest])
    assert got["y"][3].isnan().all() and got["y"][11].isnan().any()


def test_gradient_against_differences():
    """Central differences of the forward kernel, h = 2^-7: h^2 of curvature and u / h of
    rounding, together below 2^-9 of the sum of |y * g|."""
    x, w, b, g = _case((6, 50), torch.float32)
    got = _run(x, w, b, g)
    size = (got["y"].double() * g.double()).abs().sum()
    h = 2.0 ** -7
    for i, name in enumerate(("dx", "dw", "db")):
        step = torch.randn_like((x, w, b)[i])
        step = step / step.norm()
        f = [(ops.layer_norm(*[t + s * step if j == i else t for j, t in enumerate((x, w, b))]).double()
              * g.double()).sum() for s in (h, -h)]
        assert abs((f[0] - f[1]) / (2 * h) - (got[name].double() * step.double()).sum()) <= size * 2.0 ** -9, name


def test_empty_and_refusals():
    w = torch.ones(8, device="cuda", requires_grad=True)
    x = torch.empty(0, 8, device="cuda", requires_grad=True)
    y = ops.layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert y.shape == dx.shape == (0, 8) and not dw.any()
    x = torch.randn(3, 8, device="cuda")
    L = ops.layer_norm
    for args, text in (((x, w[:7]), r"\(dim,\)"), ((x, w, w.bfloat16()), "same dtype"), ((x.half(),), "float32 or bfloat16"),
                       ((x, w.detach().cpu()), "device"), ((x[:, :0],), "last dimension")):
        with pytest.raises(ValueError, match=text):
            L(*args)
    with pytest.raises(RuntimeError, match="on the GPU"):
        L(x.cpu())
    with pytest.raises(RuntimeError, match="at most 16384"):
        L(torch.zeros(1, 16385, device="cuda"))
    with pytest.raises(RuntimeError, match="once only"):
        torch.autograd.grad(L(x, w).sum(), w, create_graph=True)
