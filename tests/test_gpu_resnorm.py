"""residual_norm against its definition in 64 bits.

u = 2^-24; a sum of a row's values is off by at most N u times their absolute sum (N = 160
terms one after the other, then pairwise).  Errors are carried through the formulas term by
term: sigmoid(gate) and 1 - sigmoid(gate) are off by s = (2 |gate| + 6) u relatively (the
exponent's argument, a power, a sum, a reciprocal), the sum by its terms' errors and a
rounding, a mean by the mean of its terms' errors, and so on (_norm, _norm_back).  Column
sums are off by (rows + 64) u of their absolute sums.  Outputs are rounded once (r = u in
f32, 2^-8 in bf16)."""
import pytest
import torch

from tgengine_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
N = 160
F, B = torch.float32, torch.bfloat16
PARTS = ("x", "residual", "weight", "bias", "gate", "scale", "post_weight")
ALL = ("weight", "bias", "gate", "scale", "post_weight")


def _case(shape, dtype, parts=ALL, wdtype=None, center=True, seed=0, shift=0.3):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=g, device="cuda")

    d, wt = shape[-1], wdtype or dtype
    c = {"x": r(*shape).to(dtype), "residual": (r(*shape) * 1.5 + shift).to(dtype), "weight": (r(d) * 0.2 + 1).to(wt),
         "bias": r(d).to(wt), "gate": (r(*shape) * 2).to(dtype), "scale": (r(d) * 0.2 + 0.5).to(wt),
         "post_weight": (r(d) * 0.2 + 1).to(wt), "center": center, "eps": 1e-5, "grads": (r(*shape).to(dtype), r(*shape).to(dtype))}
    return {k: None if k in ALL and k not in parts else v for k, v in c.items()}


def _norm(v, e, center, eps):
    """h, its error, 1 / deviation, its relative error"""
    m = v.mean(1, keepdim=True) if center else 0.0
    em = N * U * v.abs().mean(1, keepdim=True) + e.mean(1, keepdim=True) if center else 0.0
    f = v - m
    ef = e + em + U * f.abs()
    r = (f.square().mean(1, keepdim=True) + eps).rsqrt()
    er = r * r * (f.abs() * ef).mean(1, keepdim=True) + N * U
    h = f * r
    return h, r * ef + h.abs() * (er + 2 * U), r, er


def _norm_back(g, eg, h, eh, r, er, center):
    a1 = g.mean(1, keepdim=True) if center else torch.zeros_like(r)
    e1 = eg.mean(1, keepdim=True) + N * U * g.abs().mean(1, keepdim=True) if center else 0.0
    a2 = (g * h).mean(1, keepdim=True)
    e2 = (g.abs() * eh + eg * h.abs() + N * U * (g * h).abs()).mean(1, keepdim=True)
    q = g - a1 - h * a2
    eq = eg + e1 + eh * a2.abs() + h.abs() * e2 + 4 * U * (g.abs() + a1.abs() + (h * a2).abs())
    return r * q, r * eq + (r * q).abs() * (er + 3 * U)


def _exact(c):
    """{name: (value, bound)}"""
    d = c["x"].shape[-1]
    get = {n: c[n].double().reshape(-1, d) if c[n] is not None and c[n].dim() > 1 else None if c[n] is None else c[n].double()
           for n in PARTS}
    x, residual, w, b, gate, scale, post = (get[n] for n in PARTS)
    zero = torch.zeros_like(x)
    rows, center = x.shape[0], c["center"]

    def r(t):
        return U if t.dtype == F else 2.0 ** -8

    n, en, hx, ehx, rx, erx = x, zero, None, None, None, None
    if post is not None:
        hx, ehx, rx, erx = _norm(x, zero, center, c["eps"])
        n = hx * post
        en = ehx * post.abs() + 2 * U * n.abs()
    sig, rest = (torch.sigmoid(gate), torch.sigmoid(-gate)) if gate is not None else (torch.ones_like(x), torch.ones_like(x))
    sg = (2 * gate.abs() + 6) * U if gate is not None else zero
    by = sig * scale if scale is not None else sig
    s = residual + by * n
    es = by.abs() * en + (by * n).abs() * (sg + 2 * U) + U * s.abs()
    h, eh, rs, ers = _norm(s, es, center, c["eps"])
    W = w if w is not None else torch.ones(d, device="cuda", dtype=torch.float64)
    bias = b if b is not None else torch.zeros_like(W)
    y = h * W + bias
    out = {"y": (y, eh * W.abs() + 3 * U * ((h * W).abs() + bias.abs()) + r(c["x"]) * y.abs()),
           "sum": (s, es + r(c["x"]) * s.abs())}
    gy, gs = (g.double().reshape(-1, d) for g in c["grads"])
    g = gy * W
    v, ev = _norm_back(g, U * g.abs(), h, eh, rs, ers, center)
    dd = gs + v
    ed = ev + 2 * U * dd.abs()
    out["residual"] = dd, ed + r(c["x"]) * dd.abs()
    dn = dd * by
    edn = ed * by.abs() + dn.abs() * (sg + 2 * U)
    if gate is not None:
        dg = dn * n * rest
        out["gate"] = dg, edn * (n * rest).abs() + (dn * rest).abs() * en + dg.abs() * (sg + 3 * U + r(c["x"]))
    dx, edx = dn, edn
    if post is not None:
        q = dn * post
        dx, edx = _norm_back(q, edn * post.abs() + U * q.abs(), hx, ehx, rx, erx, center)
    out["x"] = dx, edx + r(c["x"]) * dx.abs()

    def column(name, t, e):
        total = t.sum(0)
        out[name] = total, e.sum(0) + (rows + 64) * U * t.abs().sum(0) + r(c[name]) * total.abs()

    if w is not None:
        column("weight", gy * h, gy.abs() * eh)
    if b is not None:
        column("bias", gy, zero)
    if scale is not None:
        t = dd * sig * n
        column("scale", t, ed * (sig * n).abs() + (dd * sig).abs() * en + t.abs() * (sg + 2 * U))
    if post is not None:
        column("post_weight", dn * hx, edn * hx.abs() + dn.abs() * ehx)
    return out


def _call(c, **more):
    t = {**c, **more}
    return ops.residual_norm(*(t[n] for n in ("x", "residual", "weight", "bias")), gate=t["gate"], scale=t["scale"],
                             post_weight=t["post_weight"], center=t["center"], eps=t["eps"])


def _run(c, names=PARTS, grads=None):
    leaves = {n: c[n].detach().requires_grad_() for n in names if c[n] is not None}
    y = _call(c, **leaves)
    pairs = [(o, g) for o, g in zip(y, grads or c["grads"]) if g is not None]
    d = torch.autograd.grad([p[0] for p in pairs], list(leaves.values()), [p[1] for p in pairs])
    return {"y": y[0].detach(), "sum": y[1].detach(), **dict(zip(leaves, d))}


def _check(c):
    got = _run(c)
    for name, (y, e) in _exact(c).items():
        t = got[name]
        off = (t.double().reshape(y.shape) - y).abs()
        assert bool((off <= 1.01 * e + 1e-37).all()), f"{name}: {float((off / (1.01 * e + 1e-37)).max()):.3g} of the bound"
    for n in ("y", "sum"):
        assert got[n].shape == c["x"].shape and got[n].dtype == c["x"].dtype
    with torch.no_grad():
        y, s = _call(c)
    assert torch.equal(y, got["y"]) and torch.equal(s, got["sum"])
    again = _run(c)
    assert all(torch.equal(again[n], got[n]) for n in got)
    return got


SHAPES = [(1, 1), (7, 2), (3, 5, 3), (240, 172), (1000, 8), (33, 100), (65, 64), (5, 129), (300, 255), (17, 257), (12, 513),
          (9, 1000), (40, 2047), (3, 4099), (2, 8191), (2, 16384), (3, 16383), (5000, 50), (70_001, 12), (1, 777)]


@pytest.mark.parametrize("dtype,wdtype", [(F, None), (B, None), (B, F), (F, B)])
@pytest.mark.parametrize("shape", SHAPES)
def test_against_64_bits(shape, dtype, wdtype):
    _check(_case(shape, dtype, wdtype=wdtype))
    _check(_case(shape, dtype, ("weight", "bias"), wdtype))


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("parts", [(), ("gate",), ("scale",), ("post_weight",), ("gate", "scale"), ("weight", "post_weight"),
                                   ("bias", "gate", "post_weight"), ("weight",), ALL])
def test_parts(parts, dtype):
    """Every part there or not; layer norms and root mean squares; a large eps."""
    for center in (True, False):
        for shape in ((90, 172), (4, 3000)):
            _check(_case(shape, dtype, parts, center=center))
    _check({**_case((50, 60), dtype, parts), "eps": 0.7})


@pytest.mark.parametrize("center", [True, False])
@pytest.mark.parametrize("dim", [12, 172, 1500])
def test_far_from_zero_and_constant_rows(dim, center):
    c = _case((64, dim), F, shift=1500.0, center=center)
    _check(c)
    c = _case((64, dim), F, ("weight", "bias"), center=center)
    c["x"][5:7], c["residual"][5], c["residual"][6] = 0.0, 3.25, 0.0
    y, s = _call(c)
    assert torch.equal(y[6], c["bias"]) and torch.equal(s[5], c["residual"][5])
    if center:
        assert torch.equal(y[5], c["bias"])


def test_many_rows():
    _check(_case((200_003, 24), B))
    _check(_case((200_003, 24), B, ("weight", "bias")))


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("parts", [("weight", "bias"), ALL])
@pytest.mark.parametrize("dim", [5, 50, 172, 600])
def test_layouts(dim, parts, dtype):
    """Strided rows, shifted starts and non-contiguous gradients give the bits of contiguous ones."""
    c = _case((90, dim), dtype, parts)
    want = _run(c)
    rows = [n for n in ("x", "residual", "gate") if c[n] is not None]

    def same(**more):
        got = _run({**c, **more})
        assert all(torch.equal(got[n], want[n]) for n in want)

    for n in rows:
        wide = torch.randn(90, dim + 11, device="cuda").to(dtype)
        wide[:, 3:3 + dim] = c[n]
        odd = torch.empty(90 * dim + 1, device="cuda", dtype=dtype)[1:].view(90, dim)
        same(**{n: wide[:, 3:3 + dim]})
        same(**{n: odd.copy_(c[n])})
        same(**{n: c[n].t().contiguous().t()})
    same(**{n: c[n].view(9, 10, dim).transpose(0, 1).contiguous().transpose(0, 1).reshape(90, dim) for n in rows})
    same(grads=tuple(torch.stack([g] * 2, -1)[..., 0] for g in c["grads"]))
    same(weight=torch.stack([c["weight"]] * 2, -1)[:, 0])
    for n in rows:  # one row for all
        one = {**c, n: c[n][:1].expand(90, dim)}
        got, full = _run(one), _run({**one, n: one[n].contiguous()})
        assert all(torch.equal(got[k], full[k]) for k in full)
    cube = {**c, **{n: c[n].view(9, 10, dim) for n in rows}, "grads": tuple(g.view(9, 10, dim) for g in c["grads"])}
    got = _run(cube)
    assert all(torch.equal(got[n].view(want[n].shape), want[n]) for n in want)


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("parts", [("weight", "bias"), ALL])
def test_partial_gradients(parts, dtype):
    c = _case((40, 172), dtype, parts)
    want = _run(c)
    there = [n for n in PARTS if c[n] is not None]
    for names in [(n,) for n in there] + [("residual", "weight"), ("x", "bias"), ("x", "residual")]:
        got = _run(c, names)
        assert all(torch.equal(got[n], want[n]) for n in got), names
    for i in (0, 1):  # one of the two outputs used
        only, full = list(c["grads"]), list(c["grads"])
        only[i], full[i] = None, torch.zeros_like(full[i])
        a, b = _run(c, grads=only), _run(c, grads=full)
        for n in a:
            assert torch.equal(a[n], b[n]), n


def test_same_tensor_twice():
    """x and residual one tensor: its gradient is the sum of both."""
    c = _case((30, 100), F, ("weight", "bias"))
    c["residual"] = c["x"]
    want = _run(c)
    x = c["x"].detach().requires_grad_()
    (_call(c, x=x, residual=x)[0] * c["grads"][0] + _call(c, x=x, residual=x)[1] * 0).sum().backward()
    a = _run(c, grads=(c["grads"][0], torch.zeros_like(c["x"])))
    assert torch.equal(x.grad, a["x"] + a["residual"]) and torch.equal(a["y"], want["y"])


def test_not_finite_rows_stay_apart():
    c = _case((20, 100), F)
    want = _run(c)
    c["x"][3, 7], c["residual"][11, 0], c["gate"][15, 2] = float("nan"), float("inf"), float("-inf")
    got = _run(c)
    rest = [i for i in range(20) if i not in (3, 11, 15)]
    for n in ("y", "sum", "x", "residual", "gate"):
        assert torch.equal(got[n][rest], want[n][rest])
    assert got["y"][3].isnan().all() and got["y"][11].isnan().any()
    assert got["sum"][15, 2] == c["residual"][15, 2] and got["y"][15].isfinite().all()


@pytest.mark.parametrize("center", [True, False])
def test_gradient_against_differences(center):
    """Central differences of the forward kernel, h = 2^-7: h^2 of curvature and u / h of
    rounding, together below 2^-8 of the sum of |output * g| (two outputs, sums of seven
    parts each)."""
    c = _case((6, 50), F, center=center)
    got = _run(c)
    size = sum((got[n].double() * g.double()).abs().sum() for n, g in zip(("y", "sum"), c["grads"]))
    h = 2.0 ** -7
    for name in PARTS:
        step = torch.randn_like(c[name])
        step = step / step.norm()
        f = [sum((o.double() * g.double()).sum() for o, g in zip(_call(c, **{name: c[name] + s * step}), c["grads"]))
             for s in (h, -h)]
        assert abs((f[0] - f[1]) / (2 * h) - (got[name].double() * step.double()).sum()) <= size * 2.0 ** -8, name


@pytest.mark.parametrize("parts", [("weight", "bias"), ALL])
def test_streams_and_graph_replays(parts):
    c = _case((500, 172), B, parts)
    want = _run(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(c)
    side.synchronize()
    assert all(torch.equal(got[n], want[n]) for n in want)
    static = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _run(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _run(static)
    for seed in range(4):
        new = {**_case((500, 172), B, parts, seed=10 + seed), "grads": c["grads"]}
        for n in PARTS:
            if new[n] is not None:
                static[n].copy_(new[n])
        graph.replay()
        torch.cuda.synchronize()
        want = _run(new)
        assert all(torch.equal(held[n], want[n]) for n in want)


def test_empty_and_refusals():
    c = _case((0, 8), F)
    got = _run(c)
    assert got["y"].shape == got["x"].shape == (0, 8) and not got["weight"].any() and not got["post_weight"].any()
    R = ops.residual_norm
    x, w = torch.randn(3, 8, device="cuda"), torch.ones(8, device="cuda")
    for args, more, text in (((x, x[:2]), {}, "shape of x"), ((x, x.bfloat16()), {}, "same dtype"), ((x.half(), x.half()), {}, "float32 or bfloat16"),
                             ((x, x.cpu()), {}, "device"), ((x, x, w[:7]), {}, r"\(dim,\)"), ((x, x, w, w.bfloat16()), {}, "same dtype"),
                             ((x, x, w), {"scale": w.bfloat16()}, "same dtype"), ((x, x), {"gate": x[:, :4]}, "shape of x"),
                             ((x, x), {"gate": x.bfloat16()}, "same dtype"), ((x, x), {"scale": w.cpu()}, "device"),
                             ((x, x), {"post_weight": x}, r"\(dim,\)"), ((x[:, :0], x[:, :0]), {}, "last dimension")):
        with pytest.raises(ValueError, match=text):
            R(*args, **more)
    with pytest.raises(RuntimeError, match="on the GPU"):
        R(x.cpu(), x.cpu())
    with pytest.raises(RuntimeError, match="at most 16384"):
        R(torch.zeros(1, 16385, device="cuda"), torch.zeros(1, 16385, device="cuda"))
    v = w.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="once only"):
        torch.autograd.grad(R(x, x, v)[0].sum(), v, create_graph=True)
