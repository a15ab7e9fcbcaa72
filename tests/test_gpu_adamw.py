"""adamw_ and AdamW against the step in 64 bits.

u = 2^-24.  With 32-bit averages the constants, the clipped gradient, two products and a sum
round once each: m is off by 6 u (|b1 m| + |c1 g|), v, whose terms are not negative, by 8 u v,
its root by 5 u relatively.  The update divides by a root times a factor plus eps and is
off by 16 u (with a unit more for the division) and by m's error over the same divisor; the
decayed parameter is off by 3 u.  8-bit averages are updated in 64 bits and then rounded: their
codes and scales are compared for equality, by a table of the format's values.  A
parameter is rounded once to its type (u, or 2^-8 in bf16)."""
import numpy as np
import pytest
import torch

from tgengine_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F, B, E = torch.float32, torch.bfloat16, torch.float8_e4m3fn
TABLE = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** e for e in range(-9, 6) for m in range(8)] + [512.0]


def held(x, which, step):
    """(codes as values, scales) of 64-bit values: the definition, by numpy."""
    x = x.detach().cpu().double().numpy().reshape(-1)
    n = x.size
    size = np.abs(np.pad(x, (0, -n % 256))).reshape(-1, 256)
    fine = np.isfinite(size)
    top = np.where(fine, size, 0.0).max(1, keepdims=True) if n else size[:, :1]
    k = np.where(top == 0, -126, np.maximum(np.frexp(top)[1] - 8, -126)).astype(np.int64)
    y = np.ldexp(np.where(fine, size, 0.0), -k)
    table = np.array(TABLE)
    at = np.searchsorted(table, y, side="right") - 1
    w = (np.arange(n, dtype=np.uint64) * 0xC13FA9A9 + np.uint64((step * 0x91E10DA5 + which * 2 ** 31) % 2 ** 32)) % 2 ** 32
    u = np.pad(w.astype(np.float64) / 2.0 ** 32, (0, -n % 256)).reshape(-1, 256)
    low, high = table[at], table[at + 1]
    # one spacing is (high - low): the place between the two neighbours plus the dither
    out = np.where((y - low) / (high - low) + u >= 1.0, high, low)
    if which:
        out = np.where((size > 0) & fine & (out == 0), TABLE[1], out)
    out = np.where(fine, out, np.nan).reshape(-1)[:n]
    out = np.where(x == 0, 0.0, np.copysign(out, x)) if not which else out
    return torch.from_numpy(out), torch.from_numpy(np.ldexp(1.0, k)[:, 0])


def _make(sizes, dtypes, bits, seed=0, gdtypes=None, steps=None, fresh=False):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(n, s, t=F):
        return (torch.randn(n, generator=g, device="cuda") * s).to(t)

    bits = [bits] * len(sizes) if isinstance(bits, int) else bits
    c = {"params": [r(n, 0.05, t) for n, t in zip(sizes, dtypes)], "grads": [r(n, 0.01, t) for n, t in zip(sizes, gdtypes or dtypes)],
         "exp_avg": [], "exp_avg_sq": [], "scales": [], "steps": [torch.tensor(s, device="cuda") for s in steps or [7 + 100 * i for i in range(len(sizes))]]}
    for n, b in zip(sizes, bits):
        m, v = (r(n, 0.002), (r(n, 0.002) + 0.008).square()) if not fresh else (torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda"))
        if b == 8:
            blocks = -(-n // 256)
            (m, a), (v, q) = held(m, 0, 3), held(v.sqrt(), 1, 3)
            c["scales"].append(torch.zeros(2, blocks, device="cuda") if fresh else torch.stack([a, q]).float().cuda())
            c["exp_avg"].append(m.cuda().float().to(E))
            c["exp_avg_sq"].append(v.cuda().float().to(E))
        else:
            c["scales"].append(None)
            c["exp_avg"].append(m)
            c["exp_avg_sq"].append(v)
    return c


def _clone(c):
    return {k: [x.clone() if x is not None else None for x in v] for k, v in c.items()}


def _spread(x, scale):
    return x.double().view(-1) * scale.double().repeat_interleave(256)[:x.numel()]


def _check(c, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, wd=1e-2, norm=None, max_norm=None, **more):
    before = _clone(c)
    ops.adamw_(**c, lr=lr, betas=betas, eps=eps, weight_decay=wd, grad_norm=norm, max_norm=max_norm, **more)
    lr = float(lr)
    clip = 1.0 if norm is None else min(1.0, max_norm / (float(norm) + 1e-6))
    b1, b2 = betas
    for i, p0 in enumerate(before["params"]):
        t = int(before["steps"][i]) + 1
        assert int(c["steps"][i]) == t and torch.equal(c["grads"][i], before["grads"][i])
        if p0.numel() == 0:
            continue
        g = before["grads"][i].double() * clip
        m0, v0 = before["exp_avg"][i], before["exp_avg_sq"][i]
        wide = m0.dtype == F
        if wide:
            m0, v0 = m0.double(), v0.double()
        else:
            m0, v0 = (_spread(x, before["scales"][i][j]).view(p0.shape) for j, x in enumerate((m0, v0)))
            v0 = v0 * v0
        m, v = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * (g * g)
        root = v.sqrt()
        by = lr / (1 - b1 ** t)
        div = root / (1 - b2 ** t) ** 0.5 + eps
        up = by * m / div
        p = p0.double() * (1 - lr * wd) - up
        em = 6 * U * ((b1 * m0).abs() + ((1 - b1) * g).abs()) if wide else U * m.abs()
        e = 3 * U * p0.double().abs() + 16 * U * up.abs() + by * em / div + p.abs() * (U if p0.dtype == F else 2.0 ** -8)
        got = c["params"][i]
        assert got.dtype == p0.dtype
        off = (got.double() - p).abs()
        assert bool((off <= 1.01 * e + 1e-37).all()), f"parameter {i}: {float((off / (1.01 * e + 1e-37)).max()):.3g} of the bound"
        if wide:
            assert bool(((c["exp_avg"][i].double() - m).abs() <= em + 1e-44).all())
            assert bool(((c["exp_avg_sq"][i].double() - v).abs() <= 8 * U * v + 1e-44).all())
        else:
            for j, (name, x) in enumerate((("exp_avg", m), ("exp_avg_sq", root))):
                want, scale = held(x, j, t)
                assert torch.equal(c["scales"][i][j].cpu().double(), scale), (i, name)
                assert torch.equal(c[name][i].cpu().double().view(-1), want), (i, name)
    return c


SIZES = [((1,), (F,)), ((7,), (B,)), ((256,), (F,)), ((255, 257, 1, 1024), (F, B, F, B)), ((20_000, 116, 1, 20_001), (F,) * 4),
         ((300_001, 5, 0, 77), (B, F, B, B)), (tuple(range(1, 120)), (F, B, F) * 40), ((3_000_003, 8_191, 8_193), (F, F, B)),
         ((0, 0, 5), (F, B, F))]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes,dtypes", SIZES)
def test_step(sizes, dtypes, bits):
    c = _check(_make(sizes, dtypes, bits))
    _check(c)  # from its own state
    norm = torch.tensor(3.0, device="cuda")
    _check(_make(sizes, dtypes, bits, 1), norm=norm, max_norm=1.0)
    _check(_make(sizes, dtypes, bits, 2), norm=norm, max_norm=100.0, lr=0.02, betas=(0.8, 0.95), eps=1e-4, wd=0.3)


@pytest.mark.parametrize("bits", [32, 8])
def test_fresh_and_mixed(bits):
    """First steps from zeros; gradients of another type; 8 and 32 bits in one call."""
    sizes = (5000, 300, 4096)
    _check(_make(sizes, (F, B, F), bits, fresh=True, steps=[0] * 3))
    _check(_make(sizes, (B, F, B), bits, gdtypes=(F, B, B)))
    _check(_make(sizes, (F, B, F), [bits, 40 - bits, bits]))
    _check(_make(sizes, (F,) * 3, bits), betas=(0.0, 0.0), eps=0.1)
    _check(_make(sizes, (F,) * 3, bits), lr=0.0)
    _check(_make((70,) * 130, (F,) * 130, [8, 32] * 65, steps=[2 ** 33 + i for i in range(130)]))


def test_lists_of_any_length():
    _check(_make((3,) * 700, (F,) * 700, 32))


@pytest.mark.parametrize("bits", [32, 8])
def test_shifted_and_shaped(bits):
    base = _make((50_003, 4_000), (B, F), bits)
    c = _clone(base)
    for k in ("params", "grads", "exp_avg", "exp_avg_sq"):
        big = torch.zeros(50_005, device="cuda").to(c[k][0].dtype)
        big[2:] = c[k][0]
        c[k] = [big[2:], c[k][1].view(40, 100)]
    _check(c)
    ops.adamw_(**base)
    assert all(torch.equal(a.view(-1).float(), b.view(-1).float()) for k in ("params", "exp_avg", "exp_avg_sq") for a, b in zip(base[k], c[k]))


def test_values_far_apart():
    """Blocks of zeros, blocks whose values span the format's range and more, tiny and large ones."""
    c = _make((256 * 9 + 30,), (F,), 8, fresh=True, steps=[0])
    g = c["grads"][0]
    g[256:512] = 0
    g[512:768] *= 10.0 ** torch.linspace(-12, 6, 256, device="cuda")
    g[768:1024] *= 1e-30
    g[1024:1280] *= 1e25
    g[1280:1536] = 2.0 ** torch.arange(-128, 128, device="cuda").clamp(-140, 60).float()
    g[1536:1792] *= 1e-38
    for _ in range(3):
        _check(c, norm=torch.tensor(1.0, device="cuda"), max_norm=1.0)
    root = c["exp_avg_sq"][0].float()
    assert bool((root[g != 0] > 0).all()) and not root[g == 0].any()


def test_averages_on_borders():
    """Averages that are powers of two and numbers of the format themselves: gradients equal to the first
    average, whose squares' roots are those numbers."""
    c = _make((2048,), (F,), 8, fresh=True, steps=[0])
    values = torch.tensor(TABLE[:-1] * 20, device="cuda")[:2048].float()
    c["grads"][0].copy_(torch.where(torch.arange(2048, device="cuda") % 2 == 0, values, -values))
    for betas in ((0.0, 0.0), (0.5, 0.0), (0.9, 0.0), (0.9, 0.75), (0.5, 0.5), (0.9, 0.999)):
        for _ in range(3):
            _check(c, betas=betas, eps=1e-3)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_not_finite_stays_in_its_place(bits, bad):
    c = _make((1000, 40), (F, B), bits)
    d = _clone(c)
    d["grads"][0][300] = bad
    ops.adamw_(**c)
    ops.adamw_(**d)
    rest = torch.arange(1000, device="cuda") != 300
    for k in ("params", "exp_avg", "exp_avg_sq"):
        if bits == 32 or k == "params":
            assert torch.equal(c[k][0][rest], d[k][0][rest]) and torch.equal(c[k][1], d[k][1])
    assert d["params"][0][300].isnan() and (bits == 32 or d["exp_avg"][0][300].float().isnan())
    if bits == 8:  # its block's scale is the largest finite value's
        d["grads"][0][300] = 0
        ops.adamw_(**d)
        assert int(d["params"][0].isnan().sum()) == 1 and d["exp_avg"][0].float()[rest].isfinite().all()
    norm = torch.tensor(float("nan"), device="cuda")
    ops.adamw_(**c, grad_norm=norm, max_norm=1.0)
    assert c["params"][0].isnan().all()


def test_slow_averages_move():
    """A root that shrinks by 1 - sqrt(0.999) = d a step: rounded to the nearest it would never leave its place.

    In units of its spacing a root is n = 8 .. 15, and n (1 - d) + u falls below n where u < n d, 8 d = 0.004001 at
    least.  u turns by 0x91E10DA5 / 2^32 a step, modulo 1; the times between two visits of a turning point to an
    interval are of three lengths at most, for one of 0.004001 of 451 steps at most (counted).  In 2,000 steps every
    root falls at least 4 times, by a place of the format each.  That each step is the definition's is compared bit
    by bit, on the way down and up."""
    c = _make((4096,), (F,), 8, fresh=True, steps=[0])
    c["exp_avg_sq"][0].copy_((torch.rand(4096, device="cuda") + 1) * 128)
    c["scales"][0].fill_(2.0 ** -7)

    def now():
        return _spread(c["exp_avg_sq"][0].cpu(), c["scales"][0][1].cpu())

    def place(x):  # a root's number among all of the format's, 8 for every octave
        f, e = np.frexp(x.numpy())
        return e * 8 + (f * 16).astype(int)

    first = now()
    for g, steps in ((0.0, 2000), (1.0, 300)):
        c["grads"][0].fill_(g)
        want = now()
        for t in range(int(c["steps"][0]) + 1, int(c["steps"][0]) + 1 + steps):
            ops.adamw_(**c, lr=0.0)
            if t % 100 < 20:  # every step of some, from where it is
                v, s = held((0.999 * (want * want) + (1 - 0.999) * (torch.full_like(want, g) ** 2)).sqrt(), 1, t)
                assert torch.equal(now(), _spread(v, s)), t
            want = now()
        if g == 0.0:
            assert bool((place(now()) <= place(first) - 4).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_graph_replays(bits):
    """A captured step counts, and takes new gradients, a new norm and a new rate, at every replay."""
    lr, norm = torch.tensor(1e-3, device="cuda"), torch.tensor(2.0, device="cuda")
    c = _make((5000, 300), (F, B), bits)
    want = _clone(c)
    static = c["grads"]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.adamw_(**c, lr=lr, grad_norm=norm, max_norm=1.0)
    for k in range(5):
        for i, g in enumerate(_make((5000, 300), (F, B), bits, 20 + k)["grads"]):
            static[i].copy_(g)
            want["grads"][i].copy_(g)
        lr.fill_(1e-3 * (k + 1))
        norm.fill_(0.5 + k)
        graph.replay()
        torch.cuda.synchronize()
        ops.adamw_(**want, lr=lr, grad_norm=norm, max_norm=1.0)
        for name in c:
            assert all(a is None or torch.equal(a.float(), b.float()) for a, b in zip(c[name], want[name])), (k, name)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.adamw_(**c, lr=lr)
    side.synchronize()
    ops.adamw_(**want, lr=lr)
    assert all(torch.equal(a, b) for a, b in zip(c["params"], want["params"]))


# ---------------------------------------------------------------- the optimizer
def _model(dtype=F, seed=0):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(64, 80), torch.nn.GELU(), torch.nn.Linear(80, 3)).to("cuda", dtype)


def _backward(model, k):
    x = torch.randn(32, 64, generator=torch.Generator(device="cuda").manual_seed(k), device="cuda").to(next(model.parameters()).dtype)
    model.zero_grad(set_to_none=True)
    model(x).float().square().sum().backward()


def test_optimizer_follows_torch():
    """Ten steps beside torch.optim.AdamW on the same gradients.  A step's two results differ by at most 30 u
    of the update, which is below 4 lr here, and 6 u of the parameter, below 1; ten of them."""
    a, b = _model(), _model()
    mine, theirs = ops.AdamW(a.parameters(), lr=1e-3), torch.optim.AdamW(b.parameters(), lr=1e-3)
    for k in range(10):
        _backward(b, k)
        for p, q in zip(a.parameters(), b.parameters()):
            p.grad = q.grad.clone()
        mine.step()
        theirs.step()
    for p, q in zip(a.parameters(), b.parameters()):
        assert bool(((p - q).abs() <= 10 * U * (30 * 4e-3 + 6)).all())
        assert p.grad is not None and int(mine.state[p]["step"]) == 10


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_state_is_kept(bits, dtype, tmp_path):
    """Saved and loaded, the next steps are the same bits; types survive; small tensors stay in 32 bits."""
    a = _model(dtype)
    one = ops.AdamW(a.parameters(), lr=1e-2, bits=bits)
    for k in range(3):
        _backward(a, k)
        one.step()
    kinds = {tuple(p.shape): one.state[p]["exp_avg"].dtype for p in a.parameters()}
    assert kinds[(80, 64)] == (E if bits == 8 else F) and kinds[(80,)] == F
    torch.save({"m": a.state_dict(), "o": one.state_dict()}, tmp_path / "x.pt")
    saved = torch.load(tmp_path / "x.pt", weights_only=True)
    b = _model(dtype, 5)
    b.load_state_dict(saved["m"])
    two = ops.AdamW(b.parameters(), bits=bits)
    two.load_state_dict(saved["o"])
    for k in range(3, 6):
        for m, o in ((a, one), (b, two)):
            _backward(m, k)
            o.step()
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q) and one.state[p]["exp_avg"].dtype == two.state[q]["exp_avg"].dtype
        assert int(two.state[q]["step"]) == 6 and two.state[q]["step"].dtype == torch.int64


def test_optimizer_clips_as_it_reads():
    """The norm alone, and the step that scales by it, give the step of clipped gradients within a rounding of each:
    clipped gradients round once more, u of m and of the root, 20 u of the update in all; it is below 4 lr, the
    parameters below 1."""
    a, b = _model(), _model()
    one, two = ops.AdamW(a.parameters(), lr=1e-2), ops.AdamW(b.parameters(), lr=1e-2)
    for m in (a, b):
        _backward(m, 0)
    before = [p.grad.clone() for p in a.parameters()]
    norm = ops.clip_grad_norm_(a.parameters(), float("inf"))
    assert all(torch.equal(p.grad, g) for p, g in zip(a.parameters(), before)) and float(norm) > 0.5
    one.step(grad_norm=norm, max_norm=0.5)
    ops.clip_grad_norm_(b.parameters(), 0.5)
    two.step()
    for p, q in zip(a.parameters(), b.parameters()):
        assert bool(((p - q).abs() <= U * (50 * 4e-2 + 6)).all())


def test_optimizer_groups_closures_and_capture():
    a = _model()
    ps = list(a.parameters())
    o = ops.AdamW([{"params": ps[:2], "lr": 0.0, "weight_decay": 0.0}, {"params": ps[2:]}], lr=1e-2)
    before = [p.detach().clone() for p in ps]
    _backward(a, 0)
    ps[3].grad = None
    assert o.step(lambda: torch.tensor(2.5)) == 2.5
    assert all(torch.equal(p, q) for p, q in zip(ps[:2] + ps[3:], before[:2] + before[3:])) and not torch.equal(ps[2], before[2])
    assert not o.state[ps[3]]
    ps[2].grad = ps[2].grad.t().contiguous().t()  # not contiguous
    o.step()
    n = torch.nn.Parameter(torch.zeros(5, device="cuda"))
    n.grad = torch.ones_like(n)
    fresh = ops.AdamW([n])
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="first step"):
        with torch.cuda.graph(graph):
            fresh.step()
    fresh.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fresh.step()
    for k in range(3):
        graph.replay()
    assert int(fresh.state[n]["step"]) == 4 and bool((n < -3.9e-3).all())


def test_versions():
    """What autograd saved of a parameter is stale after a step."""
    p = torch.nn.Parameter(torch.randn(8, device="cuda"))
    y = p.square().sum()
    p.grad = torch.ones_like(p)
    ops.AdamW([p]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


def test_refusals():
    c = _make((600, 40), (F, B), 8)
    A = ops.adamw_

    def no(text, **more):
        before = _clone(c)
        with pytest.raises(ValueError, match=text):
            A(**{**c, **more})
        assert all(x is None or torch.equal(x.float(), y.float()) for k in c for x, y in zip(c[k], before[k]))

    x, y = c["params"]
    no("no parameters", params=[])
    no("one tensor per parameter", grads=c["grads"][:1])
    no("must be contiguous", params=[torch.zeros(1200, device="cuda")[::2], y])
    no("device", grads=[c["grads"][0].cpu(), c["grads"][1]])
    no("shapes", grads=[c["grads"][0][:5], c["grads"][1]])
    no("int64", steps=[torch.tensor(1.0, device="cuda"), c["steps"][1]])
    no("float32 or bfloat16", params=[x.half(), y])
    no("both float32 or both", exp_avg=[c["exp_avg"][0].float(), c["exp_avg"][1]])
    no("need scales", scales=None)
    no("need scales", scales=[c["scales"][0][:, :1], c["scales"][1]])
    no("overlap", params=[x, x[:40]], grads=[c["grads"][0], c["grads"][1].float()])
    no("overlap", steps=[c["steps"][0]] * 2)
    no("overlap", grads=[x, c["grads"][1]])
    no("come together", max_norm=1.0)
    no("come together", grad_norm=torch.ones((), device="cuda"))
    no("one value", grad_norm=torch.ones(2, device="cuda"), max_norm=1.0)
    no("one value", lr=torch.ones((), device="cuda", dtype=torch.float64))
    no("max_norm", grad_norm=torch.ones((), device="cuda"), max_norm=float("nan"))
    for bad in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8), dict(weight_decay=-1.0), dict(lr=float("nan"))):
        no("lr=", **bad)
    z = x.detach().requires_grad_()
    no("leaves", params=[z * 1, y])
    with pytest.raises(RuntimeError, match="on the GPU"):
        A(*([t.cpu()] for t in (x, x, x, x, c["steps"][0])))
    for bad in (dict(lr=-1.0), dict(bits=4), dict(betas=(0.9, 1.0))):
        with pytest.raises(ValueError):
            ops.AdamW([torch.nn.Parameter(x)], **bad)
