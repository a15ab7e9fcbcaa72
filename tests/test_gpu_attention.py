"""cross_attention forward and backward against the definition in 64 bits.

The bounds follow from the arithmetic.  u = 2^-24 and r = 2^-8 (bf16 keeps 8 bits; u in f32) are
the rounding units of 32-bit sums and of outputs.  A score is a dot product of D
terms, so it is off by at most E = (D + 4) u scale max |q|.|k| in absolute terms, and a
probability by about 2 E + (Lk + 16) u in relative terms; products take probabilities
and score gradients rounded to the inputs' type (r), and the backward pass takes the
output as it was rounded (r).  Everything else is a sum of at most Lk or Lq * group
terms in 32 bits."""
import pytest
import torch

from tgengine_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _inputs(b, lq, lk, h, kv, d, dtype, seed=0, gain=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s):
        return (torch.randn(*s, generator=g, device="cuda") * gain).to(TYPES[dtype])

    return r(b, lq, h, d), r(b, lk, kv, d), r(b, lk, kv, d), r(b, lq, h, d)


def _mask(kind, b, lk, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if kind is None:
        return None
    if kind == "holes":
        m = torch.rand(b, lk, generator=g, device="cuda") < 0.5
        if b > 1:
            m[b // 2] = False  # a row that keeps nothing
        return m
    n = torch.randint(0, lk + 1, (b, 1), generator=g, device="cuda")
    n[0] = 0
    at = torch.arange(lk, device="cuda")
    return at >= lk - n if kind == "recent" else at < n


def _exact(q, k, v, g, mask, scale):
    """Outputs and gradients in 64 bits, and bounds on what 32-bit sums and one
    rounding of every product's operand may differ by."""
    b, lq, h, d = q.shape
    lk, kv = k.shape[1:3]
    r = U if q.dtype == torch.float32 else 2.0 ** -8

    def rows(x):
        return x.double().permute(0, 2, 1, 3).contiguous()

    def spread(x):
        return rows(x).repeat_interleave(h // kv, 1)

    def cols(x):
        return x.permute(0, 2, 1, 3)

    def shared(x):
        return x.reshape(b, kv, h // kv, lk, d).sum(2).permute(0, 2, 1, 3)

    keep = torch.ones(b, 1, 1, lk, device="cuda", dtype=torch.bool) if mask is None else mask[:, None, None, :]
    Q, K, V, G = rows(q), spread(k), spread(v), rows(g)
    K, V = (torch.where(keep[:, :, 0, :, None], x, 0.0) for x in (K, V))
    S = torch.where(keep, Q @ K.mT * scale, -torch.inf)
    m = S.amax(-1, keepdim=True) if lk else torch.full((b, h, lq, 1), -torch.inf, device="cuda", dtype=torch.float64)
    P = torch.exp(S - torch.where(m == -torch.inf, 0.0, m))
    P = P / P.sum(-1, keepdim=True).clamp_min(1e-300)
    O = P @ V
    delta = (G * O).sum(-1, keepdim=True)
    dP = G @ V.mT
    dS = P * (dP - delta) * scale
    E = (d + 4) * U * abs(scale) * ((Q.abs() @ K.abs().mT) * keep).amax(-1, keepdim=True) if lk else 0 * m
    rel = 2 * E + (lk + 16) * U
    eP = P * (rel + r)
    eS = P * abs(scale) * ((dP.abs() + delta.abs()) * rel + (d + 4) * U * (G.abs() @ V.abs().mT)
                           + (r + rel + (d + 4) * U) * (G.abs() * (P @ V.abs())).sum(-1, keepdim=True)) + dS.abs() * r
    n = (lq * (h // kv) + 8) * U
    out = {"out": (cols(O), cols(eP @ V.abs() + O.abs() * (r + U))),
           "dq": (cols(dS @ K), cols(eS @ K.abs() + (lk + 8) * U * (dS.abs() @ K.abs()) + (dS @ K).abs() * r)),
           "dk": (shared(dS.mT @ Q), shared(eS.mT @ Q.abs() + n * (dS.abs().mT @ Q.abs()))),
           "dv": (shared(P.mT @ G), shared(eP.mT @ G.abs() + n * (P.mT @ G.abs())))}
    return {x: (y, e + (y.abs() * r if x in ("dk", "dv") else 0) + 1e-30) for x, (y, e) in out.items()}


def _run(q, k, v, g, mask, scale=None):
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    o = ops.cross_attention(*leaves, mask=mask, scale=scale)
    return dict(zip(("out", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, leaves, g))))


def _check(q, k, v, g, mask, scale=None):
    got = _run(q, k, v, g, mask, scale)
    ref = _exact(q, k, v, g, mask, q.shape[-1] ** -0.5 if scale is None else scale)
    for name, (y, e) in ref.items():
        x = got[name]
        assert x.dtype == q.dtype and x.shape == y.shape, name
        off = (x.double() - y).abs()
        assert torch.isfinite(x.double()).all(), name
        assert bool((off <= e).all()), f"{name}: {float((off / e).max()):.3g} of the bound"
    with torch.no_grad():  # the same call without a gradient to keep
        assert torch.equal(ops.cross_attention(q, k, v, mask=mask, scale=scale), got["out"])
    return got


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("b,lq,lk,h,kv,d,mask", [
    (3, 1, 1, 1, 1, 1, None), (5, 1, 10, 2, 2, 50, "recent"), (7, 1, 32, 2, 2, 86, "holes"),
    (2, 1, 512, 2, 1, 172, "recent"), (3, 2, 20, 4, 2, 7, "prefix"), (4, 1, 33, 8, 1, 64, "holes"),
    (1, 4, 2100, 8, 2, 128, "prefix"), (2, 1, 3001, 2, 2, 100, "holes"), (3, 3, 700, 1, 1, 256, None),
    (5, 65, 65, 2, 2, 100, "recent"), (3, 33, 33, 2, 1, 50, "holes"), (2, 17, 129, 4, 2, 32, None),
    (2, 100, 31, 3, 3, 172, "prefix"), (1, 300, 257, 8, 2, 128, "holes"), (1, 64, 64, 4, 4, 64, None),
    (2, 130, 70, 2, 2, 255, "holes"), (1, 513, 1030, 4, 1, 96, "prefix"), (2, 16, 16, 1, 1, 16, "holes"),
    (1, 40, 300, 16, 1, 33, "recent")])
def test_against_64_bits(b, lq, lk, h, kv, d, mask, dtype):
    _check(*_inputs(b, lq, lk, h, kv, d, dtype), _mask(mask, b, lk))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("b,lq,lk", [(0, 3, 4), (2, 0, 4), (2, 3, 0), (2, 1, 0), (3, 70, 0)])
def test_lengths_of_zero(b, lq, lk, dtype):
    q, k, v, g = _inputs(b, lq, lk, 2, 1, 24, dtype)
    got = _run(q, k, v, g, None)
    for name, like in (("out", q), ("dq", q), ("dk", k), ("dv", v)):
        assert got[name].shape == like.shape and not got[name].any(), name


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lq,lk,d", [(1, 40, 50), (3, 900, 64), (70, 90, 100), (65, 300, 128)])
def test_masked_places_hold_anything(lq, lk, d, dtype):
    """NaN, infinities and the type's lowest value behind the mask change nothing, and take a gradient of zero."""
    q, k, v, g = _inputs(4, lq, lk, 4, 2, d, dtype)
    mask = _mask("holes", 4, lk)
    clean = _run(q, k, v, g, mask)
    for x in (float("nan"), float("inf"), float("-inf"), torch.finfo(TYPES[dtype]).min):
        off = ~mask[:, :, None, None]
        dirty = _run(q, torch.where(off, x, k).to(k.dtype), torch.where(off, x, v).to(v.dtype), g, mask)
        for name in clean:
            assert torch.equal(clean[name], dirty[name]), (x, name)
    assert not clean["dk"][~mask].any() and not clean["dv"][~mask].any()
    none = ~mask.any(1)
    assert none.any() and not clean["out"][none].any() and not clean["dq"][none].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lq,lk", [(1, 30), (1, 1500), (40, 100)])
def test_large_scores(lq, lk, dtype):
    """Scores of hundreds: one key takes all, and the running maximum moves late."""
    q, k, v, g = _inputs(3, lq, lk, 2, 2, 64, dtype, gain=1.0)
    ramp = torch.linspace(0.1, 20, lk, device="cuda")[None, :, None, None]
    _check(q, (k * ramp).to(k.dtype), v, g, _mask("holes", 3, lk), scale=0.6)
    _check(q, (k * ramp.flip(1)).to(k.dtype), v, g, None, scale=-0.6)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lq,lk,d", [(1, 21, 50), (2, 1300, 86), (65, 65, 100), (66, 140, 128)])
def test_strides_and_alignment(lq, lk, d, dtype):
    """Inputs in other layouts give the bits of contiguous ones."""
    b, h, kv = 3, 4, 2
    q, k, v, g = _inputs(b, lq, lk, h, kv, d, dtype)
    mask = _mask("holes", b, lk)
    want = _run(q, k, v, g, mask)
    both = torch.stack([k, v], 2)  # one projection's keys and values
    heads = [x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (q, k, v)]
    wide = torch.full((b, lk, kv, d + 5), float("nan"), device="cuda", dtype=k.dtype)
    wide[..., 3:3 + d] = k
    odd = torch.empty(q.numel() + 1, device="cuda", dtype=q.dtype)[1:].view(q.shape)
    odd.copy_(q)
    last = [x.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0) for x in (q, k, v)]  # last dimension not dense
    padded = torch.cat([mask, mask], 1)[:, :lk]
    for layout in ((q, both[:, :, 0], both[:, :, 1], mask), (*heads, mask), (odd, wide[..., 3:3 + d], v, padded),
                   (*last, mask.t().contiguous().t())):
        got = _run(*layout[:3], g, layout[3])
        for name in want:
            assert torch.equal(got[name], want[name]), name
    gs = torch.stack([g, g], -1)[..., 0]  # a gradient that is not contiguous
    assert torch.equal(_run(q, k, v, gs, mask)["dk"], want["dk"])


@pytest.mark.parametrize("lq", [1, 48])
def test_broadcast_inputs(lq):
    """One sequence of states for all batch rows: its gradient is the sum over them."""
    b, lk, h, kv, d = 6, 50, 4, 2, 64
    q, k, v, g = _inputs(b, lq, lk, h, kv, d, "f32")
    mask = _mask("holes", 1, lk).expand(b, lk)
    k1, v1 = k[:1].clone().requires_grad_(), v[:1].clone().requires_grad_()
    o = ops.cross_attention(q, k1.expand(b, -1, -1, -1), v1.expand(b, -1, -1, -1), mask=mask)
    dk, dv = torch.autograd.grad(o, (k1, v1), g)
    ref = _exact(q, k[:1].expand(b, -1, -1, -1), v[:1].expand(b, -1, -1, -1), g, mask, d ** -0.5)
    for x, name in ((o, "out"), (dk, "dk"), (dv, "dv")):
        y, e = ref[name]
        if name != "out":
            y, e = y.sum(0, keepdim=True), e.sum(0, keepdim=True) + 8 * U * y.abs().sum(0, keepdim=True)
        assert bool(((x.double() - y).abs() <= e).all()), name


@pytest.mark.parametrize("lq,lk", [(1, 37), (50, 70), (2, 2000)])
def test_partial_gradients(lq, lk):
    """Only the asked-for gradients, with the bits of the full backward pass."""
    q, k, v, g = _inputs(3, lq, lk, 4, 2, 72, "bf16")
    mask = _mask("recent", 3, lk)
    want = _run(q, k, v, g, mask)
    for ask in ("q", "k", "v", "kv", "qv"):
        x = {n: t.detach().requires_grad_(n in ask) for n, t in (("q", q), ("k", k), ("v", v))}
        o = ops.cross_attention(x["q"], x["k"], x["v"], mask=mask)
        for n, d in zip(ask, torch.autograd.grad(o, [x[n] for n in ask], g)):
            assert torch.equal(d, want["d" + n]), (ask, n)


@pytest.mark.parametrize("lq,lk,d", [(1, 20, 30), (30, 40, 64), (1, 1200, 50)])
def test_gradient_against_differences(lq, lk, d):
    """Central differences of the forward kernel along random directions.  With steps of
    h = 2^-7 the third derivative leaves about h^2, and 32-bit outputs about u / h, of the
    sum of |output * dout|; 2^-9 of it holds both with room."""
    q, k, v, g = _inputs(2, lq, lk, 4, 2, d, "f32", seed=5)
    mask = _mask("holes", 2, lk, seed=9)
    got = _run(q, k, v, g, mask)
    dirs = _inputs(2, lq, lk, 4, 2, d, "f32", seed=6)[:3]
    h = 2.0 ** -7
    with torch.no_grad():
        size = (got["out"].double() * g.double()).abs().sum()
        for i, name in enumerate(("dq", "dk", "dv")):
            step = dirs[i] / dirs[i].norm() * 4
            f = [(ops.cross_attention(*[x + s * step if j == i else x for j, x in enumerate((q, k, v))], mask=mask)
                  .double() * g.double()).sum() for s in (h, -h)]
            slope = (got[name].double() * step.double()).sum()
            assert abs((f[0] - f[1]) / (2 * h) - slope) <= size * 2.0 ** -9, name


def test_long_caches_pass_32_bits():
    """Keys whose element offsets pass 2^31, in a cache of 4.4 GB."""
    step, lk, d = 60_000_000, 37, 64
    cache = torch.empty(step * lk, device="cuda", dtype=torch.bfloat16)
    k = torch.as_strided(cache, (1, lk, 1, d), (step * lk, step, d, 1))
    v = torch.as_strided(cache, (1, lk, 1, d), (step * lk, step, d, 1), storage_offset=128)
    for lq in (1, 50):
        q, k0, v0, g = _inputs(1, lq, lk, 2, 1, d, "bf16")
        k.copy_(k0)
        v.copy_(v0)
        assert torch.equal(_run(q, k, v, g, None)["dk"], _run(q, k0, v0, g, None)["dk"])
        assert torch.equal(ops.cross_attention(q, k, v), ops.cross_attention(q, k0, v0))


def test_other_streams_and_repeats():
    """Work queued on the caller's stream, and the same bits on every call."""
    q, k, v, g = _inputs(8, 33, 400, 4, 2, 100, "bf16")
    q1, k1, v1, g1 = _inputs(8, 1, 3000, 4, 2, 100, "bf16")
    want, want1 = _run(q, k, v, g, None), _run(q1, k1, v1, g1, None)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(4):
            big = big @ big * 1e-2
        late = [x.clone() for x in (q, k, v, g)]  # ready only after the products
        got, got1 = _run(*late, None), _run(q1, k1, v1, g1, None)
    torch.cuda.current_stream().wait_stream(side)
    for name in want:
        assert torch.equal(got[name], want[name]) and torch.equal(got1[name], want1[name]), name


def test_graph_replays():
    """Captured forward and backward calls, replayed between eager work."""
    q, k, v, g = _inputs(4, 20, 90, 4, 2, 64, "bf16")
    q1, k1, v1, _ = _inputs(2, 1, 2500, 4, 2, 64, "bf16")
    _run(q, k, v, g, None), ops.cross_attention(q1, k1, v1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, got1 = _run(q, k, v, g, None), ops.cross_attention(q1, k1, v1)
    for n in range(3):
        with torch.no_grad():
            for x, y in ((q, 1), (k, 2), (v, 3), (g, 4), (q1, 5), (k1, 6)):
                x.copy_(_inputs(*x.shape[:2], 1, *x.shape[2:3], 1, x.shape[3], "bf16", seed=10 * n + y)[0].reshape(x.shape))
        graph.replay()
        torch.cuda.synchronize()
        want = _run(q, k, v, g, None)
        for name in want:
            assert torch.equal(got[name], want[name]), (n, name)
        assert torch.equal(got1, ops.cross_attention(q1, k1, v1))


def test_refusals():
    q, k, v, g = _inputs(2, 3, 5, 4, 2, 16, "f32")
    A = ops.cross_attention
    for args, text in (((q, k, v[:, :4]), "same shape"), ((q, k[:1], v[:1]), "batch or dim"),
                       ((q[..., :8], k, v), "batch or dim"), ((q[:, :, :3], k, v), "multiple"),
                       ((q.bfloat16(), k, v), "same dtype"), ((q.half(), k.half(), v.half()), "float32 or bfloat16"),
                       ((q[0], k[0], v[0]), r"\(batch, tokens, heads, dim\)"),
                       ((q, k, v, torch.ones(2, 4, device="cuda", dtype=torch.bool)), "mask must be"),
                       ((q, k, v, torch.ones(2, 5, device="cuda")), "mask must be bool"),
                       ((q, k, v, torch.ones(2, 5, dtype=torch.bool)), "device"),
                       ((q.repeat(1, 1, 1, 17), k.repeat(1, 1, 1, 17), v.repeat(1, 1, 1, 17)), "1 to 256")):
        with pytest.raises(ValueError, match=text):
            A(*args)
    with pytest.raises(RuntimeError, match="on the GPU"):
        A(q.cpu(), k.cpu(), v.cpu())
    leaf = q.detach().requires_grad_()
    with pytest.raises(RuntimeError, match="once only"):
        torch.autograd.grad(A(leaf, k, v).sum(), leaf, create_graph=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("b,lq,lk,h,kv,d,mask", [(1, 300, 500, 4, 2, 64, "holes"), (3, 40, 70, 2, 2, 100, "recent"),
                                                 (1, 2000, 60, 2, 1, 112, "holes"), (1, 90, 2600, 3, 3, 176, "prefix")])
def test_gradients_one_at_a_time(b, lq, lk, h, kv, d, mask, dtype):
    """Each gradient asked for alone, within the bounds of the whole backward pass: few
    workgroups, whose rows and keys are cut in ranges, and f32 without kept scores."""
    q, k, v, g = _inputs(b, lq, lk, h, kv, d, dtype, seed=3)
    m = _mask(mask, b, lk, seed=4)
    ref = _exact(q, k, v, g, m, d ** -0.5)
    for name in "qkv":
        x = {n: t.detach().requires_grad_(n == name) for n, t in (("q", q), ("k", k), ("v", v))}
        (got,) = torch.autograd.grad(ops.cross_attention(x["q"], x["k"], x["v"], mask=m), x[name], g)
        y, e = ref["d" + name]
        assert bool(((got.double() - y).abs() <= e).all()), name


@pytest.mark.parametrize("lk", [1, 2, 6, 40, 64, 65, 128])
@pytest.mark.parametrize("lq,group,d", [(33, 1, 64), (40, 2, 40), (7, 1, 32)])
def test_few_keys_round_the_output_only(lk, lq, group, d):
    """bf16 with few keys: probabilities keep 16 bits (what their rounding to 2^-8 took is
    rounded to 2^-8 of itself), so that the output is off by its own rounding, 2^-8, and by
    2^-16 of the sum of p |v|.  A score's 32-bit sum of d <= 64 products whose magnitudes
    add up to less than 24 is off by less than 64 x 2^-24 x 24 < 2^-13, which moves its
    probability, and the sum of all, by as much: 2^-11 of the sum of p |v| covers both."""
    q, k, v, _ = _inputs(5, lq, lk, 2 * group, 2, d, "bf16", seed=lk)
    m = _mask("holes", 5, lk, seed=lk)
    zero = torch.zeros_like(q)
    y = _exact(q, k, v, zero, m, d ** -0.5)["out"][0]
    spread = _exact(q, k, v.abs(), zero, m, d ** -0.5)["out"][0]
    got = ops.cross_attention(q, k, v, mask=m)
    assert bool(((got.double() - y).abs() <= 2.0 ** -8 * y.abs() + 2.0 ** -11 * spread).all())
