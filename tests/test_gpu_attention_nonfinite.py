"""cross_attention where inputs are NaN or infinite: they reach what the formulas lead them to and nothing else."""
import pytest
import torch

from tgengine_amd import ops

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")
# (lq, lk, d) with 2 heads a key/value head: few rows, cut keys, matrix units, f32 kept scores and without, wide heads
SHAPES = [(1, 40, 50), (2, 900, 64), (1, 3000, 172), (70, 90, 100), (65, 300, 128), (40, 3000, 64), (20, 70, 200)]
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _inputs(lq, lk, d, dtype, seed=0):
    """q, k, v, g and a mask with holes; batch row 2 keeps no key."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = [torch.randn(*s, generator=g, device="cuda").to(TYPES[dtype])
         for s in ((4, lq, 4, d), (4, lk, 2, d), (4, lk, 2, d), (4, lq, 4, d))]
    mask = torch.rand(4, lk, generator=g, device="cuda") < 0.5
    mask[:, lk // 3] = True
    mask[2] = False
    return *x, mask


def _run(q, k, v, g, mask):
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    o = ops.cross_attention(*leaves, mask=mask)
    return dict(zip(("out", "dq", "dk", "dv"), (o.detach(), *torch.autograd.grad(o, leaves, g))))


def _same_but(got, want, nan):
    """``got`` is NaN where ``nan`` says (a mask for each output), and elsewhere has ``want``'s bits."""
    for name, x in got.items():
        at = nan.get(name, torch.zeros((), device="cuda", dtype=torch.bool)).expand(x.shape)
        assert bool(x[at].isnan().all()), name
        assert torch.equal(x[~at], want[name][~at]), name


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lq,lk,d", SHAPES)
def test_rows_without_keys_hold_anything(lq, lk, d, dtype):
    """Queries and gradients of a batch row whose mask is empty change nothing."""
    q, k, v, g, mask = _inputs(lq, lk, d, dtype)
    want = _run(q, k, v, g, mask)
    for x in (NAN, INF, -INF):
        for which in ("q", "g", "qg"):
            q1, g1 = q.clone(), g.clone()
            if "q" in which:
                q1[2] = x
            if "g" in which:
                g1[2] = x
            got = _run(q1, k, v, g1, mask)
            _same_but(got, want, {})
            assert not any(got[n][2].any() for n in got)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lq,lk,d", SHAPES)
def test_masked_keys_take_no_gradient(lq, lk, d, dtype):
    """A gradient of NaN in one row reaches the kept keys of its batch row and head, and no masked key."""
    q, k, v, g, mask = _inputs(lq, lk, d, dtype)
    want = _run(q, k, v, g, mask)
    g[1, lq - 1, 0] = NAN
    row = torch.zeros(4, lq, 4, 1, device="cuda", dtype=torch.bool)
    row[1, lq - 1, 0] = True
    keys = torch.zeros(4, lk, 2, 1, device="cuda", dtype=torch.bool)
    keys[1, :, 0, 0] = mask[1]
    _same_but(_run(q, k, v, g, mask), want, {"dq": row, "dk": keys, "dv": keys})


def _spread(q, mask, lq, lk, rows):
    """What a score of NaN in ``rows`` of batch row 1 and head 0 reaches."""
    row = torch.zeros(4, lq, 4, 1, device="cuda", dtype=torch.bool)
    row[1, rows, 0] = True
    keys = torch.zeros(4, lk, 2, 1, device="cuda", dtype=torch.bool)
    keys[1, :, 0, 0] = mask[1]
    return {"out": row, "dq": row, "dk": keys, "dv": keys}


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lq,lk,d", SHAPES)
def test_scores_of_nan(lq, lk, d, dtype):
    """A NaN query makes all its probabilities NaN, so out and dq of its row and dk and dv of
    every kept key of its head; a NaN key does so for every row of its head."""
    q, k, v, g, mask = _inputs(lq, lk, d, dtype)
    want = _run(q, k, v, g, mask)
    q1 = q.clone()
    q1[1, lq - 1, 0, d // 2] = NAN
    _same_but(_run(q1, k, v, g, mask), want, _spread(q, mask, lq, lk, lq - 1))
    k1 = k.clone()
    k1[1, lk // 3, 0, 0] = NAN
    nan = _spread(q, mask, lq, lk, slice(None))
    for name in ("out", "dq"):
        nan[name][1, :, 1] = True  # the head's second query head
    _same_but(_run(q, k1, v, g, mask), want, nan)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lq,lk,d", SHAPES)
def test_scores_of_infinity(lq, lk, d, dtype):
    """A score of +inf: exp(inf - inf) is NaN, and so is the row's sum."""
    q, k, v, g, mask = _inputs(lq, lk, d, dtype)
    k[1, lk // 3, 0, 0] = 2.0
    want = _run(q, k, v, g, mask)
    q[1, lq - 1, 0] = 0.0
    q[1, lq - 1, 0, 0] = INF
    k1 = k.clone()
    k1[1, mask[1], 0, 0] = k1[1, mask[1], 0, 0].abs() + 1.0  # all of the row's scores are +inf or masked
    for keys in (k, k1):
        got = _run(q, keys, v, g, mask)
        assert got["out"][1, lq - 1, 0].isnan().all() and got["dq"][1, lq - 1, 0].isnan().all()
        assert got["dv"][1, mask[1], 0].isnan().all() and not got["dv"][1, ~mask[1]].any()
        for n in got:
            assert torch.equal(got[n][[0, 2, 3]], want[n][[0, 2, 3]]), n


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lq,lk,d", SHAPES)
@pytest.mark.parametrize("x", [INF, -INF])
def test_infinite_values_and_gradients(lq, lk, d, dtype, x):
    """An infinite value at a kept key gives infinite outputs in its column, an infinite
    gradient infinite dv in its: a probability above zero times an infinity is that infinity."""
    q, k, v, g, mask = _inputs(lq, lk, d, dtype)
    want = _run(q, k, v, g, mask)
    v1, g1 = v.clone(), g.clone()
    v1[1, lk // 3, 0, 3] = x
    g1[1, lq - 1, 0, 2] = x
    out, dv = _run(q, k, v1, g, mask)["out"], _run(q, k, v, g1, mask)["dv"]
    assert bool((out[1, :, :2, 3] == x).all()) and bool((dv[1, mask[1], 0, 2] == x).all())
    out[1, :, :2, 3] = want["out"][1, :, :2, 3]
    dv[1, mask[1], 0, 2] = want["dv"][1, mask[1], 0, 2]
    assert torch.equal(out, want["out"]) and torch.equal(dv, want["dv"])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lq,lk,d", SHAPES)
def test_infinite_score_gradients(lq, lk, d, dtype):
    """With a value of +inf and gradients above zero, out . dout is +inf and so every other
    kept key's score gradient -inf; queries above zero take it to a dk of -inf."""
    q, k, v, g, mask = _inputs(lq, lk, d, dtype)
    q, g = q.abs() + 2.0 ** -4, g.abs() + 2.0 ** -4
    v[1, lk // 3, 0, 3] = INF
    dk = _run(q, k, v, g, mask)["dk"]
    other = mask[1].clone()
    other[lk // 3] = False
    assert bool((dk[1, other, 0] == -INF).all()) and dk[1, lk // 3, 0].isnan().all() and not dk[1, ~mask[1]].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lq,lk,d", SHAPES)
def test_zeros_stay_zeros(lq, lk, d, dtype):
    """A row whose gradient is zero has a dq of zero, and where all rows' are, so are dk and dv."""
    q, k, v, g, mask = _inputs(lq, lk, d, dtype)
    g[0] = 0.0
    g[1, lq - 1, 0] = 0.0
    g[3, :, 2:] = 0.0
    got = _run(q, k, v, g, mask)
    assert not got["dq"][0].any() and not got["dk"][0].any() and not got["dv"][0].any()
    assert not got["dq"][1, lq - 1, 0].any() and not got["dk"][3, :, 1].any() and not got["dv"][3, :, 1].any()
    zero = _run(q, k, torch.zeros_like(v), g, mask)
    assert not zero["out"].any() and not zero["dq"].any() and not zero["dk"].any()
