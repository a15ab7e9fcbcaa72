"""bf16 cross_attention rounds outputs and gradients once, however many keys there are and
however many of them the mask keeps.

Matrix products take probabilities and score gradients in two parts, bf16 and what rounding
to it took, and the gradient takes the output likewise: r = 2^-8 of what r took, so s = 2^-16
of the value is left out.  Results add their own rounding, r.  Scores, sums and exponentials are of 32 bits, u = 2^-24: a score is off by at most
E = (D + 4) u scale max |q|.|k|, a probability by 2 E + (Lk + 16) u relatively."""
import pytest
import torch

from tgengine_amd import ops

pytestmark = pytest.mark.gpu
U, R, S = 2.0 ** -24, 2.0 ** -8, 2.0 ** -16


def _inputs(b, lq, lk, h, kv, d, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(*s, generator=g, device="cuda").bfloat16()
            for s in ((b, lq, h, d), (b, lk, kv, d), (b, lk, kv, d), (b, lq, h, d))]


def _few(b, lk, most, seed):
    """A mask that keeps 1 to ``most`` keys of a row, anywhere, and none of the last row's; all keys for most = 0."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    if most == 0:
        return None
    order = torch.rand(b, lk, generator=g, device="cuda").argsort(1)
    mask = order < torch.randint(1, most + 1, (b, 1), generator=g, device="cuda")
    mask[-1] = False
    return mask


def _exact(q, k, v, g, mask):
    """{name: (value, bound)} in 64 bits."""
    b, lq, h, d = q.shape
    lk, kv = k.shape[1:3]
    scale = d ** -0.5

    def rows(x):
        return x.double().permute(0, 2, 1, 3).contiguous()

    def cols(x):
        return x.permute(0, 2, 1, 3)

    keep = torch.ones(b, 1, 1, lk, device="cuda", dtype=torch.bool) if mask is None else mask[:, None, None, :]
    Q, K, V = rows(q), *(rows(x).repeat_interleave(h // kv, 1) for x in (k, v))
    sc = torch.where(keep, Q @ K.mT * scale, -torch.inf)
    m = sc.amax(-1, keepdim=True)
    P = torch.exp(sc - torch.where(m == -torch.inf, 0.0, m))
    P = P / P.sum(-1, keepdim=True).clamp_min(1e-300)
    O = P @ V
    E = (d + 4) * U * scale * ((Q.abs() @ K.abs().mT) * keep).amax(-1, keepdim=True)
    rel = 2 * E + (lk + 16) * U
    eP = P * (rel + S)
    out = {"out": (cols(O), cols(eP @ V.abs() + O.abs() * (R + U)))}
    if g is None:
        return out
    G = rows(g)
    delta = (G * O).sum(-1, keepdim=True)
    dP = torch.where(keep, G @ V.mT, 0.0)
    dS = P * (dP - delta) * scale
    dot = (d + 4) * U  # a product's or delta's own sum of d terms
    eS = P * scale * ((dP.abs() + delta.abs()) * rel + dot * (G.abs() @ V.abs().mT)
                      + (S + rel + dot) * (G.abs() * (P @ V.abs())).sum(-1, keepdim=True)) + dS.abs() * S
    n = (lq * (h // kv) + 8) * U

    def shared(x):
        return x.reshape(b, kv, h // kv, lk, d).sum(2).permute(0, 2, 1, 3)

    dq, dk, dv = cols(dS @ K), shared(dS.mT @ Q), shared(P.mT @ G)
    out["dq"] = dq, cols(eS @ K.abs() + (lk + 8) * U * (dS.abs() @ K.abs())) + dq.abs() * R
    out["dk"] = dk, shared(eS.mT @ Q.abs() + n * (dS.abs().mT @ Q.abs())) + dk.abs() * R
    out["dv"] = dv, shared(eP.mT @ G.abs() + n * (P.mT @ G.abs())) + dv.abs() * R
    return out


def _check(got, ref):
    for name, (y, e) in ref.items():
        off = (got[name].double() - y).abs()
        assert bool((off <= e + 1e-30).all()), f"{name}: {float((off / (e + 1e-30)).max()):.3g} of the bound"


SHAPES = [(33, 1, 64), (40, 2, 40), (7, 1, 100), (1, 8, 128), (130, 1, 96), (20, 2, 256)]


@pytest.mark.parametrize("lk,most", [(129, 2), (300, 8), (1000, 1), (1000, 8), (5000, 3), (129, 0), (300, 0), (1100, 0)])
@pytest.mark.parametrize("lq,group,d", SHAPES)
def test_output(lq, group, d, lk, most):
    q, k, v, g = _inputs(3, lq, lk, 2 * group, 2, d, lk + most)
    mask = _few(3, lk, most, lk)
    _check({"out": ops.cross_attention(q, k, v, mask=mask)}, _exact(q, k, v, None, mask))


@pytest.mark.parametrize("lk,most", [(6, 2), (64, 0), (129, 2), (300, 8), (1000, 1), (5000, 3), (300, 0), (1100, 0)])
@pytest.mark.parametrize("lq,group,d", SHAPES)
def test_gradients(lq, group, d, lk, most):
    q, k, v, g = _inputs(3, lq, lk, 2 * group, 2, d, lk + most)
    mask = _few(3, lk, most, lk)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    o = ops.cross_attention(*leaves, mask=mask)
    got = dict(zip(("out", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, leaves, g))))
    with torch.no_grad():
        _check(got, _exact(q, k, v, g, mask))


def test_padding_changes_nothing():
    """The same kept keys, padded by 2 or by 300 masked ones: the same bits."""
    q, k, v, _ = _inputs(4, 40, 30, 4, 2, 64, 7)
    keep = torch.ones(4, 30, device="cuda", dtype=torch.bool)
    want = ops.cross_attention(q, k, v)
    for pad in (2, 98, 99, 300):
        kp, vp = (torch.cat([x, torch.full_like(x[:, :1].expand(-1, pad, -1, -1), float("nan"))], 1) for x in (k, v))
        mask = torch.cat([keep, torch.zeros(4, pad, device="cuda", dtype=torch.bool)], 1)
        assert torch.equal(ops.cross_attention(q, kp, vp, mask=mask), want), pad
