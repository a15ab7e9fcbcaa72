"""gated_scan's branches for long rows of few channels and for tensors that reach past 4 GiB.

Long rows: 64 or 72 tokens a piece where channels are few, so 40,000 tokens are 625 pieces and 25,000 are 348.  Up to
256 pieces each of the 32 threads that join them keeps its pieces in registers; beyond, as here, they are read twice.
The recurrences are taken in 64 bits by spans of doubled length, for values, absolute sums and errors alike.

Past 4 GiB offsets are of 64 bits: a batch stride of 2^33 that nothing reads takes that branch, and so do rows that far
apart and outputs that large.  Both branches do the same arithmetic, so their bits are compared."""
import pytest
import torch

from tgengine_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F, B = torch.float32, torch.bfloat16
FAR = 1 << 33


def _case(shape, dtype, mask=None, state=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    b, n, d = shape

    def r(*s):
        return torch.randn(*s, generator=g, device="cuda")

    c = {"x": r(b, n, d).to(dtype), "gate": (r(b, n, d) * 2).to(dtype), "state": r(b, d) if state else None, "mask": None,
         "grads": (r(b, n, d).to(dtype), r(b, d))}
    if mask == "holes":
        c["mask"] = torch.rand(b, n, generator=g, device="cuda") < 0.6
    elif mask == "recent":
        c["mask"] = torch.arange(n, device="cuda") >= n - torch.randint(n // 2, n, (b, 1), generator=g, device="cuda")
    return c


def _run(c):
    leaves = {n: c[n].detach().requires_grad_() for n in ("x", "gate", "state") if c[n] is not None}
    out, last = ops.gated_scan(leaves["x"], leaves["gate"], c["mask"], leaves.get("state"))
    d = torch.autograd.grad((out, last), list(leaves.values()), c["grads"])
    return {"out": out.detach(), "last": last.detach(), **dict(zip(leaves, d))}


def _along(a, b):
    """v_t = a_t v_{t-1} + b_t along dimension 1 from 0."""
    off = 1
    while off < b.shape[1]:
        b = torch.cat([b[:, :off], b[:, off:] + a[:, off:] * b[:, :-off]], 1)
        a = torch.cat([a[:, :off], a[:, off:] * a[:, :-off]], 1)
        off *= 2
    return b


def _exact(c):
    """{name: (value, bound)}: a gate is off by s = (2 |gate| + 6) u, a token adds (s + 3 u) of the absolute sum to the
    error, and what is there shrinks by the gate; outputs are rounded once."""
    x, gate, (gout, glast) = c["x"].double(), c["gate"].double(), c["grads"]
    b, n, d = x.shape
    r = U if c["x"].dtype == F else 2.0 ** -8
    keep = (torch.ones(b, n, device="cuda", dtype=torch.bool) if c["mask"] is None else c["mask"])[..., None]
    x, gate = torch.where(keep, x, 0.0), torch.where(keep, gate, 0.0)
    a, rest = torch.where(keep, torch.sigmoid(gate), 1.0), torch.where(keep, torch.sigmoid(-gate), 0.0)
    s = torch.where(keep, (2 * gate.abs() + 6) * U, 0.0)
    h0 = torch.zeros(b, 1, d, device="cuda", dtype=torch.float64) if c["state"] is None else c["state"].double()[:, None]

    def ahead(first, terms):  # from the value before the first token
        return _along(a, torch.cat([a[:, :1] * first + terms[:, :1], terms[:, 1:]], 1))

    h, m = ahead(h0, rest * x), ahead(h0.abs(), rest * x.abs())
    e = ahead(torch.zeros_like(h0), (s + 3 * U) * m)
    old, eold = torch.cat([h0, h[:, :-1]], 1), torch.cat([torch.zeros_like(h0), e[:, :-1]], 1)
    out = {"out": (h, e + r * h.abs()), "last": (h[:, -1], e[:, -1] + U * h[:, -1].abs())}

    def back(terms, last):  # dh_t = terms_t + a_{t+1} dh_{t+1}
        after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
        terms = torch.cat([terms[:, :-1], terms[:, -1:] + last], 1)
        return _along(after.flip(1), terms.flip(1)).flip(1)

    g, last = gout.double(), glast.double()[:, None]
    dh, dm = back(g, last), back(g.abs(), last.abs())
    nxt = torch.cat([(a * (s + 3 * U) * dm)[:, 1:], torch.zeros_like(dm[:, :1])], 1)  # what a token passes on, at its left
    de = back(2 * U * dm + nxt, torch.zeros_like(last))
    off = old - x
    v, w = dh * rest, dh * a * rest * off
    out["x"] = v, de * rest + v.abs() * (s + 2 * U + r)
    out["gate"] = w, (de * rest * a * off.abs() + dh.abs() * rest * a * (eold + U * off.abs())
                      + w.abs() * (2 * s + 4 * U + r))
    z = a[:, 0] * dh[:, 0]
    out["state"] = z, a[:, 0] * (de[:, 0] + (s[:, 0] + 3 * U) * dm[:, 0]) + U * z.abs()
    return out


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("mask", [None, "holes", "recent"])
@pytest.mark.parametrize("shape", [(1, 40_000, 2), (3, 25_000, 5), (2, 19_001, 1)])
def test_more_pieces_than_registers_hold(shape, mask, dtype):
    for state in (True, False):
        c = _case(shape, dtype, mask, state)
        got, want = _run(c), _exact(c)
        for name, t in got.items():
            y, e = want[name]
            off, e = (t.double() - y).abs(), 1.01 * e + 1e-37
            assert bool((off <= e).all()), f"{name}: {float((off / e).max()):.3g} of the bound"
        again = _run(c)
        assert all(torch.equal(again[n], got[n]) for n in got)
        with torch.no_grad():
            out, last = ops.gated_scan(c["x"], c["gate"], c["mask"], c["state"])
        assert torch.equal(out, got["out"]) and torch.equal(last, got["last"])


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("mask", [None, "holes"])
@pytest.mark.parametrize("shape", [(1, 1, 172), (1, 45, 7), (1, 3, 1), (1, 1000, 6), (1, 1001, 1), (1, 20_000, 3)])
def test_far_strides(shape, mask, dtype):
    """A batch stride past 4 GiB, of x, of the gate and of both: one piece, several and many."""
    for state in (True, False):
        c = _case(shape, dtype, mask, state)
        want = _run(c)
        for names in (("x",), ("gate",), ("x", "gate")):
            d = {**c, **{k: c[k].as_strided(shape, (FAR, shape[2], 1)) for k in names}}
            assert all(d[k].stride(0) == FAR for k in names)
            got = _run(d)
            assert all(torch.equal(got[k], want[k]) for k in want)
            with torch.no_grad():
                out, last = ops.gated_scan(d["x"], d["gate"], d["mask"], d["state"])
            assert torch.equal(out, want["out"]) and torch.equal(last, want["last"])


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("shape", [(2, 37, 50), (2, 700, 5)])
def test_rows_far_apart(shape, dtype):
    """Rows 4 GiB and some bytes apart, and tokens a MiB apart, in one storage of x and gate."""
    c = _case(shape, dtype, "holes")
    want = _run(c)
    b, n, d = shape
    size = 4 if dtype == F else 2
    row, token = (1 << 32) // size + 24, (1 << 20) // size + 8
    room = torch.empty(row + (2 * n + 2) * token, device="cuda", dtype=dtype)
    far = {}
    for i, k in enumerate(("x", "gate")):
        far[k] = room.as_strided(shape, (row, token, 1), i * (n + 1) * token)
        far[k].copy_(c[k])
    got = _run({**c, **far})
    assert all(torch.equal(got[k], want[k]) for k in want)


def test_outputs_past_4_gib():
    """16,500 rows of 512 tokens and 256 bf16 channels, one row broadcast, against 300 of them: enough for rows in one
    piece, and every row gives the same bits."""
    b, n, d = 16_500, 512, 256
    c = _case((1, n, d), B, "holes")
    assert b * n * d * 2 > 1 << 32

    def rows(k):
        return {**{n: v.expand(k, *v.shape[1:]) for n, v in c.items() if isinstance(v, torch.Tensor)},
                "grads": tuple(g.expand(k, *g.shape[1:]) for g in c["grads"])}

    want = {k: t[:1].clone() for k, t in _run(rows(300)).items()}
    for k, t in _run(rows(b)).items():
        for part in t.split(1000):
            assert torch.equal(part, want[k].expand_as(part)), k
