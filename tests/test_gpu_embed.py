"""embed: lookup bit for bit, gradient against sums in 64 bits.

A gradient row is a sum of c terms in 32 bits, in any order off by at most
c u sum |g| before the scale (one more rounding) and the output's rounding r
(u = 2^-24; r = u in f32 and 2^-8 in bf16, which keeps 8 bits)."""
import numpy as np
import pytest
import torch

from tgengine_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _case(n, dim, shape, dtype, seed, skew=1.0, ids_dtype=torch.int32):
    rng = np.random.default_rng(seed)
    count = int(np.prod(shape))
    ids = np.minimum((n * rng.random(count) ** (1 + 4 * skew)).astype(np.int64), max(n - 1, 0))
    bad = rng.random(count)
    ids[bad < 0.2] = -1
    ids[(bad >= 0.2) & (bad < 0.22)] = n
    ids[(bad >= 0.22) & (bad < 0.23)] = n + 12345
    ids[(bad >= 0.23) & (bad < 0.24)] = -(2 ** 31)
    g = torch.Generator(device="cuda").manual_seed(seed)
    table = torch.randn(n, dim, generator=g, device="cuda").to(dtype)
    dout = torch.randn(*shape, dim, generator=g, device="cuda").to(dtype)
    return table, torch.from_numpy(ids).to(ids_dtype).cuda().reshape(shape), dout


def _check(table, ids, dout, scale):
    n, dim = table.shape
    leaf = table.detach().requires_grad_()
    out = ops.embed(leaf, ids, scale=scale)
    ok = (ids >= 0) & (ids.long() < n)
    at = torch.where(ok, ids.long(), 0)
    if n:
        want = torch.where(ok[..., None], (table.float()[at] * scale), 0.0).to(table.dtype)
        assert torch.equal(out, want)
    assert out.shape == (*ids.shape, dim) and out.dtype == table.dtype
    with torch.no_grad():
        assert torch.equal(ops.embed(table, ids, scale=scale), out)
    (grad,) = torch.autograd.grad(out, leaf, dout)
    assert grad.shape == table.shape and grad.dtype == table.dtype
    flat = torch.where(ok, ids.long(), n).reshape(-1)
    terms = dout.reshape(-1, dim).double()
    zeros = torch.zeros(n + 1, dim, device="cuda", dtype=torch.float64)
    y = zeros.index_add(0, flat, terms)[:n] * scale
    size = zeros.index_add(0, flat, terms.abs())[:n] * abs(scale)
    count = torch.zeros(n + 1, device="cuda", dtype=torch.float64).index_add(0, flat, torch.ones_like(flat).double())
    bound = (count[:n, None] + 3) * U * size + y.abs() * (U if table.dtype == torch.float32 else 2.0 ** -8)
    assert bool(((grad.double() - y).abs() <= bound).all())
    assert not grad[count[:n] == 0].any()
    (again,) = torch.autograd.grad(ops.embed(leaf, ids, scale=scale), leaf, dout)
    assert torch.equal(again, grad)
    return out, grad


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,dim,shape,skew", [
    (50, 1, (3, 4), 0.0), (1, 8, (70,), 0.0), (9_228, 172, (600, 32), 1.0), (100, 32, (12, 10), 0.0),
    (1_000, 7, (5, 200), 2.0), (30_000, 100, (700, 20), 1.0), (5, 3, (40_000,), 0.0), (200_000, 16, (3_000, 20), 2.0),
    (2, 600, (1_500,), 0.0), (1_048_575, 4, (2_000,), 0.0), (700, 33, (64, 65), 0.0), (3_000, 1_100, (40, 9), 0.0)])
def test_embed(n, dim, shape, skew, dtype):
    _check(*_case(n, dim, shape, dtype, n + dim, skew), 1.0)
    _check(*_case(n, dim, shape, dtype, n + dim + 1, skew, torch.int64), -3.7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_row_takes_everything(dtype):
    """A hub: every token the same row, over many tiles, and beside it none."""
    table, ids, dout = _case(77, 20, (9_000,), dtype, 3)
    for fill in (0, 76, 40):
        _check(table, torch.full_like(ids, fill), dout, 0.5)
    _check(table, torch.full_like(ids, -1), dout, 0.5)


def test_empty():
    table = torch.randn(6, 5, device="cuda", requires_grad=True)
    out = ops.embed(table, torch.empty(0, 3, dtype=torch.int32, device="cuda"))
    assert out.shape == (0, 3, 5)
    (g,) = torch.autograd.grad(out, table, torch.empty_like(out))
    assert not g.any()
    none = torch.empty(0, 5, device="cuda", requires_grad=True)
    out = ops.embed(none, torch.tensor([0, -1, 4], device="cuda"))
    assert not out.any()
    assert torch.autograd.grad(out, none, torch.ones_like(out))[0].shape == (0, 5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(dtype):
    """A table of strided or shifted rows, ids and gradients that are not contiguous."""
    table, ids, dout = _case(300, 50, (40, 16), dtype, 8)
    want, grad = _check(table, ids, dout, 2.0)
    wide = torch.randn(300, 61, device="cuda").to(dtype)
    wide[:, 7:57] = table
    odd = torch.empty(300 * 50 + 1, device="cuda", dtype=dtype)[1:].view(300, 50)
    odd.copy_(table)
    for t in (wide[:, 7:57], odd, table.t().contiguous().t()):
        leaf = t.detach().requires_grad_()
        out = ops.embed(leaf, ids.t().contiguous().t(), scale=2.0)
        assert torch.equal(out, want)
        (g,) = torch.autograd.grad(out, leaf, torch.stack([dout, dout], -1)[..., 0])
        assert torch.equal(g, grad)


def test_rows_past_32_bits():
    """A table of 2.2e9 values: row offsets and the gradient's pass 32 bits."""
    n, dim = 4_300_000, 512
    table = torch.empty(n, dim, device="cuda", dtype=torch.bfloat16)
    ids = torch.tensor([0, n - 1, n - 2, n - 1, -1, 5, n], device="cuda")
    table[ids[:4]] = torch.randn(4, dim, device="cuda").bfloat16()
    table[5] = 3.0
    leaf = table.detach().requires_grad_()
    out = ops.embed(leaf, ids)
    assert torch.equal(out[:4], table[ids[:4]]) and not out[4].any() and not out[6].any()
    (g,) = torch.autograd.grad(out, leaf, torch.ones_like(out))
    assert bool((g[n - 1] == 2).all()) and bool((g[n - 2] == 1).all()) and bool((g[5] == 1).all())
    assert float(g.sum(dtype=torch.float64)) == 5 * dim


def test_gradient_against_differences():
    """The lookup is linear: its difference quotient is exact up to rounding (2 u / h of
    the output, h = 1)."""
    table, ids, dout = _case(90, 24, (30, 8), torch.float32, 4)
    _, grad = _check(table, ids, dout, 1.5)
    step = torch.randn_like(table)
    f = [(ops.embed(table + s * step, ids, scale=1.5).double() * dout.double()).sum() for s in (1, -1)]
    size = ((table.abs() + step.abs()).max() * 1.5 * dout.abs().sum()).double()
    assert abs((f[0] - f[1]) / 2 - (grad.double() * step.double()).sum()) <= 64 * U * size


def test_graph_replays():
    table, ids, dout = _case(400, 40, (50, 10), torch.float32, 6)
    table.requires_grad_()
    torch.autograd.grad(ops.embed(table, ids), table, dout)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.embed(table, ids)
        (grad,) = torch.autograd.grad(out, table, dout)
    for n in range(3):
        ids.copy_(_case(400, 40, (50, 10), torch.float32, 20 + n)[1])
        graph.replay()
        torch.cuda.synchronize()
        want = ops.embed(table, ids)
        assert torch.equal(out, want) and torch.equal(grad, torch.autograd.grad(want, table, dout)[0]), n


def test_refusals():
    t = torch.randn(5, 4, device="cuda")
    i = torch.zeros(3, dtype=torch.int32, device="cuda")
    for args, text in (((t[0], i), r"\(rows, dim\)"), ((t, i.float()), "int32 or int64"),
                       ((t.half(), i), "float32 or bfloat16"), ((t, i.cpu()), "device")):
        with pytest.raises(ValueError, match=text):
            ops.embed(*args)
    with pytest.raises(RuntimeError, match="on the GPU"):
        ops.embed(t.cpu(), i.cpu())
    leaf = t.detach().requires_grad_()
    with pytest.raises(RuntimeError, match="once only"):
        torch.autograd.grad(ops.embed(leaf, i).sum(), leaf, create_graph=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [1, 7, 50])
def test_broadcast_and_overlapping_tables(dim, dtype):
    """One row for all ids, whose gradient is the sum of theirs; rows that share values."""
    _, ids, dout = _case(40, dim, (30, 8), dtype, 9)
    row = torch.randn(1, dim, device="cuda").to(dtype).requires_grad_()
    ok = (ids >= 0) & (ids < 40)
    out = ops.embed(row.expand(40, dim), ids, scale=1.5)
    assert torch.equal(out, torch.where(ok[..., None], (row.float() * 1.5).to(dtype), 0.0))
    (g,) = torch.autograd.grad(out, row, dout)
    (full,) = torch.autograd.grad(ops.embed(row.expand(40, dim).contiguous(), ids, scale=1.5), row, dout)
    assert torch.equal(g, full)
    flat = torch.randn(40 + dim, device="cuda").to(dtype)
    windows = flat.unfold(0, dim, 1)[:40]
    assert torch.equal(ops.embed(windows, ids), ops.embed(windows.contiguous(), ids))
    both = flat[:1].expand(40, dim)  # one value for all
    assert torch.equal(ops.embed(both, ids), ops.embed(both.contiguous(), ids))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [400, 150_000, 3_000_000])  # keys of one, two and three digits
@pytest.mark.parametrize("n,dim", [(8_193, 6), (65_536, 5), (65_537, 5), (131_073, 12), (300_001, 20),
                                   (2 ** 21 + 1, 3), (2 ** 21 + 1, 8)])
def test_many_tokens(n, dim, rows, dtype):
    """Every way to sort: one workgroup's limit, few and many ranges, tiles of 16 to 64 tokens,
    long parts, and a hub over many tiles.  The sums in 64 bits are taken on the host: a hub's
    hundreds of thousands of additions to one place are slow on the device."""
    table, ids, dout = _case(rows, dim, (n,), dtype, n + rows, 1.0)
    ids[n // 3:n // 2] = rows - 2
    leaf = table.requires_grad_()
    (grad,) = torch.autograd.grad(ops.embed(leaf, ids, scale=0.75), leaf, dout)
    (again,) = torch.autograd.grad(ops.embed(leaf, ids, scale=0.75), leaf, dout)
    assert torch.equal(grad, again)
    flat = ids.cpu().numpy().astype(np.int64)
    ok = (flat >= 0) & (flat < rows)
    flat, terms = flat[ok], dout.double().cpu().numpy()[ok]
    count = np.bincount(flat, minlength=rows)
    r = U if dtype == torch.float32 else 2.0 ** -8
    for c in range(dim):
        y = np.bincount(flat, weights=terms[:, c], minlength=rows) * 0.75
        size = np.bincount(flat, weights=np.abs(terms[:, c]), minlength=rows) * 0.75
        off = np.abs(grad[:, c].double().cpu().numpy() - y)
        assert (off <= (count + 3) * U * size + np.abs(y) * r).all(), c
