"""AdamW steps whose parts take several rounds.

A part is 1,024 values, and more where all tensors of a width hold above 67,108,864 values in 8 bits or 134,217,728 in
32.  In such a step a wavefront takes one block after the other with the next one on its way, and ragged tensors end
after whole rounds.  With 32 bits every value is stepped alone, so tensors cut in slices, whose parts are of one round,
have to give the same bits; with 8 bits codes and scales are compared with the definition over all values."""
import pytest
import torch

from tgengine_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F, B, E = torch.float32, torch.bfloat16, torch.float8_e4m3fn
TABLE = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** e for e in range(-9, 6) for m in range(8)] + [512.0]
SMALL = (3000, 2049, 5121, 4095, 4097, 12_543, 1, 256, 8192)  # ragged ones between whole rounds of 4,096
PART = 50_000 * 256


def _r(n, gen, scale, dtype=F):
    return torch.empty(n, device="cuda").normal_(0, scale, generator=gen).to(dtype)


def _pow2(k):
    return ((k.long() + 1023) << 52).view(torch.float64)


def _held(x, which, step, first):
    """(codes, the scale of every block) of 64-bit values, the first of which is value `first` of its tensor."""
    n = x.numel()
    size = torch.nn.functional.pad(x.abs(), (0, -n % 256)).view(-1, 256)
    top = size.amax(1, keepdim=True)
    k = torch.where(top == 0, -126, (torch.frexp(top).exponent - 8).clamp(min=-126))
    y = size * _pow2(-k)
    table = torch.tensor(TABLE, device="cuda", dtype=torch.float64)
    at = torch.searchsorted(table, y, right=True) - 1
    w = ((torch.arange(n, device="cuda") + first) * 0xC13FA9A9 + (step * 0x91E10DA5 + which * 2 ** 31) % 2 ** 32) & 0xFFFFFFFF
    u = torch.nn.functional.pad(w.double() / 2.0 ** 32, (0, -n % 256)).view(-1, 256)
    low, high = table[at], table[at + 1]
    out = torch.where((y - low) / (high - low) + u >= 1.0, high, low)
    if which:
        out = torch.where((size > 0) & (out == 0), TABLE[1], out)
    out = torch.copysign(out.view(-1)[:n], x)
    return torch.where(x == 0, 0.0, out), _pow2(k).view(-1)


def _state(sizes, bits, seed, dtype):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c = {"params": [_r(n, gen, 0.05, dtype) for n in sizes], "grads": [_r(n, gen, 0.01, dtype) for n in sizes],
         "steps": [torch.tensor(10 + i, device="cuda") for i in range(len(sizes))], "exp_avg": [], "exp_avg_sq": [], "scales": []}
    for n in sizes:
        m, v = _r(n, gen, 1.0), _r(n, gen, 1.0).square()
        if bits == 8:  # codes of up to 448, scales of some powers of two
            c["exp_avg"].append((m * 100).clamp(-400, 400).to(E))
            c["exp_avg_sq"].append((v * 100).clamp(0.01, 400).to(E))
            k = torch.randint(-16, -13, (2, -(-n // 256)), generator=gen, device="cuda")
            c["scales"].append(_pow2(k).float())
        else:
            c["exp_avg"].append(m * 0.002)
            c["exp_avg_sq"].append(v * 1e-5)
            c["scales"].append(None)
    return c


def _clone(c, which=slice(None)):
    return {k: [x if x is None else x.clone() for x in v[which]] for k, v in c.items()}


def _same(a, b):
    def bits(x):
        return x.reshape(-1).view(torch.uint8)

    return all(x is None or torch.equal(bits(x), bits(y)) for k in a for x, y in zip(a[k], b[k]))


HOW = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


def test_8_bits():
    sizes = SMALL[:5] + (205_000_003,) + SMALL[5:]
    assert sum(sizes) > 3 * 65536 * 1024  # rounds a part: 4
    c = _state(sizes, 8, 0, F)
    small = [i for i, n in enumerate(sizes) if n < 100_000]
    alone = {k: [v[i].clone() for i in small] for k, v in c.items()}
    big = len(SMALL[:5])
    before = {k: v[big].clone() for k, v in c.items()}
    norm = torch.tensor(2.0, device="cuda")
    ops.adamw_(**c, **HOW, grad_norm=norm, max_norm=1.0)
    ops.adamw_(**alone, **HOW, grad_norm=norm, max_norm=1.0)
    assert _same({k: [v[i] for i in small] for k, v in c.items()}, alone)
    t, n = int(before["steps"]) + 1, sizes[big]
    assert int(c["steps"][big]) == t
    clip, (b1, b2) = 1.0 / (2.0 + 1e-6), HOW["betas"]
    for lo in range(0, n, PART):
        hi = min(lo + PART, n)
        at, blocks = slice(lo, hi), slice(lo // 256, -(-hi // 256))
        by = [before["scales"][j, blocks].double().repeat_interleave(256)[:hi - lo] for j in (0, 1)]
        g = before["grads"][at].double() * clip
        m = b1 * (before["exp_avg"][at].double() * by[0]) + (1 - b1) * g
        v0 = before["exp_avg_sq"][at].double() * by[1]
        root = (b2 * (v0 * v0) + (1 - b2) * (g * g)).sqrt()
        for j, (name, x) in enumerate((("exp_avg", m), ("exp_avg_sq", root))):
            codes, scale = _held(x, j, t, lo)
            assert torch.equal(c["scales"][big][j, blocks].double(), scale), (name, lo)
            assert torch.equal(c[name][big][at].double(), codes), (name, lo)
        up = HOW["lr"] / (1 - b1 ** t) * m / (root / (1 - b2 ** t) ** 0.5 + HOW["eps"])
        p0 = before["params"][at].double()
        p = p0 * (1 - HOW["lr"] * HOW["weight_decay"]) - up
        # the constants, the averages in 32 bits, the reciprocal and its products: 16 u of the update; the decayed
        # parameter 3 u; the sum u
        bound = U * (3 * p0.abs() + 17 * up.abs() + p.abs())
        assert bool(((c["params"][big][at].double() - p).abs() <= 1.01 * bound).all()), lo


@pytest.mark.parametrize("dtype", [F, B])
def test_32_bits(dtype):
    sizes = SMALL[:5] + (410_000_003,) + SMALL[5:]
    assert sum(sizes) > 3 * 131072 * 1024
    c = _state(sizes, 32, 1, dtype)
    before = _clone(c)
    ops.adamw_(**c, **HOW)
    big = len(SMALL[:5])
    small = [i for i in range(len(sizes)) if i != big]
    alone = {k: [v[i] for i in small] for k, v in before.items()}
    ops.adamw_(**alone, **HOW)
    assert _same({k: [v[i] for i in small] for k, v in c.items()}, alone)
    # the large one in four slices of odd lengths, each in a step of its own
    cuts = [0, 100_000_001, 200_000_000, 300_000_007, sizes[big]]
    start = int(before["steps"][big])
    for lo, hi in zip(cuts, cuts[1:]):
        part = {k: [before[k][big][lo:hi]] for k in ("params", "grads", "exp_avg", "exp_avg_sq")}
        ops.adamw_(**part, steps=[torch.tensor(start, device="cuda")], **HOW)
    for k in ("params", "exp_avg", "exp_avg_sq", "grads"):
        assert torch.equal(c[k][big].view(torch.uint8), before[k][big].view(torch.uint8)), k
