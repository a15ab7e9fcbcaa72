"""Timed cases of the operators around attention: the rest of a model's block over a
node's history, and the step that trains it.

* ``scan``: the gated recurrence h = a h + (1 - a) x, a = sigmoid(gate), along the
  tokens of every row under a key mask, from a state and to one; with ``train``,
  the gradients of x, gate and state too.
* ``block``: the residual sum after a block, with the block's own norm, gate and
  residual scale, and the norm before the next block; with ``train``, all gradients.
* ``adamw``: one step over all of a model's tensors, with the averages in 32 bits or
  in 8, from gradients clipped by their global norm.

``own`` says whether ``run`` calls the framework's operators or computes them in
elementary torch operations.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-5
# the costliest listed passes move about this much; a drawn one no more
MOST_BYTES = 2.8e9

SCAN = {"op": "scan", "mask": "recent", "full": 0.6, "packed": False, "state": True, "train": True}
BLOCK = {"op": "block", "center": True, "post": False, "gate": False, "scale": False, "train": True}
ADAMW = {"op": "adamw", "table": 0, "dtype": "f32", "clipped": True}

# AdamW's constants, and the 8-bit averages: blocks of values that share a power of two,
# rounded with a dither of the value's place and the step
LR, BETA1, BETA2, ADAM_EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 1e-2
HELD = 256
PLACE, TURN = 0xC13FA9A9, 0x91E10DA5  # 2^32 / p and 2^32 / p^2, p the real root of p^3 = p + 1


def listed():
    return [
        # the newest event of a handful of nodes: one token into the nodes' states
        {"name": "scan_serve", **SCAN, "mask": "none", "train": False, "batch": 12, "length": 1, "dim": 172,
         "dtype": "f32"},
        # every query's 32 neighbours in the largest training batches
        {"name": "scan_recent", **SCAN, "state": False, "batch": 24_576, "length": 32, "dim": 172, "dtype": "bf16"},
        # a batch of the shape with the most neighbours a query
        {"name": "scan_sequence", **SCAN, "batch": 600, "length": 512, "dim": 100, "dtype": "f32", "packed": True},
        # two whole histories: few rows, so the tokens have to be shared out
        {"name": "scan_long", **SCAN, "mask": "prefix", "batch": 2, "length": 30_001, "dim": 256, "dtype": "bf16"},
        # tokens of a few online queries
        {"name": "block_serve", **BLOCK, "train": False, "rows": 240, "dim": 172, "dtype": "f32"},
        # every neighbour token of the largest batches, trained: sum and layer norm
        {"name": "block_train", **BLOCK, "rows": 786_432, "dim": 172, "dtype": "bf16"},
        # sequences of 65 tokens through a block with all of its parts
        {"name": "block_parts", **BLOCK, "center": False, "post": True, "gate": True, "scale": True, "rows": 26_000,
         "dim": 200, "dtype": "f32"},
        # wide states, gated
        {"name": "block_wide", **BLOCK, "center": False, "gate": True, "scale": True, "rows": 8_001, "dim": 4_096,
         "dtype": "bf16"},
        # a small model's layers: launches decide
        {"name": "adamw_layers", **ADAMW, "tensors": 16, "size": 20_000, "bits": 32},
        # a node table of 1M rows in bf16 and its model
        {"name": "adamw_table", **ADAMW, "tensors": 13, "size": 60_000, "table": 100_000_000, "dtype": "bf16",
         "bits": 32},
        # a larger model's layers with 8-bit averages
        {"name": "adamw_layers8", **ADAMW, "tensors": 12, "size": 300_000, "bits": 8},
        # a table of 1M rows of 172 values, whose averages would be the largest part of its memory
        {"name": "adamw_table8", **ADAMW, "tensors": 11, "size": 60_000, "table": 172_000_000, "bits": 8},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["scan", "scan", "block", "adamw"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "scan":
        kind = rng.choice(["serve", "recent", "sequence", "long"])
        c = {**SCAN, "dtype": dtype, "train": rng.random() < 0.7, "state": rng.random() < 0.6,
             "packed": rng.random() < 0.3, "full": rng.choice([0.2, 0.6, 0.9]),
             "dim": rng.choice([16, 100, 172, 256, _log(rng, 1, 2_048)])}
        if kind == "serve":
            c.update(batch=_log(rng, 1, 20_000), length=rng.randint(1, 3), mask="none", state=True)
        elif kind == "recent":
            c.update(batch=_log(rng, 4, 24_576), length=_log(rng, 5, 64), mask=rng.choice(["recent", "holes"]))
        elif kind == "sequence":
            c.update(batch=_log(rng, 4, 2_000), length=_log(rng, 32, 1_024),
                     mask=rng.choice(["recent", "prefix", "holes", "none"]))
        else:
            c.update(batch=rng.randint(1, 8), length=_log(rng, 1_000, 40_000), mask=rng.choice(["prefix", "none"]))
        sizes = ["batch", "length", "dim"]
    elif op == "block":
        c = {**BLOCK, "rows": _log(rng, 1, 786_432), "dim": rng.choice([100, 172, 256, _log(rng, 1, 8_192)]),
             "dtype": dtype, "train": rng.random() < 0.7, "center": rng.random() < 0.5, "post": rng.random() < 0.3,
             "gate": rng.random() < 0.5, "scale": rng.random() < 0.5}
        sizes = ["rows"]
    else:
        c = {**ADAMW, "tensors": rng.randint(1, 11), "size": _log(rng, 50, 1_000_000), "dtype": dtype,
             "table": rng.choice([0, _log(rng, 10_000, 172_000_000)]), "bits": rng.choice([8, 32]),
             "clipped": rng.random() < 0.7}
        sizes = ["table", "size"]
    i = 0
    while work(c)["bytes"] > MOST_BYTES:
        s = sizes[i % len(sizes)]
        i += 1
        if c[s] > 1:
            c[s] = c[s] // 2 + 1
    return c


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def _mask(c, gen):
    b, n = c["batch"], c["length"]
    if c["mask"] == "none":
        return None
    if c["mask"] == "holes":
        return torch.rand(b, n, generator=gen, device="cuda") < c["full"]
    # a share of the rows is full, the others hold any number from none on
    some = torch.randint(0, n + 1, (b,), generator=gen, device="cuda")
    held = torch.where(torch.rand(b, generator=gen, device="cuda") < c["full"], torch.full_like(some, n), some)[:, None]
    at = torch.arange(n, device="cuda")
    # neighbours stand at a row's end, the most recent last; a sequence's states at its start
    return at >= n - held if c["mask"] == "recent" else at < held


def _shapes(c):
    """A model's tensors: a node table first, then matrices, biases and odd vectors around ``size``."""
    out = [c["table"]] if c["table"] else []
    kinds = [c["size"], max(1, c["size"] // 172), max(1, c["size"] // 7), c["size"] + 1]
    return out + [kinds[i % 4] for i in range(c["tensors"])]


def prepare(case, seed):
    c, gen, dt = case, _gen(seed), DTYPES[case["dtype"]]
    s = {"case": c}
    if c["op"] == "scan":
        b, n, d = c["batch"], c["length"], c["dim"]
        if c["packed"]:  # tokens and gates side by side, as one projection gives them
            both = _randn(gen, b, n, 2, d, dtype=dt)
            s["x"], s["gate"] = both[:, :, 0], both[:, :, 1]
        else:
            s["x"], s["gate"] = _randn(gen, b, n, d, dtype=dt), _randn(gen, b, n, d, dtype=dt, scale=2.0)
        s["mask"] = _mask(c, gen)
        s["state"] = _randn(gen, b, d) if c["state"] else None
        if c["train"]:
            s["grad"] = _randn(gen, b, n, d, dtype=dt), _randn(gen, b, d)
            s.update({x: s[x].detach().requires_grad_() for x in ("x", "gate", "state") if s[x] is not None})
    elif c["op"] == "block":
        n, d = c["rows"], c["dim"]
        s["x"], s["residual"] = _randn(gen, n, d, dtype=dt), (_randn(gen, n, d) * 1.5 + 0.3).to(dt)
        s["gate"] = _randn(gen, n, d, dtype=dt) if c["gate"] else None
        s["scale"] = (_randn(gen, d, scale=0.1) + 0.5).to(dt) if c["scale"] else None
        s["post_weight"] = (_randn(gen, d, scale=0.1) + 1).to(dt) if c["post"] else None
        s["weight"] = (_randn(gen, d, scale=0.1) + 1).to(dt)
        s["bias"] = _randn(gen, d, dtype=dt, scale=0.1) if c["center"] else None
        if c["train"]:
            s["grad"] = _randn(gen, n, d, dtype=dt), _randn(gen, n, d, dtype=dt)
            s.update({x: s[x].requires_grad_() for x in PARTS if s[x] is not None})
    else:
        # layers in 32 bits, the table in the case's type
        shapes = _shapes(c)
        types = [dt if c["table"] and i == 0 else torch.float32 for i in range(len(shapes))]
        s["params"] = [_randn(gen, n, dtype=t, scale=0.05) for n, t in zip(shapes, types)]
        s["grads"] = [_randn(gen, n, dtype=t, scale=0.01) for n, t in zip(shapes, types)]
        # averages as they stand in the middle of a run
        s["exp_avg"] = [_randn(gen, n, scale=0.002) for n in shapes]
        s["exp_avg_sq"] = [(_randn(gen, n, scale=0.002) + 0.008).square() for n in shapes]
        s["steps"] = [torch.tensor(1_000, device="cuda") for _ in shapes]
        s["scales"] = None
        if c["bits"] == 8:
            first = [_held(m.double(), 0, 1_000) for m in s["exp_avg"]]
            second = [_held(v.double().sqrt(), 1, 1_000) for v in s["exp_avg_sq"]]
            s["exp_avg"], s["exp_avg_sq"] = [x[0] for x in first], [x[0] for x in second]
            s["scales"] = [torch.stack([x[1], y[1]]) for x, y in zip(first, second)]
        expected = 0.01 * math.sqrt(sum(shapes))
        s["norm"] = torch.tensor(expected, device="cuda")
        s["max_norm"] = expected * (0.5 if c["clipped"] else 2.0)
    return s


PARTS = ("x", "residual", "weight", "bias", "gate", "scale", "post_weight")


# ---------------------------------------------------------------- the plain forms
def _doubled(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 1 from h = 0: spans of twice the length each time
    (a running product in logarithms would lose what far tokens leave)."""
    off = 1
    while off < b.shape[1]:
        b = torch.cat([b[:, :off], b[:, off:] + a[:, off:] * b[:, :-off]], 1)
        a = torch.cat([a[:, :off], a[:, off:] * a[:, :-off]], 1)
        off *= 2
    return b


def _plain_scan(s):
    dt = s["x"].dtype
    x, gate = s["x"].float(), s["gate"].float()
    a, rest = 1 / (1 + torch.exp(-gate)), 1 / (1 + torch.exp(gate))
    if s["mask"] is not None:
        keep = s["mask"][:, :, None]
        a, rest, x = torch.where(keep, a, 1.0), torch.where(keep, rest, 0.0), torch.where(keep, x, 0.0)
    h0 = s["state"][:, None].float() if s["state"] is not None else torch.zeros_like(x[:, :1])
    b = rest * x
    b = torch.cat([b[:, :1] + a[:, :1] * h0, b[:, 1:]], 1)
    h = _doubled(a, b)
    if not s["case"]["train"]:
        return h.to(dt), h[:, -1].contiguous()
    g, g_last = s["grad"]
    g = g.float()
    g = torch.cat([g[:, :-1], g[:, -1:] + g_last[:, None]], 1)
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    dh = _doubled(after.flip(1), g.flip(1)).flip(1)
    before = torch.cat([h0, h[:, :-1]], 1)
    out = [h.to(dt), h[:, -1].contiguous(), (dh * rest).to(dt), (dh * (before - x) * a * rest).to(dt)]
    return out + ([dh[:, 0] * a[:, 0]] if s["state"] is not None else [])


def _norm_forward(x, center):
    x = x - x.mean(-1, keepdim=True) if center else x
    r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return x * r, r


def _norm_backward(g, h, r, center):
    g = g - h * (g * h).mean(-1, keepdim=True) - (g.mean(-1, keepdim=True) if center else 0.0)
    return g * r


def _plain_block(s):
    c, dt = s["case"], s["x"].dtype
    x, residual, weight = s["x"].float(), s["residual"].float(), s["weight"].float()
    bias, gate, scale, post = (s[n].float() if s[n] is not None else None for n in ("bias", "gate", "scale", "post_weight"))
    if post is not None:
        hx, rx = _norm_forward(x, c["center"])
        n = hx * post
    else:
        n = x
    sig = 1 / (1 + torch.exp(-gate)) if gate is not None else 1.0
    by = sig * scale if scale is not None else sig
    total = residual + by * n
    h, r = _norm_forward(total, c["center"])
    y = h * weight + (bias if bias is not None else 0.0)
    if not c["train"]:
        return y.to(dt), total.to(dt)
    gy, gs = s["grad"][0].float(), s["grad"][1].float()
    d = gs + _norm_backward(gy * weight, h, r, c["center"])
    dn = d * by
    dx = _norm_backward(dn * post, hx, rx, c["center"]) if post is not None else dn
    out = [y, total, dx, d, (gy * h).sum(0)]
    if bias is not None:
        out.append(gy.sum(0))
    if gate is not None:
        out.append(dn * n * (1 - sig))
    if scale is not None:
        out.append((d * sig * n).sum(0))
    if post is not None:
        out.append((dn * hx).sum(0))
    return [t.to(dt) for t in out]


def _pow2(k):
    return ((k.long() + 1023) << 52).view(torch.float64)


def _dither(n, which, step):
    at = torch.arange(n, device="cuda") * PLACE + (step * TURN + (which << 31))
    return (at & 0xFFFFFFFF).double() * 2.0 ** -32


def _blocks(x, n):
    return torch.nn.functional.pad(x, (0, -n % HELD)).view(-1, HELD)


def _held(x, which, step):
    """64-bit values as e4m3 and a power of two for each block, whose largest value comes to lie in [128, 256).
    Between two neighbours of the format the dither decides; a second average (which = 1) above zero stays so."""
    n = x.numel()
    x, u = _blocks(x, n), _blocks(_dither(n, which, step), n)
    e = torch.frexp(x).exponent - 1
    k = (torch.where(x == 0, -2_000, e).amax(1, keepdim=True) - 7).clamp(min=-126)
    finest = torch.clamp(e - k, min=-6) - 3
    steps = torch.floor(x.abs() * _pow2(-k) * _pow2(-finest) + u)
    if which:
        steps = torch.where(x > 0, steps.clamp(min=1), steps)
    y = torch.where(x == 0, 0.0, steps * _pow2(finest)) * x.sign()
    return y.view(-1)[:n].to(torch.float8_e4m3fn), _pow2(k).view(-1).float()


def _plain_adamw(s):
    c = s["case"]
    wide = c["bits"] == 8  # values next to a border between two of the 8-bit ones
    for i, (p, g) in enumerate(zip(s["params"], s["grads"])):
        m, v, n = s["exp_avg"][i], s["exp_avg_sq"][i], p.numel()
        t = s["steps"][i].add_(1)
        clip = torch.clamp(s["max_norm"] / (s["norm"].double() + 1e-6), max=1.0)
        if wide:
            first, second = ((_blocks(x.double(), n) * s["scales"][i][j].double()[:, None]).view(-1)[:n]
                             for j, x in enumerate((m, v)))
            g = g.double() * clip
            first = BETA1 * first + (1 - BETA1) * g
            second = BETA2 * second.square() + (1 - BETA2) * g.square()
            root = second.sqrt()
            for j, (to, x) in enumerate(((m, first), (v, root))):
                held, scale = _held(x, j, t)
                to.copy_(held)
                s["scales"][i][j].copy_(scale)
            first, root = first.float(), root.float()
        else:
            g = g.float() * clip.float()
            first = m.mul_(BETA1).add_((1 - BETA1) * g)
            root = v.mul_(BETA2).add_((1 - BETA2) * g * g).sqrt()
        by = (LR / (1 - BETA1 ** t.double())).float()
        even = (1 - BETA2 ** t.double()).rsqrt().float()
        p.copy_(p.float() * (1 - LR * DECAY) - by * first / (root * even + ADAM_EPS))
    return _stepped(s)


def _stepped(s):
    return [s["params"], s["exp_avg"], s["exp_avg_sq"], s["scales"]]


PLAIN = {"scan": _plain_scan, "block": _plain_block, "adamw": _plain_adamw}


# ---------------------------------------------------------------- the framework's operators
def _own(s):
    from tgengine_amd import ops
    c = s["case"]
    if c["op"] == "adamw":
        ops.adamw_(s["params"], s["grads"], s["exp_avg"], s["exp_avg_sq"], s["steps"], lr=LR, betas=(BETA1, BETA2),
                   eps=ADAM_EPS, weight_decay=DECAY, scales=s["scales"], grad_norm=s["norm"], max_norm=s["max_norm"])
        return _stepped(s)
    if c["op"] == "scan":
        out = ops.gated_scan(s["x"], s["gate"], mask=s["mask"], state=s["state"])
        names = ("x", "gate", "state")
    else:
        out = ops.residual_norm(s["x"], s["residual"], s["weight"], s["bias"], gate=s["gate"], scale=s["scale"],
                                post_weight=s["post_weight"], center=c["center"], eps=EPS)
        names = PARTS
    if not c["train"]:
        return out
    return [*out, *torch.autograd.grad(out, [s[x] for x in names if s[x] is not None], s["grad"])]


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_scan(s):
    """One token after the other, there and back."""
    c = s["case"]
    b, n, d = c["batch"], c["length"], c["dim"]
    new = lambda: torch.zeros(b, n, d, device="cuda", dtype=torch.float64)  # noqa: E731
    h = torch.zeros(b, d, device="cuda", dtype=torch.float64) if s["state"] is None else s["state"].detach().double()
    out = new()
    keep = s["mask"][:, :, None] if s["mask"] is not None else torch.ones(b, n, 1, device="cuda", dtype=torch.bool)
    x, a = s["x"].detach(), s["gate"].detach()
    for t in range(n):
        f = torch.sigmoid(a[:, t].double())
        h = torch.where(keep[:, t], h * f + x[:, t].double() * (1 - f), h)
        out[:, t] = h
    if not c["train"]:
        return out, h
    dx, da, dh = new(), new(), s["grad"][1].double()
    for t in range(n - 1, -1, -1):
        dh = dh + s["grad"][0][:, t].double()
        f = torch.sigmoid(a[:, t].double())
        old = out[:, t - 1] if t else torch.zeros_like(h) if s["state"] is None else s["state"].detach().double()
        dx[:, t] = torch.where(keep[:, t], dh * (1 - f), 0.0)
        da[:, t] = torch.where(keep[:, t], dh * (old - x[:, t].double()) * f * (1 - f), 0.0)
        dh = torch.where(keep[:, t], dh * f, dh)
    return [out, h, dx, da] + ([dh] if s["state"] is not None else [])


def _exact_norm(x, center):
    if center:
        return (x - x.mean(-1, keepdim=True)) / torch.sqrt(x.var(-1, keepdim=True, unbiased=False) + EPS)
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)


def _exact_block(s):
    c = s["case"]
    p = {n: s[n].detach().double().requires_grad_(c["train"]) for n in PARTS if s[n] is not None}
    part = max(1, int(2e8 / c["dim"]))
    rows = [[], []]
    grads = {n: [] for n in p}
    for i in range(0, c["rows"], part):
        cut = {n: (v[i:i + part] if v.dim() == 2 else v) for n, v in p.items()}
        n = _exact_norm(cut["x"], c["center"]) * cut["post_weight"] if c["post"] else cut["x"]
        for f in ([torch.sigmoid(cut["gate"])] if c["gate"] else []) + ([cut["scale"]] if c["scale"] else []):
            n = n * f
        total = cut["residual"] + n
        y = _exact_norm(total, c["center"]) * cut["weight"]
        y = y + cut["bias"] if "bias" in cut else y
        if c["train"]:
            asked = {k: cut[k] if p[k].dim() == 2 else p[k] for k in p}
            got = torch.autograd.grad((y, total), list(asked.values()), [g[i:i + part].double() for g in s["grad"]])
            for k, g in zip(asked, got):
                grads[k].append(g)
        rows[0].append(y.detach())
        rows[1].append(total.detach())
    out = [torch.cat(r) for r in rows]
    return out + ([torch.cat(g) if p[n].dim() == 2 else sum(g) for n, g in grads.items()] if c["train"] else [])


def _exact_held(x, which, step):
    """By a table of the format's values."""
    table = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** e for e in range(-9, 6) for m in range(8)] + [512.0]
    table = torch.tensor(table, device="cuda", dtype=torch.float64)
    n = x.numel()
    size = torch.nn.functional.pad(x.abs(), (0, -n % HELD)).view(-1, HELD)
    top = size.amax(1, keepdim=True).cpu().numpy()
    k = np.maximum(np.frexp(top)[1] - 8, -126)
    k = torch.from_numpy(np.where(top == 0, -126, k)).cuda()
    y = size * torch.from_numpy(np.ldexp(1.0, -k.cpu().numpy())).cuda()
    at = torch.searchsorted(table, y, right=True) - 1
    low, high = table[at], table[at + 1]
    i = np.arange(n, dtype=np.uint32)
    with np.errstate(over="ignore"):
        u = i * np.uint32(PLACE) + np.uint32((step * TURN + which * 2 ** 31) % 2 ** 32)
    u = torch.nn.functional.pad(torch.from_numpy(u.astype(np.int64)).cuda().double() / 2.0 ** 32, (0, -n % HELD)).view(-1, HELD)
    y = torch.where((y - low) >= (1 - u) * (high - low), high, low)
    if which:
        y = torch.where((size > 0) & (y == 0), table[1], y)
    scale = torch.from_numpy(np.ldexp(1.0, k.cpu().numpy())).cuda()
    return torch.copysign(y.view(-1)[:n], x), scale.view(-1)


def _exact_adamw(s):
    out = [[], [], [], []]
    norm = float(s["norm"])
    clip = min(1.0, s["max_norm"] / (norm + 1e-6))
    for i, p in enumerate(s["params"]):
        n, t = p.numel(), int(s["steps"][i]) + 1
        g = s["grads"][i].double() * clip
        m, v = s["exp_avg"][i].double(), s["exp_avg_sq"][i].double()
        if s["scales"] is not None:
            m, v = (x * s["scales"][i][j].double().repeat_interleave(HELD)[:n] for j, x in enumerate((m, v)))
            v = v * v
        m, v = m * BETA1 + g * (1 - BETA1), v * BETA2 + g * g * (1 - BETA2)
        root = torch.sqrt(v)
        p = p.double()
        p = p - LR * DECAY * p - LR * (m / (1 - BETA1 ** t)) / (root / math.sqrt(1 - BETA2 ** t) + ADAM_EPS)
        out[0].append(p)
        if s["scales"] is not None:
            (m, a), (v, b) = _exact_held(m, 0, t), _exact_held(root, 1, t)
            out[3].append(torch.stack([a, b]))
        out[1].append(m)
        out[2].append(v)
    if s["scales"] is None:
        out[3] = None
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"scan": _exact_scan, "block": _exact_block, "adamw": _exact_adamw}[case["op"]](s)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "scan":
        kept = 1.0 if c["mask"] == "none" else c["full"] if c["mask"] == "holes" else c["full"] + (1 - c["full"]) / 2
        one = c["batch"] * c["length"] * c["dim"]
        states = c["batch"] * c["dim"] * 4 * (2 if c["state"] else 1)
        masks = 0 if c["mask"] == "none" else c["batch"] * c["length"]
        # x, gate -> out; then x, gate, dout -> dx, dgate: masked tokens are written, and their x and gate not read
        moved, done = (2 * kept + 1) * one * size + states + masks, 10 * one * kept
        if c["train"]:
            moved, done = moved + (2 * kept + 3) * one * size + states + masks, done + 20 * one * kept
    elif c["op"] == "block":
        one = c["rows"] * c["dim"]
        more = c["gate"] * 1
        scaled = c["gate"] or c["scale"] or c["post"]
        # x, residual, gate -> y, sum; then those, dy, dsum -> dx, dresidual, dgate (the sum alone where nothing scales x)
        moved, done = (4 + more) * one * size, (10 + 6 * more + 6 * c["post"]) * one
        if c["train"]:
            moved += ((6 + 2 * more) if scaled else 4) * one * size
            done += (20 + 10 * more + 14 * c["post"]) * one
    else:
        shapes = _shapes(c)
        held = 16 if c["bits"] == 32 else 4 + 16 / HELD
        layers = sum(shapes) - c["table"]
        moved = layers * (12 + held) + c["table"] * (3 * size + held)
        done = (20 if c["bits"] == 32 else 60) * sum(shapes)
    return {"bytes": float(moved), "flops": float(done)}
