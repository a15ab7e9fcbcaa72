"""The model-side operators without a GPU: the C ABI's argument checks, its struct
layout against the ctypes mirror, and refusal of CPU tensors."""
import ctypes
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from tgengine_amd import ops
from tgengine_amd.core import _lib

ROOT = Path(__file__).resolve().parent.parent


def _err():
    return _lib.lib().tgx_last_error().decode()


def _att(**more):
    a = _lib.TgxAttentionArgs(q=8, k=8, v=8, out=8, batch=2, lq=3, lk=4, heads=4, kv_heads=2, dim=16)
    for n, v in more.items():
        setattr(a, n, v)
    return ctypes.byref(a)


def test_attention_struct_layout(tmp_path):
    names = [n for n, _ in _lib.TgxAttentionArgs._fields_]
    src = tmp_path / "p.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "tgx.h"\nint main(void) {\n' + "".join(
        f'printf("%zu\\n", offsetof(tgx_attention_args, {n}));\n' for n in names)
        + 'printf("%zu\\n", sizeof(tgx_attention_args));\nreturn 0; }\n')
    subprocess.run(["gcc", "-std=c99", f"-I{ROOT / 'include'}", str(src), "-o", str(tmp_path / "p")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "p")], capture_output=True, text=True).stdout.split()]
    assert got == [getattr(_lib.TgxAttentionArgs, n).offset for n in names] + [ctypes.sizeof(_lib.TgxAttentionArgs)]


def test_attention_checks():
    L = _lib.lib()
    for fn in (L.tgx_attention, L.tgx_attention_grad):
        assert fn(None, None) == 1 and "args is NULL" in _err()
        assert fn(_att(heads=3), None) == 1 and "heads=3" in _err()
        assert fn(_att(dim=0), None) == 1
        assert fn(_att(lk=-1), None) == 1
        assert fn(_att(dim=257), None) == 3 and "dim=257" in _err()
        assert fn(_att(dtype=2), None) == 2
        assert fn(_att(q=None), None) == 1 and "q and out" in _err()
        assert fn(_att(v=None), None) == 1 and "k and v" in _err()
        assert fn(_att(lk=1 << 31), None) == 3
        assert fn(_att(batch=1 << 30), None) == 3
        assert fn(_att(batch=0), None) == 0 and fn(_att(lq=0, lk=0), None) == 0  # nothing to do
    assert L.tgx_attention_grad(_att(), None) == 1 and "grad_out and lse" in _err()
    assert L.tgx_attention_workspace_size(None) == 0 and L.tgx_attention_grad_workspace_size(_att(dim=300)) == 0


def test_embed_checks():
    L = _lib.lib()
    assert L.tgx_embed(8, 5, 0, 4, 0, 8, 1, 3, 1.0, 8, None) == 1
    assert L.tgx_embed(8, 5, 4, 4, 9, 8, 1, 3, 1.0, 8, None) == 2
    assert L.tgx_embed(8, 5, 65537, 65537, 0, 8, 1, 3, 1.0, 8, None) == 3
    assert L.tgx_embed(8, 1 << 31, 4, 4, 0, 8, 1, 3, 1.0, 8, None) == 3
    assert L.tgx_embed(8, 5, 4, 3, 0, 8, 1, 3, 1.0, 8, None) == 1 and "stride" in _err()
    assert L.tgx_embed(8, 5, 4, 4, 0, None, 1, 3, 1.0, 8, None) == 1
    assert L.tgx_embed(8, 5, 4, 4, 0, None, 1, 0, 1.0, None, None) == 0
    assert L.tgx_embed_grad(8, 8, 1, 3, 5, 4, 0, 1.0, 16, None, 0, None) == 1 and "workspace" in _err()
    assert L.tgx_embed_grad(8, 8, 1, 3, 5, 4, 0, 1.0, None, None, 0, None) == 1
    assert L.tgx_embed_grad(None, None, 1, 0, 0, 4, 0, 1.0, None, None, 0, None) == 0
    assert L.tgx_embed_grad_workspace_size(0, 4) == 0 and L.tgx_embed_grad_workspace_size(100, 4) > 1600


def test_layer_norm_checks():
    L = _lib.lib()
    assert L.tgx_layer_norm(8, 3, 0, 4, 0, None, None, 0, 1e-5, 8, None, None, None) == 1
    assert L.tgx_layer_norm(8, 3, 4, 4, 0, None, None, 5, 1e-5, 8, None, None, None) == 2
    assert L.tgx_layer_norm(8, 3, 16385, 16385, 0, None, None, 0, 1e-5, 8, None, None, None) == 3
    assert L.tgx_layer_norm(None, 3, 4, 4, 0, None, None, 0, 1e-5, 8, None, None, None) == 1
    assert L.tgx_layer_norm(8, 3, 4, 4, 0, None, None, 0, 1e-5, 8, 8, None, None) == 1 and "together" in _err()
    assert L.tgx_layer_norm(None, 0, 4, 4, 0, None, None, 0, 1e-5, None, None, None, None) == 0
    assert L.tgx_layer_norm_grad(8, 8, 3, 4, 4, 0, None, 0, None, None, 8, None, None, None, 0, None) == 1
    assert L.tgx_layer_norm_grad(8, 8, 3, 4, 4, 0, None, 0, 8, 8, 8, 8, None, None, 0, None) == 1
    assert "workspace" in _err()


def test_clip_checks():
    L = _lib.lib()
    P, I, S = ctypes.c_void_p * 1, ctypes.c_int32 * 1, ctypes.c_int64 * 1
    C = L.tgx_clip_grad_norm
    assert C(None, None, None, None, None, 1, 1.0, 8, None, 0, None) == 1
    assert C(None, None, None, None, None, 0, 1.0, None, None, 0, None) == 1
    assert C(P(8), I(0), P(8), I(0), S(-1), 1, 1.0, 8, None, 0, None) == 1
    assert C(P(8), I(3), P(8), I(0), S(5), 1, 1.0, 8, None, 0, None) == 2
    assert C(P(8), I(0), P(8), I(1), S(5), 1, 1.0, 8, None, 0, None) == 1 and "another dtype" in _err()
    assert C(P(8), I(0), P(8), I(0), S(5), 1, 1.0, 8, None, 0, None) == 1 and "workspace" in _err()
    assert L.tgx_clip_grad_norm_workspace_size(S(5), 1) == 4


def test_no_cpu_path():
    x = torch.randn(2, 3, 4, 8)
    for call in (lambda: ops.cross_attention(x, x, x), lambda: ops.layer_norm(x),
                 lambda: ops.embed(x[0, 0], torch.zeros(2, dtype=torch.int32)), lambda: ops.clip_grad_norm_([x], 1.0)):
        with pytest.raises(RuntimeError, match="on the GPU"):
            call()
    with pytest.raises(ValueError, match="no gradients"):
        ops.clip_grad_norm_([torch.nn.Parameter(x)], 1.0)


def test_grids_that_one_launch_does_not_take():
    L = _lib.lib()
    for lq in (1, 40):  # few rows a problem, and a tile of them
        a = _att(batch=1 << 28, lq=lq, heads=2, kv_heads=2)
        assert L.tgx_attention(a, None) == 3 and "one launch" in _err()
    assert L.tgx_embed_grad(8, 8, 1, 1 << 29, 5, 4, 0, 1.0, 8, 8, 1 << 50, None) == 3 and "2^29" in _err()


def test_clip_refuses_overlaps():
    """Outputs that are written twice, or read for another tensor: refused before any launch."""
    L = _lib.lib()

    def call(grads, outs, sizes, types=None, out_types=None):
        n = len(sizes)
        P, I, S = ctypes.c_void_p * n, ctypes.c_int32 * n, ctypes.c_int64 * n
        types = types or [0] * n
        return L.tgx_clip_grad_norm(P(*grads), I(*types), P(*outs), I(*(out_types or types)), S(*sizes), n, 1.0, 8, None,
                                    0, None)

    a, b, c = 0x10000, 0x20000, 0x30000
    for args in (([a, b, a], [a, b, a], [5, 7, 5]),               # a tied gradient, in place
                 ([a, b], [c, c], [5, 7]),                        # two gradients to one output
                 ([a, b], [b, a], [5, 5]),                        # outputs that trade places
                 ([a, b], [c, a + 16], [5, 3]),                   # an output inside another gradient
                 ([a], [a + 4], [5]),                             # one that is shifted against its own
                 ([a, b, c], [a, b, c + 8], [8192, 8192, 3]),     # ... and in a list
                 ([a, a + 8], [a, a + 8], [3, 3]),                # gradients that share a value
                 ([a, b], [a, a + 9], [5, 2], [1, 1]),            # the last byte of bf16
                 ([a, b], [c, c + 18], [5, 2], [0, 0], [0, 1])):
        assert call(*args) == 1 and "overlap" in _err(), args
    for args in (([a, b], [a, b], [5, 7]), ([a, a + 20], [a, a + 20], [5, 5]), ([a, a], [b, c], [5, 5]),
                 ([a, a + 4], [b, c], [5, 5]), ([a, a], [a, b], [0, 5]), ([a, b], [a, a + 10], [5, 2], [1, 1])):
        assert call(*args) == 1 and "workspace" in _err(), args  # apart: the next check speaks


def test_launches_of_2_32_threads_are_refused():
    """Before any launch, at the first size that reaches them."""
    L = _lib.lib()

    def norm(rows, dim, dtype):
        return L.tgx_layer_norm(8, rows, dim, 0, dtype, None, None, dtype, 1e-5, 8, None, None, None)

    for rows, dim, dtype in ((1 << 28, 257, 1), (1 << 28, 129, 0), (1 << 24, 16384, 1), (1 << 24, 4096, 0),
                             ((1 << 31) - 100, 3, 0)):
        assert norm(rows, dim, dtype) == 3 and "one launch" in _err(), (rows, dim)
    for n, rc in (((1 << 29) - 1, 3), ((1 << 29) - 63, 3), ((1 << 29) - 64, 1)):  # the last: no workspace
        assert L.tgx_embed_grad(8, 8, 1, n, 5, 4, 0, 1.0, 16, None, 0, None) == rc, n


def test_attention_rows_that_no_grid_takes():
    """Tiles of rows that pass 32 bits: refused, where their count came to zero and divided by it.  In a process
    of its own, which such a division would end."""
    code = """
import ctypes, sys
sys.path.insert(0, sys.argv[1])
from tgengine_amd.core import _lib
L = _lib.lib()
for dtype in (0, 1):
    for lq, heads, kv in ((1 << 30, 512, 1), ((1 << 31) - 1, 512, 1), (1 << 27, 4096, 64), (1 << 30, 8, 8)):
        a = ctypes.byref(_lib.TgxAttentionArgs(q=8, k=8, v=8, out=8, lse=8, grad_out=8, grad_q=8, grad_k=8, grad_v=8, batch=1,
                                               lq=lq, lk=10, heads=heads, kv_heads=kv, dim=1, dtype=dtype))
        assert L.tgx_attention_workspace_size(a) == 0 and L.tgx_attention_grad_workspace_size(a) == 0
        for fn in (L.tgx_attention, L.tgx_attention_grad):
            assert fn(a, None) == 3 and b"one launch" in L.tgx_last_error(), (lq, heads)
"""
    r = subprocess.run([sys.executable, "-c", code, str(ROOT)], capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stderr)
