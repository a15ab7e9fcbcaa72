"""The operators around attention without a GPU: the C ABI's argument checks, its structs'
layouts against the ctypes mirrors, and refusal of CPU tensors."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from tgengine_amd import ops
from tgengine_amd.core import _lib

ROOT = Path(__file__).resolve().parent.parent

STRUCTS = {"tgx_scan_args": _lib.TgxScanArgs, "tgx_residual_norm_args": _lib.TgxResidualNormArgs}


def _err():
    return _lib.lib().tgx_last_error().decode()


@pytest.mark.parametrize("name", STRUCTS)
def test_struct_layout(tmp_path, name):
    kind = STRUCTS[name]
    names = [n for n, _ in kind._fields_]
    src = tmp_path / "p.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "tgx.h"\nint main(void) {\n' + "".join(
        f'printf("%zu\\n", offsetof({name}, {n}));\n' for n in names) + f'printf("%zu\\n", sizeof({name}));\nreturn 0; }}\n')
    subprocess.run(["gcc", "-std=c99", f"-I{ROOT / 'include'}", str(src), "-o", str(tmp_path / "p")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "p")], capture_output=True, text=True).stdout.split()]
    assert got == [getattr(kind, n).offset for n in names] + [ctypes.sizeof(kind)]


def _scan(**more):
    a = _lib.TgxScanArgs(x=8, gate=8, out=8, last=8, batch=2, length=3, dim=4)
    for n, v in more.items():
        setattr(a, n, v)
    return ctypes.byref(a)


def test_scan_checks():
    L = _lib.lib()
    for fn in (L.tgx_scan, L.tgx_scan_grad):
        assert fn(None, None) == 1 and "args is NULL" in _err()
        assert fn(_scan(batch=-1), None) == 1 and "batch=-1" in _err()
        assert fn(_scan(dim=0), None) == 1 and fn(_scan(length=-1), None) == 1
        assert fn(_scan(dtype=2), None) == 2
        assert fn(_scan(length=(1 << 30) + 1), None) == 3 and fn(_scan(batch=1 << 20, dim=1 << 20), None) == 3
        assert fn(_scan(batch=1 << 30, dim=5), None) == 3
        assert fn(_scan(gate=None), None) == 1 and "x and gate" in _err()
        assert fn(_scan(batch=0, x=None, gate=None, out=None, last=None), None) == 0
    assert L.tgx_scan(_scan(batch=1 << 30, length=1), None) == 3 and "one launch" in _err()
    assert L.tgx_scan(_scan(last=None), None) == 1 and "out and last" in _err()
    assert L.tgx_scan(_scan(out=None), None) == 1
    assert L.tgx_scan_grad(_scan(), None) == 0  # no gradient asked for
    assert L.tgx_scan_grad(_scan(length=40, grad_x=8), None) == 1 and "starts" in _err()
    # long rows of few channels are cut, and their pieces need room
    need = L.tgx_scan_workspace_size(_scan(length=5000))
    assert need > 0 and L.tgx_scan(_scan(length=5000), None) == 1 and "workspace" in _err()
    assert L.tgx_scan(_scan(length=5000, workspace=8, workspace_bytes=need), None) == 1  # not aligned
    assert L.tgx_scan(_scan(length=5000, workspace=16, workspace_bytes=need - 1), None) == 1
    assert L.tgx_scan_workspace_size(None) == 0 and L.tgx_scan_workspace_size(_scan()) == 0
    assert L.tgx_scan_workspace_size(_scan(dtype=7, length=5000)) == 0
    assert [L.tgx_scan_starts(n) for n in (0, 1, 16, 17, 32, 33)] == [0, 0, 0, 1, 1, 2]


def _res(**more):
    a = _lib.TgxResidualNormArgs(x=8, residual=8, out=8, sum=8, rows=3, dim=4, x_stride=4, residual_stride=4, eps=1e-5)
    for n, v in more.items():
        setattr(a, n, v)
    return ctypes.byref(a)


def test_residual_norm_checks():
    L = _lib.lib()
    for fn in (L.tgx_residual_norm, L.tgx_residual_norm_grad):
        assert fn(None, None) == 1 and "args is NULL" in _err()
        assert fn(_res(rows=-1), None) == 1 and fn(_res(dim=0), None) == 1
        assert fn(_res(gate_stride=-4), None) == 1 and "strides" in _err()
        assert fn(_res(dtype=2), None) == 2 and fn(_res(wdtype=-1), None) == 2
        assert fn(_res(dim=16385), None) == 3 and fn(_res(rows=1 << 31), None) == 3
        assert fn(_res(x=None), None) == 1 and "x must" in _err()
        assert fn(_res(residual=None, scale=8), None) == 1 and "residual" in _err()
        assert fn(_res(rows=0, x=None, residual=None), None) == 0
    assert L.tgx_residual_norm(_res(residual=None), None) == 1
    assert L.tgx_residual_norm(_res(sum=None), None) == 1 and "out and sum" in _err()
    for rows, dim in ((1 << 28, 200), (1 << 24, 16384), (1 << 30, 40)):
        assert L.tgx_residual_norm(_res(rows=rows, dim=dim), None) == 3 and "one launch" in _err()
    G = L.tgx_residual_norm_grad
    assert G(_res(grad_residual=8), None) == 1 and "stats" in _err()
    assert G(_res(grad_x=8, stats=8), None) == 1 and "grad_x" in _err()
    need = L.tgx_residual_norm_grad_workspace_size(_res(scale=8))
    assert need == 4 * L.tgx_residual_norm_grad_workspace_size(_res()) // 2 > 0
    for more in (dict(), dict(workspace=16, workspace_bytes=need - 1), dict(workspace=8, workspace_bytes=need)):
        assert G(_res(scale=8, grad_scale=8, stats=8, **more), None) == 1 and "workspace" in _err()
    assert L.tgx_residual_norm_grad_workspace_size(None) == 0 == L.tgx_residual_norm_grad_workspace_size(_res(dim=0))


def test_no_cpu_path():
    x = torch.randn(2, 3, 8)
    for call in (lambda: ops.gated_scan(x, x), lambda: ops.residual_norm(x, x)):
        with pytest.raises(RuntimeError, match="on the GPU"):
            call()
