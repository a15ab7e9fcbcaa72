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

STRUCTS = {"tgx_scan_args": _lib.TgxScanArgs, "tgx_residual_norm_args": _lib.TgxResidualNormArgs,
           "tgx_adamw_tensor": _lib.TgxAdamwTensor, "tgx_adamw_args": _lib.TgxAdamwArgs}


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
        for more in (dict(x_stride=(-12, 4)), dict(x_stride=(12, -4)), dict(gate_stride=(0, -1)), dict(mask_stride=-3)):
            more = {n: (ctypes.c_int64 * 2)(*v) if isinstance(v, tuple) else v for n, v in more.items()}
            assert fn(_scan(**more), None) == 1 and "stride of -" in _err()
        assert fn(_scan(dtype=2), None) == 2
        assert fn(_scan(length=(1 << 30) + 1), None) == 3 and fn(_scan(batch=1 << 20, dim=1 << 20), None) == 3
        assert fn(_scan(batch=1 << 30, dim=5), None) == 3
        assert fn(_scan(gate=None), None) == 1 and "x and gate" in _err()
        assert fn(_scan(batch=0, x=None, gate=None, out=None, last=None), None) == 0
    assert L.tgx_scan(_scan(batch=1 << 30, length=1), None) == 3 and "one launch" in _err()
    assert L.tgx_scan(_scan(last=None), None) == 1 and "out and last" in _err()
    assert L.tgx_scan(_scan(out=None), None) == 1
    for more in (dict(), dict(grad_x=8), dict(grad_gate=8)):
        assert L.tgx_scan_grad(_scan(**more), None) == 1 and "grad_x and grad_gate" in _err()
    assert L.tgx_scan_grad(_scan(length=40, grad_x=8, grad_gate=8), None) == 1 and "starts" in _err()
    # long rows of few channels are cut, and their pieces need room
    need = L.tgx_scan_workspace_size(_scan(length=5000))
    assert need > 0 and L.tgx_scan(_scan(length=5000), None) == 1 and "workspace" in _err()
    assert L.tgx_scan(_scan(length=5000, workspace=8, workspace_bytes=need), None) == 1  # not aligned
    assert L.tgx_scan(_scan(length=5000, workspace=16, workspace_bytes=need - 1), None) == 1
    assert L.tgx_scan_workspace_size(None) == 0 and L.tgx_scan_workspace_size(_scan()) == 0
    assert L.tgx_scan_workspace_size(_scan(dtype=7, length=5000)) == 0
    assert [L.tgx_scan_starts(n) for n in (0, 1, 8, 9, 16, 17, 33)] == [0, 0, 0, 1, 1, 2, 4]


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


def _tensor(at=0x10000, **more):
    """A tensor of 300 f32 values whose memory begins at `at`, 4 KB a piece."""
    t = dict(param=at, grad=at + 0x1000, exp_avg=at + 0x2000, exp_avg_sq=at + 0x3000, scales=at + 0x4000, step=at + 0x5000,
             size=300, dtype=0, grad_dtype=0, bits=32)
    return _lib.TgxAdamwTensor(**{**t, **more})


def _adamw(*tensors, **more):
    t = (_lib.TgxAdamwTensor * max(1, len(tensors)))(*tensors)
    a = _lib.TgxAdamwArgs(tensors=t, count=len(tensors), lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=1e-2)
    for n, v in more.items():
        setattr(a, n, v)
    return _lib.lib().tgx_adamw(ctypes.byref(a), None)


def test_adamw_checks():
    L = _lib.lib()
    assert L.tgx_adamw(None, None) == 1 and "args is NULL" in _err()
    assert L.tgx_adamw_workspace_size(0) == 0 and L.tgx_adamw_workspace_size(3) >= 96
    assert _adamw() == 0 and _adamw(_tensor(), count=-1) == 1
    assert _adamw(_tensor()) == 1 and "workspace" in _err()
    for more in (dict(lr=-1.0), dict(lr=float("nan")), dict(beta1=1.0), dict(beta2=-0.1), dict(beta2=float("nan")), dict(eps=-1.0),
                 dict(weight_decay=float("nan"))):
        assert _adamw(_tensor(), **more) == 1 and "lr=" in _err()
    assert _adamw(_tensor(), lr=float("nan"), lr_device=0x90000) == 1 and "workspace" in _err()
    assert _adamw(_tensor(), grad_norm=0x90000, max_norm=-1.0) == 1 and "max_norm" in _err()
    for more in (dict(size=-1), dict(param=None), dict(grad=None), dict(exp_avg=None), dict(exp_avg_sq=None), dict(step=None)):
        assert _adamw(_tensor(), _tensor(0x20000, **more)) == 1 and "tensor 1" in _err()
    assert _adamw(_tensor(dtype=2)) == 2 and _adamw(_tensor(grad_dtype=-1)) == 2
    assert _adamw(_tensor(bits=16)) == 1 and "16 bits" in _err()
    assert _adamw(_tensor(bits=8, scales=None)) == 1 and "scales" in _err()
    assert _adamw(_tensor(bits=8)) == 1 and "workspace" in _err()
    assert _adamw(_tensor(size=0, param=None, grad=None, exp_avg=None, exp_avg_sq=None)) == 1 and "workspace" in _err()
    assert _adamw(_tensor(size=1 << 40)) == 3


def test_adamw_refuses_overlaps():
    """Memory that is written and used for anything else: refused before any launch."""
    a, b = 0x10000, 0x20000
    for tensors in ((_tensor(a), _tensor(b, param=a)), (_tensor(a), _tensor(b, step=a + 0x5000)),
                    (_tensor(a, grad=a),), (_tensor(a, exp_avg_sq=a + 0x2000),), (_tensor(a), _tensor(b, grad=a + 1196)),
                    (_tensor(a, step=a + 0x1000),), (_tensor(a, bits=8, scales=a + 0x2000 + 296),),
                    (_tensor(a, bits=8, exp_avg_sq=a + 0x2000 + 299),), (_tensor(a, dtype=1, grad=a + 599),)):
        assert _adamw(*tensors) == 1 and "overlap" in _err()
    assert _adamw(_tensor(a), grad_norm=a, max_norm=1.0) == 1 and "overlap" in _err()
    assert _adamw(_tensor(a), lr_device=a + 0x2000 + 4) == 1 and "overlap" in _err()
    for tensors in ((_tensor(a), _tensor(b, grad=a + 0x1000)),  # two that share a gradient
                    (_tensor(a, bits=8, exp_avg_sq=a + 0x2000 + 300),), (_tensor(a, dtype=1, grad=a + 600),),
                    (_tensor(a), _tensor(b, grad=a + 1200))):
        assert _adamw(*tensors) == 1 and "workspace" in _err()


def test_no_cpu_path():
    x = torch.randn(2, 3, 8)
    for call in (lambda: ops.gated_scan(x, x), lambda: ops.residual_norm(x, x),
                 lambda: ops.adamw_([x], [x], [x], [x], [torch.zeros((), dtype=torch.int64)])):
        with pytest.raises(RuntimeError, match="on the GPU"):
            call()


def test_adamw_groups_are_checked():
    one, other = (torch.nn.Parameter(torch.zeros(3)) for _ in range(2))
    adam = ops.AdamW([one], bits=8)
    with pytest.raises(ValueError, match="bits"):
        adam.add_param_group({"params": [other], "bits": 16})
    with pytest.raises(ValueError, match="bits"):
        ops.AdamW([{"params": [one], "bits": 4}])
    with pytest.raises(ValueError, match="bits"):
        ops.AdamW([one], bits=4)
    adam.add_param_group({"params": [other], "bits": 32, "lr": 1e-2})
    assert [g["bits"] for g in adam.param_groups] == [8, 32]
