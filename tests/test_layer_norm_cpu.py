"""Layer norm without a GPU: what the entry points refuse, what they do with nothing to do, workspace sizes."""
import ctypes

import pytest
import torch

import symplex_b200 as sx
from symplex_b200 import _capi

F32, BF16 = _capi.DT_F32, _capi.DT_BF16


def _buf(n=4096):
    return (ctypes.c_float * n)()


def _forward(lib, rows=4, cols=16, ldx=0, ldy=0, dtype=F32, pdtype=F32, eps=1e-5, x=True, y=True, offset=0):
    b = _buf()
    p = ctypes.addressof(b) + offset
    return lib.symplex_b200_layer_norm(p if x else None, p, p, p if y else None, None, None, rows, cols, ldx, ldy, dtype, pdtype, eps,
                                       None)


def _backward(lib, rows=4, cols=16, ldx=0, dtype=F32, pdtype=F32, ws=True, ws_bytes=1 << 20, mean=True, offset=0):
    b = _buf()
    p = ctypes.addressof(b)
    w = (p + 255) // 256 * 256 + offset
    return lib.symplex_b200_layer_norm_backward(p, p, p if mean else None, p, p, p, p, p, rows, cols, 0, ldx, 0, dtype, pdtype,
                                                w if ws else None, ws_bytes, None)


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(cols=0), dict(cols=-3), dict(cols=1 << 31), dict(ldx=15), dict(ldy=8), dict(dtype=10), dict(dtype=F32, pdtype=BF16),
    dict(pdtype=10), dict(eps=-1.0), dict(eps=float("nan")), dict(x=False), dict(y=False), dict(offset=2),
])
def test_forward_refuses(lib, bad):
    assert _forward(lib, **bad) == _capi.ERR_INVALID
    assert _capi.last_error() != "no error"


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(cols=0), dict(ldx=15), dict(dtype=10), dict(dtype=F32, pdtype=BF16), dict(ws=False), dict(ws_bytes=64),
    dict(mean=False), dict(offset=16),
])
def test_backward_refuses(lib, bad):
    assert _backward(lib, **bad) == _capi.ERR_INVALID
    assert _capi.last_error() != "no error"


def test_nothing_to_do(lib):
    assert _forward(lib, rows=0) == 0
    assert lib.symplex_b200_layer_norm_backward(None, None, None, None, None, None, None, None, 0, 8, 0, 0, 0, F32, F32, None, 0, None) == 0


def test_workspace_bytes(lib):
    f = lib.symplex_b200_layer_norm_backward_workspace_bytes
    assert f(0, 16) == 0 and f(-1, 16) == 0 and f(16, 0) == 0
    assert f(1, 100) == 2 * 100 * 4
    assert f(10**9, 100) == f(10**6, 100)  # bounded in the rows
    assert f(10**6, 2**31 - 1) < 2**63


@pytest.mark.skipif(torch.cuda.is_available(), reason="needs a box without a GPU")
def test_without_a_gpu_it_fails_loudly(lib):
    assert _forward(lib) in (_capi.ERR_DRIVER, _capi.ERR_EXEC)
    with pytest.raises(ValueError):
        sx.layer_norm(torch.zeros(2, 8))


def test_python_refuses_host_tensors():
    x = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="CUDA"):
        sx.layer_norm(x)
    with pytest.raises(ValueError, match="CUDA"):
        sx.layer_norm_backward(x, x, torch.zeros(2), torch.zeros(2))
