"""The loss of a linear head without a GPU: what the entry points refuse, workspace sizes."""
import ctypes

import pytest
import torch

import symplex_b200 as sx
from symplex_b200 import _capi

F32, BF16 = _capi.DT_F32, _capi.DT_BF16


def _args(null, off):
    b = (ctypes.c_uint8 * 8192)()
    p = (ctypes.addressof(b) + 255) // 256 * 256
    names = ("dloss", "x", "W", "targets", "lse", "dx", "dW", "loss", "ws")
    return {n: None if n in null else p + off.get(n, 0) for n in names}, b


def _forward(lib, T=4, H=16, V=32, ldx=0, ldw=0, dt=BF16, red=1, null=(), off={}, ws=1 << 40):
    a, keep = _args(null, off)
    return lib.symplex_b200_linear_cross_entropy(a["x"], a["W"], a["targets"], a["loss"], a["lse"], T, H, V, ldx, ldw, dt, -100, red,
                                                 a["ws"], ws, None)


def _backward(lib, T=4, H=16, V=32, ldx=0, ldw=0, dt=BF16, red=1, null=(), off={}, ws=1 << 40):
    a, keep = _args(null, off)
    return lib.symplex_b200_linear_cross_entropy_backward(a["dloss"], a["x"], a["W"], a["targets"], a["lse"], a["dx"], a["dW"], T, H, V,
                                                          ldx, ldw, dt, -100, red, a["ws"], ws, None)


@pytest.mark.parametrize("f", [_forward, _backward])
@pytest.mark.parametrize("bad", [
    dict(T=-1), dict(H=0), dict(V=0), dict(T=1 << 30), dict(V=1 << 31), dict(ldx=15), dict(ldw=8), dict(dt=10), dict(red=3), dict(red=-1),
    dict(null=("x",)), dict(null=("W",)), dict(null=("targets",)), dict(null=("lse",)), dict(null=("ws",)), dict(ws=100),
    dict(off={"ws": 16}), dict(off={"targets": 4}), dict(off={"x": 1}), dict(off={"W": 1}), dict(off={"lse": 2}),
])
def test_refuses(lib, f, bad):
    assert f(lib, **bad) == _capi.ERR_INVALID
    assert _capi.last_error() != "no error"


def test_refuses_its_own_pointers(lib):
    assert _forward(lib, null=("loss",)) == _capi.ERR_INVALID
    for n in ("dloss", "dx", "dW"):
        assert _backward(lib, null=(n,)) == _capi.ERR_INVALID


def test_workspace_bytes(lib):
    f, b = lib.symplex_b200_linear_cross_entropy_workspace_bytes, lib.symplex_b200_linear_cross_entropy_backward_workspace_bytes
    for fn in (f, b):
        def w(T, H, V, dt, x=256, W=512, ldx=0, ldw=0):
            return fn(x, W, T, H, V, ldx, ldw, dt)
        assert w(0, 64, 100, BF16) == 0 and w(4, 0, 100, BF16) == 0 and w(4, 64, 0, BF16) == 0 and w(4, 64, 100, 3) == 0
        for dt in (BF16, F32):
            assert w(1, 64, 100, dt) > 0
            # the logits of the whole problem never fit in it
            assert w(8192, 4096, 1 << 17, dt) < 8192 * (1 << 17) * 4
        # operands that are copied first need room for it (the backward pass has a copy of x whatever its alignment)
        aligned = w(100, 64, 1000, BF16)
        for bad in (dict(W=520), dict(ldw=68)):
            assert w(100, 64, 1000, BF16, **bad) > aligned
        for bad in (dict(x=258), dict(ldx=65)):
            assert w(100, 64, 1000, BF16, **bad) > aligned if fn is f else w(100, 64, 1000, BF16, **bad) == aligned
        assert w(100, 64, 1000, BF16, ldx=72, ldw=128) == aligned


@pytest.mark.skipif(torch.cuda.is_available(), reason="needs a box without a GPU")
def test_without_a_gpu_it_fails_loudly(lib):
    assert _forward(lib) in (_capi.ERR_DRIVER, _capi.ERR_EXEC)
    assert _backward(lib) in (_capi.ERR_DRIVER, _capi.ERR_EXEC)


def test_python_refuses_host_tensors():
    x, w, t = torch.zeros(2, 8), torch.zeros(5, 8), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        sx.linear_cross_entropy(x, w, t)
    with pytest.raises(ValueError, match="CUDA"):
        sx.linear_cross_entropy_backward(torch.ones(()), x, w, t, torch.zeros(2))
