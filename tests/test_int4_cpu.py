"""4-bit weights without a GPU: what the entry points refuse."""
import ctypes

import pytest
import torch

import symplex_b200 as sx
from symplex_b200 import _capi

F32, BF16 = _capi.DT_F32, _capi.DT_BF16


def _matvec(lib, M=2, N=4, K=64, group=32, lda=0, ldq=0, ldc=0, sdt=BF16, odt=BF16, act=0, null=(), off=0):
    b = (ctypes.c_uint8 * 4096)()
    p = ctypes.addressof(b)
    ptr = {n: None if n in null else p + (off if n == "A" else 0) for n in ("A", "codes", "scales", "C")}
    return lib.symplex_b200_int4_matvec(ptr["A"], ptr["codes"], ptr["scales"], None, None, ptr["C"], M, N, K, group, lda, ldq, ldc, sdt,
                                        odt, act, None)


def _quantize(lib, N=4, K=64, group=32, ldw=0, dt=F32, sdt=BF16, null=(), off=0):
    b = (ctypes.c_uint8 * 4096)()
    p = ctypes.addressof(b)
    ptr = {n: None if n in null else p + (off if n == "W" else 0) for n in ("W", "codes", "scales")}
    return lib.symplex_b200_int4_quantize(ptr["W"], ptr["codes"], ptr["scales"], None, N, K, group, ldw, dt, sdt, None)


@pytest.mark.parametrize("bad", [
    dict(M=-1), dict(M=65), dict(N=-1), dict(K=0), dict(K=1 << 30), dict(N=1 << 31), dict(group=0), dict(group=-32), dict(group=48),
    dict(group=1 << 30), dict(lda=63), dict(ldq=31), dict(ldc=3), dict(sdt=10), dict(odt=3), dict(act=6), dict(act=-1),
    dict(null=("A",)), dict(null=("codes",)), dict(null=("scales",)), dict(null=("C",)), dict(off=1),
])
def test_matvec_refuses(lib, bad):
    assert _matvec(lib, **bad) == _capi.ERR_INVALID
    assert _capi.last_error() != "no error"


@pytest.mark.parametrize("bad", [
    dict(N=-1), dict(K=0), dict(K=-5), dict(group=33), dict(ldw=63), dict(dt=10), dict(sdt=10), dict(null=("W",)), dict(null=("codes",)),
    dict(null=("scales",)), dict(off=2),
])
def test_quantize_refuses(lib, bad):
    assert _quantize(lib, **bad) == _capi.ERR_INVALID
    assert _capi.last_error() != "no error"


def test_nothing_to_do(lib):
    assert _matvec(lib, M=0) == 0 and _matvec(lib, N=0) == 0 and _quantize(lib, N=0) == 0


@pytest.mark.skipif(torch.cuda.is_available(), reason="needs a box without a GPU")
def test_without_a_gpu_it_fails_loudly(lib):
    assert _matvec(lib) in (_capi.ERR_DRIVER, _capi.ERR_EXEC)
    assert _quantize(lib) in (_capi.ERR_DRIVER, _capi.ERR_EXEC)


def test_python_refuses_host_tensors():
    with pytest.raises(ValueError, match="CUDA"):
        sx.int4_quantize(torch.zeros(4, 64))
    with pytest.raises(ValueError, match="CUDA"):
        sx.int4_matvec(torch.zeros(64, dtype=torch.bfloat16), torch.zeros(4, 32, dtype=torch.uint8), torch.ones(4, 1))
