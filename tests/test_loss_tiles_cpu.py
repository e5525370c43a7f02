"""The rules that pick the loss' tiles (csrc/ce_tiles.h), without a GPU."""
import ctypes
import os
import random
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "symplex_b200", "csrc")
SMS = 148


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    d = tmp_path_factory.mktemp("ce_tiles")
    src = d / "t.cpp"
    src.write_text("""#include "ce_tiles.h"
using namespace sx;
extern "C" void forward(long long T, long long V, long long H, int sms, int mode, int* out) {
  const CeTiles t = ce_forward_tiles(T, V, H, sms, mode);
  out[0] = t.mb, out[1] = t.segments, out[2] = t.bn, out[3] = ce_parts(t, V), out[4] = ce_parts_most(T, V);
}
extern "C" void gradient(long long T, long long V, long long H, long long n, int lo, int sms, int mode, int* out) {
  const CeTiles t = ce_gradient_tiles(T, V, H, n, lo != 0, sms, mode);
  out[0] = t.mb, out[1] = t.segments, out[2] = t.bn;
}
extern "C" int segment() { return CE_SEGMENT * 64; }
""")
    subprocess.run([gxx, "-std=c++17", "-shared", "-fPIC", "-I", CSRC, "-o", str(d / "t.so"), str(src)], check=True)
    lib = ctypes.CDLL(str(d / "t.so"))
    ll, i, p = ctypes.c_longlong, ctypes.c_int, ctypes.POINTER(ctypes.c_int)
    lib.forward.argtypes = [ll, ll, ll, i, i, p]
    lib.gradient.argtypes = [ll, ll, ll, ll, i, i, i, p]

    def forward(T, V, H, mode=-1, sms=SMS):
        out = (ctypes.c_int * 5)()
        lib.forward(T, V, H, sms, mode, out)
        return dict(zip(("mb", "segments", "bn", "parts", "most"), out))

    def gradient(T, V, H, n, mode=-1, sms=SMS):
        out = (ctypes.c_int * 3)()
        lib.gradient(T, V, H, n, int(T <= 64), sms, mode, out)
        return dict(zip(("mb", "segments", "bn"), out))

    forward.segment = lib.segment()
    return forward, gradient


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def test_forms(rules):
    """What the kernels rely on: instances that exist, room for the parts, the same sums in both passes."""
    forward, gradient = rules
    rng = random.Random(0)
    for _ in range(20000):
        T, V, H = _log(rng, 1, 20000), _log(rng, 1, 300000), _log(rng, 1, 20000)
        mode, sms = rng.choice([-1, -1, 0, 1, 2]), rng.choice([148, 148, 132, 74])
        f = forward(T, V, H, mode, sms)
        assert f["parts"] <= f["most"], (T, V, H, mode)
        assert f["mb"] != 1 or f["segments"]            # 256-row tiles: one form
        assert not (f["segments"] and f["mb"] == 2)     # 512-row tiles have no second accumulator
        if f["mb"] == 0:
            assert T <= 128 and f["bn"] % 16 == 0 and (64 if f["segments"] else 32) <= f["bn"] <= 256
        n = _log(rng, 1, V)
        g = gradient(T, V, H, n, mode, sms)
        assert not (g["segments"] and g["mb"] == 2)
        assert g["segments"] == (f["segments"] and H > forward.segment), (T, V, H, n, mode)
        if T <= 64:
            assert g["mb"] == 0
        if g["mb"] == 0:
            assert T <= 128 and g["bn"] % 64 == 0 and g["bn"] <= 256


def test_the_size_of_the_recorded_hang(rules):
    """256-row tiles, in segments: the kernel that it ran in has no instance any more."""
    forward, _ = rules
    assert forward(3815, 26330, 1104)["mb"] == 1 and forward(3815, 26330, 1104)["segments"]
    with open(os.path.join(CSRC, "ce_pair_sm100.cu")) as f:
        code = f.read()
    assert "launch<CE_LSE, 1>" not in code and code.count("launch<kMode, 1>(") == 1
    at = code.index("launch<kMode, 1>(")
    assert code.rindex("if constexpr (kMode == CE_GRAD)", 0, at) > code.rindex("static int launch_logits", 0, at)


def test_known_sizes(rules):
    forward, gradient = rules
    assert forward(8192, 65536, 4096) == dict(mb=2, segments=0, bn=256, parts=512, most=512)
    assert forward(37, 50257, 1024)["mb"] == 0 and not forward(37, 50257, 1024)["segments"]
    assert forward(2100, 40000, 4104) ["segments"] and gradient(2100, 40000, 4104, 20000)["segments"]
    assert gradient(4096, 65536, 4096, 16384) == dict(mb=2, segments=0, bn=256)
