"""When two matrices share memory (csrc/byte_rows.h), against sets of addresses."""
import ctypes
import os
import random
import shutil
import subprocess
import time

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "symplex_b200", "csrc")


@pytest.fixture(scope="module")
def share(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    d = tmp_path_factory.mktemp("byte_rows")
    src = d / "t.cpp"
    src.write_text('#include "byte_rows.h"\nextern "C" int share(long long a, long long ra, long long ba, long long sa, long long b, long long rb, '
                   'long long bb, long long sb) { return sx::share_bytes({(const void*)a, ra, ba, sa}, {(const void*)b, rb, bb, sb}); }\n'
                   'extern "C" long long one(long long p, long long bytes) { return sx::one_row((const void*)p, bytes).rows; }\n')
    subprocess.run([gxx, "-std=c++17", "-shared", "-fPIC", "-I", CSRC, "-o", str(d / "t.so"), str(src)], check=True)
    lib = ctypes.CDLL(str(d / "t.so"))
    lib.share.argtypes = [ctypes.c_longlong] * 8
    lib.one.argtypes = [ctypes.c_longlong] * 2
    return lib


def _addresses(p, rows, width, stride):
    return {p + i * stride + k for i in range(rows) for k in range(width)}


@pytest.mark.parametrize("one_stride", [False, True])
def test_against_sets(share, one_stride):
    rng = random.Random(0)
    seen = [0, 0]
    for _ in range(20000):
        a, b = ((rng.randrange(64, 160), rng.randrange(0, 5), w := rng.randrange(0, 9), w + rng.choice([0, 0, 1, 4, 13, 40])) for _ in range(2))
        if one_stride:
            a, b = a[:3] + (max(a[3], b[3]),), b[:3] + (max(a[3], b[3]),)
        want = bool(_addresses(*a) & _addresses(*b))
        assert bool(share.share(*a, *b)) == want, (a, b)
        seen[want] += 1
    assert min(seen) > 2000


def test_views_of_a_long_buffer_are_told_apart_at_once(share):
    """Two halves of the same rows: not one look at each of a billion of them on every call."""
    start = time.perf_counter()
    for _ in range(1000):
        assert not share.share(1 << 20, 1 << 30, 256, 512, (1 << 20) + 256, 1 << 30, 256, 512)
        assert share.share(1 << 20, 1 << 30, 256, 512, (1 << 20) + 254, 1 << 30, 256, 512)
    assert time.perf_counter() - start < 1


def test_nothing_shares_with_a_missing_operand(share):
    assert share.one(0, 100) == 0 and share.one(64, 100) == 1
    assert not share.share(0, 0, 100, 100, 0, 1, 1000, 1000)
