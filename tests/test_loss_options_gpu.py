"""The loss while another thread changes the tuning options of the library."""
import threading

import pytest
import torch

import symplex_b200 as sx
from symplex_b200 import _capi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_the_tile_option_is_read_once_a_call():
    """A pass joins as many parts of a row as its kernel wrote, whatever the option says by then."""
    g = torch.Generator(device=DEV).manual_seed(0)
    w = torch.randn(3001, 64, generator=g, device=DEV).bfloat16()
    x = (torch.randn(300, 64, generator=g, device=DEV) * 0.25).bfloat16()
    targets = torch.randint(0, 3001, (300,), generator=g, device=DEV)
    want = torch.logsumexp(x.double() @ w.double().t(), 1)
    sx.linear_cross_entropy(x, w, targets)
    bad = torch.full((1 << 20,), 0xFF, dtype=torch.uint8, device=DEV)  # NaN where a workspace is read before it is written
    del bad
    lib, stop = _capi.load(), threading.Event()

    def turn():
        k = 0
        while not stop.is_set():
            k ^= 1
            lib.symplex_b200_set_option(b"pair_mode", 1 + k)

    with _capi.option("pair_mode", 1):
        thread = threading.Thread(target=turn)
        thread.start()
        try:
            worst = torch.zeros((), device=DEV, dtype=torch.float64)
            for _ in range(8000):
                _, lse = sx.linear_cross_entropy(x, w, targets)
                worst = torch.maximum(worst, (lse - want).abs().max())
        finally:
            stop.set()
            thread.join()
    sx.sync_status()
    assert float(worst) < 1e-4
