"""A weight that is not finite is seen behind every activation of a 4-bit product."""
import pytest
import torch

import symplex_b200 as sx

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("act", [None, "relu", "gelu", "sigmoid", "tanh", "silu"])
@pytest.mark.parametrize("k", [256, 250])  # the tensor-core form, the one for any K
@pytest.mark.parametrize("m", [1, 20])
def test_nan_passes_through(act, k, m):
    g = torch.Generator(device=DEV).manual_seed(0)
    w = torch.randn(40, k, generator=g, device=DEV)
    w[3, 7], w[11, 100] = float("nan"), float("inf")
    codes, scales, zeros = sx.int4_quantize(w, 64)
    x = torch.randn(m, k, generator=g, device=DEV).bfloat16()
    y = sx.int4_matvec(x, codes, scales, zeros, group_size=64, activation=act)
    bad = torch.zeros(40, dtype=torch.bool, device=DEV)
    bad[3] = bad[11] = True
    assert torch.equal(y.isnan().any(0), bad) and torch.equal(y.isnan().all(0), bad)
    if act == "relu":
        plain = sx.int4_matvec(x, codes, scales, zeros, group_size=64)
        assert torch.equal(y[:, ~bad], torch.relu(plain[:, ~bad]))
