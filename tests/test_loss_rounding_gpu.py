"""How much the bf16 gradients of many tokens lose to the rounding of G, beside the results' own rounding.

G's entries are rounded once, independently of one another and with the same distribution as the results are. A row of dx is mostly
its target's entry times a row of W, so a row as a whole is off by one such rounding; over many rows and words the mean square of both
roundings together is twice that of one: 1.41 of the norm (less where several entries share a row). 1.5 leaves 6 % for the chance of a few
hundred rows.
"""
import math

import pytest
import torch

import symplex_b200 as sx

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("t,h,v", [(200, 512, 3000), (700, 768, 9001), (1500, 256, 5001), (300, 4104, 2000), (2100, 136, 40000)])
def test_two_roundings(t, h, v, reduction):
    g = torch.Generator(device=DEV).manual_seed(t)
    w = (torch.randn(v, h, generator=g, device=DEV) * 1.5 / math.sqrt(h)).to(BF)
    targets = torch.randint(0, v, (t,), generator=g, device=DEV)
    x = (torch.randn(t, h, generator=g, device=DEV) + 3 * torch.rand(t, 1, generator=g, device=DEV) * w[targets].float()).to(BF)
    _, lse = sx.linear_cross_entropy(x, w, targets)
    d = torch.rand(t, generator=g, device=DEV) + 0.5 if reduction == "none" else torch.ones((), device=DEV)
    got = sx.linear_cross_entropy_backward(d, x, w, targets, lse, reduction=reduction)
    sx.sync_status()
    p = torch.softmax(x.double() @ w.double().t(), 1)
    p[torch.arange(t, device=DEV), targets] -= 1
    p *= d.double()[:, None] if reduction == "none" else 1 / t
    for a, ref in zip(got, (p @ w.double(), p.t() @ x.double())):
        rounding = (ref.to(BF).double() - ref).norm()
        assert float((a.double() - ref).norm() / rounding) <= 1.5
