"""Gradients of rows that are sure of their target, against the definition in 64 bits.

The target's entry of G is p - 1 = exp(l - lse) - 1, so an absolute error of l - lse is an error relative to 1, not to 1 - p. What the
interface leaves, u = 2^-24: both passes form a logit by the same sums in the same order, and where such a row has its mass on one
word, lse is log(1 + rest) above that very logit: what the tensor core drops of it is dropped on both sides and cancels (of the others,
at most 16 k-blocks' worth of 9.8e-7 l per 512 values, it changes `rest` by a relative 2e-4 at these sizes). The sum 1 + rest takes at
most 20 rounded additions behind the target's (8 strips of a tile, 12 where parts are joined), lse is rounded once to u |lse|, 2^x in
the backward pass is good to 4 u. So the entry is off by E = (|lse| + 24) u, here 2.4e-6 at 1 - p = 1e-3 to 1e-5. G and the result
are rounded to half a step each (bf16 2^-8 relative, fp32 less than that).
"""
import math

import pytest
import torch

import symplex_b200 as sx

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("t,h,v,dtype", [
    (1, 8192, 3000, BF), (40, 4096, 2000, BF), (64, 5000, 9001, BF), (100, 4096, 20000, BF), (128, 2056, 1500, BF),  # up to 128 tokens
    (300, 8192, 3000, BF), (200, 4104, 20011, BF), (700, 6144, 20000, BF), (900, 4096, 5000, BF),                    # pairs, in segments
    (200, 2048, 3000, BF), (300, 4096, 20000, BF), (40, 1000, 3000, BF), (1300, 512, 17000, BF),                     # one sum
    (300, 1024, 20011, BF), (200, 768, 9000, BF), (256, 2048, 30000, BF), (1100, 1104, 17000, BF),                   # 256-row tiles
    (1300, 2048, 17000, BF), (4096, 2048, 21500, BF),  # 512-row tiles, one sum (the last piece of the second: 256-row ones)
    (2100, 4104, 40000, BF),                                                                                         # pieces of the vocabulary
    (100, 4096, 2000, F32), (300, 1000, 5000, F32),
])
def test_the_target_s_entry(t, h, v, dtype):
    g = torch.Generator(device=DEV).manual_seed(t + h)
    w = (torch.randn(v, h, generator=g, device=DEV) * 1.5 / math.sqrt(h)).to(dtype)
    targets = torch.randperm(v, generator=g, device=DEV)[:t]
    want = math.log(v) + 6.9 + 4.6 * torch.rand(t, 1, generator=g, device=DEV)  # the target's logit: 1 - p from 1e-3 to 1e-5
    wt = w[targets].float()
    x = (wt * (want / wt.square().sum(1, keepdim=True))).to(dtype)
    loss, lse = sx.linear_cross_entropy(x, w, targets, reduction="sum")
    dx, dw = sx.linear_cross_entropy_backward(torch.ones((), device=DEV), x, w, targets, lse, reduction="sum")
    sx.sync_status()
    xd, wd = x.double(), w.double()
    l = xd @ wd.t()
    ref = torch.logsumexp(l, 1)
    rows = torch.arange(t, device=DEV)
    p = torch.exp(l - ref[:, None])
    p[rows, targets] -= 1  # G
    own = p[rows, targets].abs()
    assert 3e-6 < float(own.min()) and float(own.max()) < 3e-3
    e = (ref.abs() + 24) * U + (2.0 ** -7 * 1.02 + 2e-4) * own
    # along the row's own x (of dW[target]) and its target's w (of dx): a mean over H values, G's entry itself
    xx, ww = xd.square().sum(1), wd[targets].square().sum(1)
    got = (dw[targets].double() * xd).sum(1) / xx
    exact = ((p.t() @ xd)[targets] * xd).sum(1) / xx
    others = ((p.abs().t() @ xd.abs())[targets] * xd.abs()).sum(1) / xx - own  # other rows' shares of that word, rounded alike
    assert bool(((got - exact).abs() <= e + 2.0 ** -7 * others).all()), f"dW: {float(((got - exact).abs() / e).max()):.2f} of the bound"
    got = (dx.double() * wd[targets]).sum(1) / ww
    exact = ((p @ wd) * wd[targets]).sum(1) / ww
    others = ((p.abs() @ wd.abs()) * wd[targets].abs()).sum(1) / ww - own
    assert bool(((got - exact).abs() <= e + 2.0 ** -7 * others).all()), f"dx: {float(((got - exact).abs() / e).max()):.2f} of the bound"
