"""Outputs that overlap an operand are refused before anything is launched; interleaved views are not overlaps."""
import pytest
import torch

import symplex_b200 as sx

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


def _product(m=2, n=64, k=64):
    g = torch.Generator(device=DEV).manual_seed(0)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device=DEV, dtype=torch.uint8)
    return torch.randn(m, k, generator=g, device=DEV).to(BF), codes, torch.rand(n, k // 32, generator=g, device=DEV).to(BF)


@pytest.mark.parametrize("m", [1, 2, 16])
def test_a_product_is_not_written_over_its_input(m):
    """Other columns' CTAs still read x when the first ones write."""
    x, codes, scales = _product(m)
    keep = x.clone()
    want = sx.int4_matvec(x, codes, scales, group_size=32)
    with pytest.raises(ValueError, match="overlap"):
        sx.int4_matvec(x, codes, scales, group_size=32, out=x)
    flat = torch.cat([x.reshape(-1), x.reshape(-1)])
    with pytest.raises(ValueError, match="overlap"):
        sx.int4_matvec(flat[:m * 64].view(m, 64), codes, scales, group_size=32, out=flat[64 * m - 8:64 * 2 * m - 8].view(m, 64))
    for part in (codes.view(BF).reshape(-1), scales.reshape(-1)):
        if part.numel() >= m * 64:
            with pytest.raises(ValueError, match="overlap"):
                sx.int4_matvec(x, codes, scales, group_size=32, out=part[:m * 64].view(m, 64))
    assert torch.equal(x, keep)
    out = flat[m * 64:].view(m, 64)  # right behind its input
    assert torch.equal(sx.int4_matvec(flat[:m * 64].view(m, 64), codes, scales, group_size=32, out=out), want)


def test_a_norm_is_written_over_its_input_or_beside_it():
    g = torch.Generator(device=DEV).manual_seed(0)
    buf = torch.randn(40, 128, generator=g, device=DEV).to(BF)
    w = torch.rand(64, generator=g, device=DEV).to(BF)
    x = buf[:, :64]
    want = sx.layer_norm(x.clone(), w)
    flat = buf.clone().view(-1)
    for out in (flat.view(40, 128)[:, 8:72], flat[:40 * 64].view(40, 64)):
        with pytest.raises(ValueError, match="overlap"):
            sx.layer_norm(flat.view(40, 128)[:, :64], w, out=out)
    with pytest.raises(ValueError, match="overlap"):
        sx.layer_norm(flat[:40 * 64].view(40, 64), w, out=flat[64:41 * 64].view(40, 64))
    with pytest.raises(ValueError, match="overlap"):
        sx.layer_norm(x.clone()[:1], w, out=w.view(1, 64))
    assert torch.equal(flat, buf.view(-1))
    beside = buf.clone()
    assert torch.equal(sx.layer_norm(beside[:, :64], w, out=beside[:, 64:]), want)
    assert torch.equal(beside[:, :64], x)
    assert torch.equal(sx.layer_norm(beside[:, :64], w, out=beside[:, :64]), want)
    # strides that are read through a copy do not tie the output to the input
    t = x.t().contiguous().t()
    assert torch.equal(sx.layer_norm(t, w, out=t.as_strided((40, 64), (64, 1))), want)


def test_sizes_that_the_library_refuses_are_the_caller_s():
    x, codes, scales = _product()
    with pytest.raises(ValueError, match="2\\^29"):
        sx.int4_matvec(x, codes, scales[:, :1].contiguous(), group_size=1 << 30)
