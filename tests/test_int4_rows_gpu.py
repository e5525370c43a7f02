"""More rows than one 4-bit product takes."""
import pytest
import torch

import symplex_b200 as sx

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_what_the_refusal_says_works():
    g = torch.Generator(device=DEV).manual_seed(0)
    codes, scales, zeros = sx.int4_quantize(torch.randn(200, 512, generator=g, device=DEV), 64)
    x = torch.randn(150, 512, generator=g, device=DEV).bfloat16()
    with pytest.raises(ValueError, match="in parts") as e:
        sx.int4_matvec(x, codes, scales, zeros, group_size=64)
    assert "gemm" not in str(e.value)  # it takes no codes
    y = torch.cat([sx.int4_matvec(part, codes, scales, zeros, group_size=64) for part in x.split(64)])
    for m in (0, 63, 64, 149):
        # a row's sum does not depend on the rows beside it but for the order in which warps share a tile: two roundings of 2^-8
        one = sx.int4_matvec(x[m], codes, scales, zeros, group_size=64).double()
        assert bool(((y[m].double() - one).abs() <= 2.0 ** -7 * one.abs() + 1e-4).all())
