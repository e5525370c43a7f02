"""4-bit products on every device of the process: what is remembered of a device is that device's."""
import pytest
import torch

import symplex_b200 as sx

pytestmark = pytest.mark.gpu


@pytest.mark.skipif(torch.cuda.is_available() and torch.cuda.device_count() < 2, reason="needs two GPUs")
@pytest.mark.parametrize("m,n,k", [(16, 2000, 8192), (16, 300, 20480), (1, 500, 1024)])
def test_each_device(m, n, k):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(m, k, generator=g).bfloat16()
    codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    scales = torch.rand(n, k // 128, generator=g).bfloat16()
    got = [sx.int4_matvec(x.to(d), codes.to(d), scales.to(d)).cpu() for d in range(torch.cuda.device_count())]
    assert all(torch.equal(got[0], y) for y in got[1:])
