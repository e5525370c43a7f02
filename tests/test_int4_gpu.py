"""Products with 4-bit weights on the GPU against the dequantised product in 64 bits.

code - zero and x are exact in the product and sums are 32-bit: with u = 2^-24, a sum whose longest chain of additions has
d steps is off by at most d u times the sum of its terms' magnitudes (tensor core sums, whose alignment drops bits below
the largest term instead of rounding, count two steps an addition). No chain here has more than K + 64 steps. The result is
rounded once: half a step of its type (bf16 2^-8, fp32 2^-24).
"""
import pytest
import torch

import symplex_b200 as sx

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
BF, F32 = torch.bfloat16, torch.float32


def _case(m, n, k, group, zeros, seed=0, sdt=BF):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(m, k, generator=g, device=DEV).to(BF)
    codes = torch.randint(0, 256, (n, (k + 1) // 2), generator=g, device=DEV, dtype=torch.uint8)
    groups = -(-k // group)
    scales = (0.01 + 0.02 * torch.rand(n, groups, generator=g, device=DEV)).to(sdt)
    z = torch.randint(0, 16, (n, groups), generator=g, device=DEV, dtype=torch.uint8) if zeros else None
    return x, codes, scales, z


def _dense(codes, scales, zeros, k, group):
    n = codes.shape[0]
    w = torch.empty(n, 2 * codes.shape[1], dtype=torch.float64, device=codes.device)
    w[:, 0::2] = (codes % 16).double()
    w[:, 1::2] = (codes // 16).double()
    w = w[:, :k]
    at = torch.arange(k, device=codes.device) // group
    w = w - (zeros.double()[:, at] if zeros is not None else 8.0)
    return w * scales.double()[:, at]


def _check(y, x, w, bias=None):
    ref = x.double() @ w.t()
    terms = x.double().abs() @ w.abs().t()
    if bias is not None:
        ref = ref + bias.double()
        terms = terms + bias.double().abs()
    tol = (2 * x.shape[-1] + 64) * U * terms
    tol = tol * 1.01 + HALF[y.dtype] * ref.abs() + 1e-38
    err = (y.double() - ref).abs()
    assert bool((err <= tol).all()), f"worst {float((err / tol).max()):.3f} of the bound"
    # the bound above is that of the longest chain; what real chains leave is near the rounding of the result itself
    rel = float(err.norm() / ref.norm())
    assert rel <= HALF[y.dtype] + 1e-5


@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 16, 17, 33, 64])
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("zeros", [False, True])
def test_rows_and_groups(m, group, zeros):
    n, k = 200, 1024
    x, codes, scales, z = _case(m, n, k, group, zeros, seed=m + group)
    _check(sx.int4_matvec(x, codes, scales, z, group_size=group), x, _dense(codes, scales, z, k, group))


@pytest.mark.parametrize("n,k,group", [
    (1, 32, 32), (1, 1, 32), (3, 2, 32), (15, 33, 32), (16, 100, 64), (17, 127, 128), (129, 255, 32), (64, 4096, 4096), (40, 4096, 8192),
    (1000, 1056, 32), (777, 2080, 64), (130, 11008, 128), (2500, 512, 64), (33, 16384, 128), (5000, 96, 32), (9, 30000, 32), (64, 544, 96),
])
@pytest.mark.parametrize("m", [1, 5])
@pytest.mark.parametrize("zeros", [False, True])
def test_sizes(m, n, k, group, zeros):
    x, codes, scales, z = _case(m, n, k, group, zeros, seed=n + k)
    w = _dense(codes, scales, z, k, group)
    _check(sx.int4_matvec(x, codes, scales, z, group_size=group), x, w)
    _check(sx.int4_matvec(x, codes, scales, z, group_size=group, out_dtype=F32), x, w)


@pytest.mark.parametrize("m,n,k,group,zeros", [
    (8, 700, 8192, 128, False), (16, 20000, 8192, 64, True), (9, 4736, 5024, 32, True), (16, 33, 16384, 128, False), (29, 5001, 8192, 32, False),
    (5, 9000, 16416, 32, True), (64, 1500, 12320, 32, True), (16, 300, 20480, 64, True), (3, 2000, 131072, 128, False), (6, 25000, 1056, 96, True),
])
def test_rows_of_a_that_do_not_fit_into_shared_memory(m, n, k, group, zeros):
    """A spread over clusters of 2, 4 and 8 CTAs (stretches of k of unequal length, CTAs with none), and in slabs."""
    x, codes, scales, z = _case(m, n, k, group, zeros, seed=k + m)
    w = _dense(codes, scales, z, k, group)
    y = sx.int4_matvec(x, codes, scales, z, group_size=group)
    _check(y, x, w)
    assert torch.equal(y, sx.int4_matvec(x, codes, scales, z, group_size=group))
    b = torch.randn(n, device=DEV)
    _check(sx.int4_matvec(x, codes, scales, z, group_size=group, bias=b, out_dtype=F32), x, w, b)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("e", [100, -100])
def test_powers_of_two_go_through(group, e):
    """x 2^e with scales 2^-e is the same product, bit by bit; codes equal to their zero give an exact 0."""
    x, codes, scales, z = _case(5, 100, 1024, group, True, seed=group)
    want = sx.int4_matvec(x, codes, scales, z, group_size=group, out_dtype=F32)
    assert torch.equal(sx.int4_matvec(x * 2.0 ** e, codes, scales * 2.0 ** -e, z, group_size=group, out_dtype=F32), want)
    z[7] = 5
    codes[7] = 0x55
    assert not sx.int4_matvec(x, codes, scales, z, group_size=group)[:, 7].any()


@pytest.mark.parametrize("sdt", [BF, F32])
@pytest.mark.parametrize("odt", [BF, F32])
def test_types(sdt, odt):
    x, codes, scales, z = _case(3, 500, 768, 128, True, sdt=sdt)
    y = sx.int4_matvec(x, codes, scales, z, out_dtype=odt)
    assert y.dtype == odt
    _check(y, x, _dense(codes, scales, z, 768, 128))


@pytest.mark.parametrize("act,f", [
    ("relu", torch.relu), ("gelu", lambda t: torch.nn.functional.gelu(t, approximate="tanh")), ("sigmoid", torch.sigmoid),
    ("tanh", torch.tanh), ("silu", torch.nn.functional.silu), ("none", lambda t: t),
])
@pytest.mark.parametrize("m", [1, 9])
def test_bias_and_activation(act, f, m):
    x, codes, scales, z = _case(m, 300, 512, 64, False)
    bias = torch.randn(300, device=DEV)
    w = _dense(codes, scales, z, 512, 64)
    _check(sx.int4_matvec(x, codes, scales, group_size=64, bias=bias, out_dtype=F32), x, w, bias)
    y = sx.int4_matvec(x, codes, scales, group_size=64, bias=bias, activation=act, out_dtype=F32)
    pre = x.double() @ w.t() + bias.double()
    # slopes are at most 1.13 (gelu), so the error in front passes through, with a few roundings of the functions themselves
    tol = 1.13 * ((2 * 512 + 64) * U * (x.double().abs() @ w.abs().t() + bias.double().abs())) + 2e-6 * (1 + pre.abs())
    assert bool(((y.double() - f(pre)).abs() <= tol).all())


def test_one_row_as_a_vector_and_out():
    x, codes, scales, z = _case(1, 64, 256, 128, False)
    y = sx.int4_matvec(x, codes, scales)
    v = sx.int4_matvec(x[0], codes, scales)
    assert v.shape == (64,) and torch.equal(v, y[0])
    out = torch.empty(1, 64, device=DEV)
    assert sx.int4_matvec(x, codes, scales, out=out) is out
    _check(out, x, _dense(codes, scales, z, 256, 128))


@pytest.mark.parametrize("pad_x,pad_c,shift", [(8, 16, 0), (1, 0, 0), (0, 1, 0), (0, 0, 1), (3, 5, 7), (0, 8, 4)])
def test_strides_and_alignment(pad_x, pad_c, shift):
    m, n, k = 4, 70, 640
    x, codes, scales, z = _case(m, n, k, 128, True)
    w = _dense(codes, scales, z, k, 128)
    xf = torch.full((m * (k + pad_x) + shift,), float("nan"), device=DEV, dtype=BF)
    xv = xf[shift:].view(m, k + pad_x)[:, :k]
    xv.copy_(x)
    cf = torch.zeros(n * (k // 2 + pad_c) + shift, device=DEV, dtype=torch.uint8)
    cv = cf[shift:].view(n, k // 2 + pad_c)[:, :k // 2]
    cv.copy_(codes)
    sf = torch.cat([scales.view(-1)[:1], scales.view(-1)])[1:].view_as(scales)
    zf = torch.cat([z.view(-1)[:1], z.view(-1)])[1:].view_as(z)
    _check(sx.int4_matvec(xv, cv, sf, zf), x, w)
    _check(sx.int4_matvec(x, codes, scales, z), x, w)
    ct = codes.t().contiguous().t()
    _check(sx.int4_matvec(x, ct, scales, z), x, w)


def test_only_its_rows_are_written():
    x, codes, scales, z = _case(3, 50, 256, 64, False)
    flat = torch.full((3 * 50 + 16,), float("nan"), device=DEV)
    sx.int4_matvec(x, codes, scales, group_size=64, out=flat[:150].view(3, 50))
    assert bool(flat[:150].isfinite().all()) and bool(flat[150:].isnan().all())


def test_values_that_are_not_finite():
    x, codes, scales, z = _case(3, 128, 512, 128, False)
    want = sx.int4_matvec(x, codes, scales)
    x2 = x.clone()
    x2[1, 100] = float("nan")
    y = sx.int4_matvec(x2, codes, scales)
    assert bool(y[1].isnan().all()) and torch.equal(y[0], want[0]) and torch.equal(y[2], want[2])
    s2 = scales.clone()
    s2[7, 2] = float("nan")
    y = sx.int4_matvec(x, codes, s2)
    assert bool(y[:, 7].isnan().all()) and torch.equal(y[:, 8:], want[:, 8:]) and torch.equal(y[:, :7], want[:, :7])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("n,k,group", [(5, 128, 128), (33, 96, 32), (7, 101, 64), (64, 1000, 128), (1, 1, 32)])
def test_quantizer(dtype, symmetric, n, k, group):
    g = torch.Generator(device=DEV).manual_seed(n + k)
    w = (torch.randn(n, k, generator=g, device=DEV) * 0.05).to(dtype)
    w[0, : k // 2] = 0
    for sdt in (BF, F32):
        codes, scales, zeros = sx.int4_quantize(w, group, symmetric=symmetric, scale_dtype=sdt)
        assert scales.dtype == sdt and (zeros is None) == symmetric
        back = _dense(codes, scales, zeros, k, group)
        at = torch.arange(k, device=DEV) // group
        s = scales.double()[:, at]
        # half a step of the code, plus what the rounded scale cuts off at the ends of the range (15 codes of 2^-8 each)
        assert bool(((back - w.double()).abs() <= s * (0.5 + 16 * 2.0 ** -8 + 1e-6)).all())
        if zeros is not None:
            assert int(zeros.max()) <= 15
    # codes against the rule, in 64 bits on the rounded scale; ties aside (none in random values)
    q = torch.round(w.double() / s + (zeros.double()[:, at] if zeros is not None else 8.0)).clamp(0, 15)
    near = ((w.double() / s) - torch.floor(w.double() / s) - 0.5).abs() < 1e-5
    lo = torch.stack([codes % 16, codes // 16], 2).view(n, -1)[:, :k].double()
    assert bool(((lo == q) | near).all())


def test_quantizer_of_rows_that_are_not_finite_and_views():
    w = torch.randn(6, 256, device=DEV)
    w[2, 130] = float("inf")
    w[4, 3] = float("nan")
    codes, scales, _ = sx.int4_quantize(w, 128)
    bad = torch.zeros(6, 2, dtype=torch.bool, device=DEV)
    bad[2, 1] = bad[4, 0] = True
    assert torch.equal(scales.isnan(), bad)
    big = torch.randn(6, 300, device=DEV)
    a, b = sx.int4_quantize(big[:, 3:259], 128), sx.int4_quantize(big[:, 3:259].contiguous(), 128)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_quantize_then_multiply():
    w = (torch.randn(1000, 2048, device=DEV) * 0.03).to(BF)
    x = torch.randn(4, 2048, device=DEV).to(BF)
    for sym in (True, False):
        packed = sx.int4_quantize(w, 64, symmetric=sym)
        y = sx.int4_matvec(x, *packed, group_size=64, out_dtype=F32)
        _check(y, x, _dense(*packed, 2048, 64))
        full = x.double() @ w.double().t()
        assert float((y.double() - full).norm() / full.norm()) < 0.15  # 4 bits: a step of about a seventh of the group's largest


def test_empty():
    x, codes, scales, z = _case(2, 16, 64, 32, False)
    assert sx.int4_matvec(x[:0], codes, scales, group_size=32).shape == (0, 16)
    assert sx.int4_matvec(x, codes[:0], scales[:0], group_size=32).shape == (2, 0)


def test_streams_and_graphs():
    x, codes, scales, z = _case(4, 3000, 1024, 64, True)
    want = sx.int4_matvec(x, codes, scales, z, group_size=64)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = sx.int4_matvec(x, codes, scales, z, group_size=64, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(got, want)
    xs = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = sx.int4_matvec(xs, codes, scales, z, group_size=64)
    for k in range(3):
        xs.copy_(x.roll(k, 0))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want.roll(k, 0))
    many = [sx.int4_matvec(x, codes, scales, z, group_size=64) for _ in range(20)]
    assert all(torch.equal(a, want) for a in many)


def test_refusals():
    x, codes, scales, z = _case(2, 16, 64, 32, True)
    for call in (lambda: sx.int4_matvec(x.float(), codes, scales, group_size=32), lambda: sx.int4_matvec(x, codes, scales, group_size=48),
                 lambda: sx.int4_matvec(x, codes, scales, group_size=64), lambda: sx.int4_matvec(x, codes[:, :16], scales, group_size=32),
                 lambda: sx.int4_matvec(x, codes.int(), scales, group_size=32), lambda: sx.int4_matvec(x, codes, scales.half(), group_size=32),
                 lambda: sx.int4_matvec(x, codes, scales, z.int(), group_size=32), lambda: sx.int4_matvec(x, codes, scales, z[:8], group_size=32),
                 lambda: sx.int4_matvec(x.expand(65, 2, 64)[:, 0], codes, scales, group_size=32),
                 lambda: sx.int4_matvec(x, codes, scales, group_size=32, bias=torch.zeros(16, device=DEV, dtype=BF)),
                 lambda: sx.int4_matvec(x, codes, scales, group_size=32, activation="softplus"),
                 lambda: sx.int4_matvec(x, codes, scales, group_size=32, out_dtype=torch.float16),
                 lambda: sx.int4_matvec(x, codes, scales, group_size=32, out=torch.empty(16, 2, device=DEV).t()),
                 lambda: sx.int4_matvec(x[:, :0], codes[:, :0], scales[:, :0]),
                 lambda: sx.int4_quantize(x.half()), lambda: sx.int4_quantize(x, 16), lambda: sx.int4_quantize(x[0]),
                 lambda: sx.int4_quantize(x, scale_dtype=torch.float16)):
        with pytest.raises(ValueError):
            call()
