"""Layer norm on the GPU against its definition in 64 bits.

Tolerances are bounds, derived per value: u = 2^-24 is half a step of fp32. Any sum of n terms in fp32 whose longest chain
of additions has d steps is off by at most d u times the sum of the terms' magnitudes; no kernel here has a longer chain
over a row than 64 + n / 32 (32 lanes or more share it), nor one over the rows longer than the rows + 64. The result is
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


def _inputs(rows, cols, dtype, pdtype=None, seed=0, spread=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device=DEV)
    if spread:
        x = x * (0.25 + 3 * torch.rand(rows, 1, generator=g, device=DEV)) + 2 * torch.randn(rows, 1, generator=g, device=DEV)
    dy = torch.randn(rows, cols, generator=g, device=DEV)
    pdtype = pdtype or dtype
    w = (1 + 0.3 * torch.randn(cols, generator=g, device=DEV)).to(pdtype)
    b = (0.3 * torch.randn(cols, generator=g, device=DEV)).to(pdtype)
    return x.to(dtype), dy.to(dtype), w, b


def _stats(x, eps):
    xd = x.double()
    mean = xd.mean(-1, keepdim=True)
    var = (xd - mean).square().mean(-1, keepdim=True)
    d = 64 + x.shape[-1] / 32
    dmean = d * U * xd.abs().mean(-1, keepdim=True)
    rstd = (var + eps) ** -0.5
    drstd = 0.5 * (dmean ** 2 / (var + eps) + (d + 4) * U) + 4 * U  # relative
    return xd, mean, rstd, dmean, drstd


def _check_forward(x, w, b, y, mean, rstd, eps=1e-5):
    xd, m, r, dm, dr = _stats(x, eps)
    wd = w.double() if w is not None else torch.ones(x.shape[-1], device=x.device, dtype=torch.float64)
    bd = b.double() if b is not None else torch.zeros_like(wd)
    xh = (xd - m) * r
    ref = xh * wd + bd
    tol = wd.abs() * r * (dm + 2 * U * (xd.abs() + m.abs())) + (xh * wd).abs() * (dr + 4 * U) + U * ref.abs()
    tol = tol * (1 + HALF[y.dtype]) + HALF[y.dtype] * ref.abs() + 1e-38
    err = (y.double() - ref).abs()
    assert bool((err <= tol).all()), f"worst {float((err / tol).max()):.3f} of the bound"
    if mean is not None:
        assert bool(((mean.double() - m[..., 0]).abs() <= dm[..., 0] + U * m[..., 0].abs() + 1e-38).all())
        assert bool(((rstd.double() - r[..., 0]).abs() <= r[..., 0] * (dr[..., 0] + U)).all())


def _check_backward(dy, x, mean, rstd, w, dx, dw, db):
    xd, gy = x.double(), dy.double()
    m, r = mean.double()[:, None], rstd.double()[:, None]
    wd = w.double() if w is not None else torch.ones(x.shape[-1], device=x.device, dtype=torch.float64)
    n = x.shape[-1]
    d = 64 + n / 32
    xh = (xd - m) * r
    ex = r * 2 * U * (xd.abs() + m.abs()) + 2 * U * xh.abs()
    g = gy * wd
    c1, c2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    dc1 = (d + 3) * U * g.abs().mean(1, keepdim=True)
    dc2 = (d + 5) * U * (g * xh).abs().mean(1, keepdim=True) + (g.abs() * ex).mean(1, keepdim=True)
    ref = r * (g - c1 - xh * c2)
    tol = r * (dc1 + xh.abs() * dc2 + c2.abs() * ex + 5 * U * (g.abs() + c1.abs() + (xh * c2).abs()))
    tol = tol * 1.01 + HALF[dx.dtype] * ref.abs() + 1e-38
    err = (dx.double() - ref).abs()
    assert bool((err <= tol).all()), f"dx: worst {float((err / tol).max()):.3f} of the bound"
    if dw is None:
        return
    depth = x.shape[0] + 64
    for got, terms, more in ((dw, gy * xh, (gy.abs() * ex).sum(0)), (db, gy, 0.0)):
        ref = terms.sum(0)
        tol = depth * U * terms.abs().sum(0) + more
        tol = tol * 1.01 + HALF[got.dtype] * ref.abs() + 1e-38
        err = (got.double() - ref).abs()
        assert bool((err <= tol).all()), f"column sums: worst {float((err / tol).max()):.3f} of the bound"


SHAPES = [(1, 1), (3, 2), (5, 7), (1, 4096), (2, 31), (7, 32), (33, 64), (129, 257), (37, 1000), (21, 1003), (300, 768), (65, 2048),
          (9, 8192), (5, 10000), (3, 16384), (2, 20001), (2, 70000)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype,pdtype", [(BF, BF), (BF, F32), (F32, F32)])
def test_forward_and_backward(rows, cols, dtype, pdtype):
    x, dy, w, b = _inputs(rows, cols, dtype, pdtype, seed=rows * 7 + cols)
    y, mean, rstd = sx.layer_norm(x, w, b, return_stats=True)
    assert y.dtype == dtype and mean.shape == (rows,) and rstd.dtype == torch.float32
    _check_forward(x, w, b, y, mean, rstd)
    dx, dw, db = sx.layer_norm_backward(dy, x, mean, rstd, w)
    assert dx.dtype == dtype and dw.dtype == pdtype and db.shape == (cols,)
    _check_backward(dy, x, mean, rstd, w, dx, dw, db)


@pytest.mark.parametrize("rows", [1, 2, 147, 148, 149, 1000, 4097])
def test_rows(rows):
    x, dy, w, b = _inputs(rows, 256, BF, seed=rows)
    y, mean, rstd = sx.layer_norm(x, w, b, return_stats=True)
    _check_forward(x, w, b, y, mean, rstd)
    _check_backward(dy, x, mean, rstd, w, *sx.layer_norm_backward(dy, x, mean, rstd, w))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_without_parameters(dtype):
    x, dy, w, b = _inputs(50, 384, dtype)
    y, mean, rstd = sx.layer_norm(x, return_stats=True)
    _check_forward(x, None, None, y, mean, rstd)
    dx, dw, db = sx.layer_norm_backward(dy, x, mean, rstd)
    assert dw is None and db is None
    _check_backward(dy, x, mean, rstd, None, dx, None, None)
    _check_backward(dy, x, mean, rstd, None, *sx.layer_norm_backward(dy, x, mean, rstd, param_grads=True))
    _check_forward(x, w, None, sx.layer_norm(x, w), None, None)
    _check_forward(x, None, b, sx.layer_norm(x, None, b), None, None)
    dx, dw, db = sx.layer_norm_backward(dy, x, mean, rstd, w, param_grads=False)
    assert dw is None and db is None
    _check_backward(dy, x, mean, rstd, w, dx, None, None)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cols,pad,shift", [(256, 8, 0), (256, 1, 0), (256, 0, 1), (1000, 24, 3), (4096, 4, 2)])
def test_strides_and_alignment(dtype, cols, pad, shift):
    rows = 19
    def view(t):
        flat = torch.full((rows * (cols + pad) + shift + 8,), float("nan"), device=DEV, dtype=dtype)
        v = flat[shift:shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
        v.copy_(t)
        return flat, v
    x, dy, w, b = _inputs(rows, cols, dtype)
    (_, xv), (_, dyv), (flat, out) = view(x), view(dy), view(torch.zeros_like(x))
    y, mean, rstd = sx.layer_norm(xv, w, b, return_stats=True, out=out)
    assert y is out
    _check_forward(x, w, b, y, mean, rstd)
    keep = torch.ones_like(flat, dtype=torch.bool)
    keep[shift:shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols] = False
    assert bool(flat[keep].isnan().all())  # nothing between or behind the rows is written
    _check_backward(dy, x, mean, rstd, w, *sx.layer_norm_backward(dyv, xv, mean, rstd, w))
    # parameters that are not aligned to 16 bytes
    wv = torch.cat([w[:1], w])[1:]
    _check_forward(x, wv, b, sx.layer_norm(x, wv, b), None, None)
    _check_backward(dy, x, mean, rstd, w, *sx.layer_norm_backward(dy, x, mean, rstd, wv))


def test_other_shapes_and_orders():
    x, dy, w, b = _inputs(24, 96, BF)
    x3 = x.view(2, 12, 96)
    y, mean, rstd = sx.layer_norm(x3, w, b, return_stats=True)
    assert y.shape == x3.shape and mean.shape == (2, 12)
    _check_forward(x, w, b, y.view(24, 96), mean.view(-1), rstd.view(-1))
    dx, dw, db = sx.layer_norm_backward(dy.view(2, 12, 96), x3, mean, rstd, w)
    assert dx.shape == x3.shape
    _check_backward(dy, x, mean.view(-1), rstd.view(-1), w, dx.view(24, 96), dw, db)
    xt = x.t().contiguous().t()  # columns contiguous: read through a copy
    assert torch.equal(sx.layer_norm(xt, w, b), y.view(24, 96))
    one = dy[:1].expand(24, 96)  # a broadcast gradient
    dx2, dw2, db2 = sx.layer_norm_backward(one, x, mean.view(-1), rstd.view(-1), w)
    _check_backward(one.contiguous(), x, mean.view(-1), rstd.view(-1), w, dx2, dw2, db2)
    v = x[0]
    y1, m1, r1 = sx.layer_norm(v, w, b, return_stats=True)
    assert y1.shape == (96,) and m1.shape == ()
    assert torch.equal(y1, y.view(24, 96)[0])


def test_in_place():
    for cols in (512, 20001):
        x, dy, w, b = _inputs(11, cols, BF)
        want = sx.layer_norm(x, w, b)
        z = x.clone()
        assert sx.layer_norm(z, w, b, out=z) is z
        assert torch.equal(z, want)


def test_no_rows():
    x = torch.empty(0, 64, device=DEV)
    w = torch.ones(64, device=DEV)
    y, mean, rstd = sx.layer_norm(x, w, return_stats=True)
    assert y.shape == (0, 64) and mean.shape == (0,)
    dx, dw, db = sx.layer_norm_backward(x, x, mean, rstd, w)
    assert dx.shape == (0, 64) and not dw.any() and not db.any()


def test_far_mean_and_constant_rows():
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(16, 4096, generator=g, device=DEV) + 1000.0  # a mean a thousand deviations away
    y, mean, rstd = sx.layer_norm(x, return_stats=True)
    _check_forward(x, None, None, y, mean, rstd)
    c = torch.full((4, 4096), 3.0, device=DEV)
    y, mean, rstd = sx.layer_norm(c, return_stats=True)
    assert not y.any() and bool((mean == 3).all())
    assert bool(((rstd - 1e-5 ** -0.5).abs() <= 1e-4).all())
    y = sx.layer_norm(c, eps=0.0)  # 0 * inf, as in the formula
    assert bool(y.isnan().all())


def test_values_that_are_not_finite_stay_in_their_row():
    x, dy, w, b = _inputs(40, 512, BF)
    want = sx.layer_norm(x, w, b)
    x[3, 5] = float("inf")
    x[17, 0] = float("nan")
    y, mean, rstd = sx.layer_norm(x, w, b, return_stats=True)
    assert bool(y[3].isnan().all()) and bool(y[17].isnan().all())
    good = [r for r in range(40) if r not in (3, 17)]
    assert torch.equal(y[good], want[good])
    dx, _, _ = sx.layer_norm_backward(dy, x, mean, rstd, w)
    assert bool(dx[good].isfinite().all()) and bool(dx[17].isnan().all())


def test_gradient_against_differences():
    """d/dx of sum(dy * norm(x) w + b), central differences of the definition in 64 bits: the step h leaves an error of
    h^2 times the third derivative (under 1e-6 here), fp32 the rest."""
    x, dy, w, b = _inputs(3, 24, F32, spread=False)
    _, mean, rstd = sx.layer_norm(x, w, b, return_stats=True)
    dx, dw, db = sx.layer_norm_backward(dy, x, mean, rstd, w)

    def f(xx, ww, bb):
        m = xx.mean(1, keepdim=True)
        v = (xx - m).square().mean(1, keepdim=True)
        return float((dy.double() * ((xx - m) / (v + 1e-5).sqrt() * ww + bb)).sum())

    xd, wd, bd, h = x.double(), w.double(), b.double(), 1e-4
    for i, j in ((0, 0), (1, 7), (2, 23)):
        e = torch.zeros_like(xd)
        e[i, j] = h
        assert abs((f(xd + e, wd, bd) - f(xd - e, wd, bd)) / (2 * h) - float(dx[i, j])) < 1e-5
    for j in (0, 11, 23):
        e = torch.zeros_like(wd)
        e[j] = h
        assert abs((f(xd, wd + e, bd) - f(xd, wd - e, bd)) / (2 * h) - float(dw[j])) < 1e-5
        assert abs((f(xd, wd, bd + e) - f(xd, wd, bd - e)) / (2 * h) - float(db[j])) < 1e-5


def test_same_bits_every_time():
    x, dy, w, b = _inputs(3000, 776, BF)
    y, mean, rstd = sx.layer_norm(x, w, b, return_stats=True)
    first = sx.layer_norm_backward(dy, x, mean, rstd, w)
    for _ in range(5):
        assert all(torch.equal(a, c) for a, c in zip(first, sx.layer_norm_backward(dy, x, mean, rstd, w)))


def test_on_another_stream_and_in_a_graph():
    x, dy, w, b = _inputs(500, 1024, BF)
    want = sx.layer_norm(x, w, b, return_stats=True)
    wantg = sx.layer_norm_backward(dy, x, want[1], want[2], w)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = sx.layer_norm(x, w, b, return_stats=True, stream=s.cuda_stream)
    gotg = sx.layer_norm_backward(dy, x, got[1], got[2], w, stream=s.cuda_stream)
    s.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(want + wantg, got + gotg))
    graph = torch.cuda.CUDAGraph()
    xs, dys = torch.zeros_like(x), torch.zeros_like(dy)
    with torch.cuda.graph(graph):
        y, m, r = sx.layer_norm(xs, w, b, return_stats=True)
        grads = sx.layer_norm_backward(dys, xs, m, r, w)
    for k in range(3):
        xs.copy_(x.roll(k, 0))
        dys.copy_(dy.roll(k, 0))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0].roll(k, 0)) and torch.equal(grads[0], wantg[0].roll(k, 0))
        _check_backward(dys, xs, m, r, w, *grads)


def test_two_streams_at_once():
    cases = [_inputs(2000, 1536, BF, seed=k) for k in range(2)]
    stats = [sx.layer_norm(x, w, b, return_stats=True) for x, dy, w, b in cases]
    want = [sx.layer_norm_backward(dy, x, m, r, w) for (x, dy, w, b), (y, m, r) in zip(cases, stats)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(10):
        for k, (x, dy, w, b) in enumerate(cases):
            with torch.cuda.stream(streams[k]):
                got[k].append(sx.layer_norm_backward(dy, x, stats[k][1], stats[k][2], w))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(a, c) for one in got[k] for a, c in zip(want[k], one))


def test_refusals():
    x, dy, w, b = _inputs(4, 64, BF)
    y, mean, rstd = sx.layer_norm(x, w, b, return_stats=True)
    for call in (lambda: sx.layer_norm(x.half()), lambda: sx.layer_norm(x, w[:32]), lambda: sx.layer_norm(x, w.double()),
                 lambda: sx.layer_norm(x, w, b.float()), lambda: sx.layer_norm(x, eps=-1.0), lambda: sx.layer_norm(x, out=y[:2]),
                 lambda: sx.layer_norm(x, out=torch.empty(64, 4, device=DEV, dtype=BF).t()), lambda: sx.layer_norm(x[:, :0]),
                 lambda: sx.layer_norm(x, w.cpu()), lambda: sx.layer_norm_backward(dy[:2], x, mean, rstd, w),
                 lambda: sx.layer_norm_backward(dy, x, mean[:2], rstd, w), lambda: sx.layer_norm_backward(dy, x, mean.double(), rstd, w),
                 lambda: sx.layer_norm_backward(dy.float(), x, mean, rstd, w)):
        with pytest.raises(ValueError):
            call()
