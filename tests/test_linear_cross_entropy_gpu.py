"""The loss of a linear head on the GPU against its definition in 64 bits.

Bounds, u = 2^-24. A logit is a sum of H exact products of bf16 values (fp32: products good to 2^-21 by the split into three
tf32 products) in tensor-core fp32, whose additions drop bits instead of rounding them: off by at most
dl = (2 H + 64) u sum|x w| (fp32: 16 u more). lse moves by at most the largest dl of its row, plus the rounding of
2^x and log2 (under 16 u relative) and of lse itself; the sum over V has chains of at most V / 32 + 64 steps.
G = (p - 1hot) s: p is off by p (dl + |lse| 4 u + 16 u); held in the inputs' type (half a step of |G|, fp32: nothing). The
products dx and dW add the chain bound again, and are rounded once. These are bounds of the longest chains and so loose;
beside them the relative error of whole results is held to what rounding G and the result independently gives.
"""
import math

import pytest
import torch

import symplex_b200 as sx
from symplex_b200 import _capi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
BF, F32 = torch.bfloat16, torch.float32


def _inputs(t, h, v, dtype, seed=0, ignored=0.15, sharp=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = (torch.randn(v, h, generator=g, device=DEV) * 1.5 / math.sqrt(h)).to(dtype)
    targets = torch.randint(0, v, (t,), generator=g, device=DEV)
    x = (torch.randn(t, h, generator=g, device=DEV) + sharp * torch.rand(t, 1, generator=g, device=DEV) * w[targets].float()).to(dtype)
    if t > 2:
        targets[torch.rand(t, generator=g, device=DEV) < ignored] = -100
    return x, w, targets


def _logits(x, w):
    xd, wd = x.double(), w.double()
    l = xd @ wd.t()
    dl = (2 * x.shape[1] + 64) * U * (xd.abs() @ wd.abs().t())
    if x.dtype == F32:
        dl = dl + 16 * U * (xd.abs() @ wd.abs().t())
    return l, dl


def _check_loss(x, w, targets, loss, lse, reduction, ignore=-100):
    l, dl = _logits(x, w)
    ref = torch.logsumexp(l, 1)
    tol = dl.max(1).values + (w.shape[0] / 32 + 64 + 32) * U + 4 * U * ref.abs() + 1e-30
    assert bool(((lse.double() - ref).abs() <= tol).all()), f"lse: {float(((lse.double() - ref).abs() / tol).max()):.3f} of the bound"
    counted = targets != ignore
    at = torch.where(counted, targets, 0)[:, None]
    rows = torch.where(counted, ref - l.gather(1, at)[:, 0], 0.0)
    row_tol = torch.where(counted, tol + dl.gather(1, at)[:, 0] + 4 * U * (ref.abs() + rows.abs()), 0.0)
    if reduction == "none":
        assert bool(((loss.double() - rows).abs() <= row_tol).all())
        assert bool((loss[~counted] == 0).all())
        return
    want, wtol = rows.sum(), row_tol.sum()
    if reduction == "mean":
        want, wtol = want / counted.sum(), wtol / counted.sum()
    assert loss.shape == () and abs(float(loss) - float(want)) <= float(wtol + 2 * U * want.abs())


def _check_grads(dloss, x, w, targets, lse, dx, dw, reduction, ignore=-100):
    l, dl = _logits(x, w)
    ls = lse.double()[:, None]
    counted = targets != ignore
    s = dloss.double() * torch.ones(len(targets), device=DEV, dtype=torch.float64)
    if reduction == "mean":
        s = s / max(1, int(counted.sum()))
    s = torch.where(counted, s, 0.0)[:, None]
    p = torch.exp(l - ls)
    onehot = torch.zeros_like(p)
    rows = counted.nonzero()[:, 0]
    onehot[rows, targets[rows]] = 1
    g = (p - onehot) * s
    half = HALF[x.dtype]
    dg = p * (dl + 4 * U * ls.abs() + 16 * U) * s.abs() + 4 * U * g.abs()
    dg = dg * 1.01 + (half if x.dtype == BF else 0) * g.abs()
    extra = 16 * U if x.dtype == F32 else 0
    # p - 1 cancels where a row is sure of its target (a vocabulary of one word: G is 0 and p off by |lse| u): what fp32 leaves
    # of G is relative to p + 1hot, not to G
    b = (p + onehot) * s.abs()
    for got, ref, base, terms, moved, n in (
            (dx, g @ w.double(), b @ w.double().abs(), g.abs() @ w.double().abs(), dg @ w.double().abs(), w.shape[0]),
            (dw, g.t() @ x.double(), b.t() @ x.double().abs(), g.abs().t() @ x.double().abs(), dg.t() @ x.double().abs(), len(targets))):
        assert got.dtype == x.dtype and got.shape == ref.shape
        tol = moved + ((2 * n + 128) * U + extra) * terms * 1.02 + half * ref.abs() * 1.01 + 1e-38
        err = (got.double() - ref).abs()
        assert bool((err <= tol).all()), f"worst {float((err / tol).max()):.3f} of the bound"
        assert float(err.norm()) <= (1.5 * half if x.dtype == BF else 4e-6) * float(ref.norm()) + 2e-6 * float(base.norm())


def _both(t, h, v, dtype, reduction, seed=0, **kw):
    x, w, targets = _inputs(t, h, v, dtype, seed, **kw)
    loss, lse = sx.linear_cross_entropy(x, w, targets, reduction=reduction)
    sx.sync_status()
    _check_loss(x, w, targets, loss, lse, reduction)
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    dloss = torch.randn(t, generator=g, device=DEV) if reduction == "none" else torch.rand((), generator=g, device=DEV) + 0.5
    dx, dw = sx.linear_cross_entropy_backward(dloss, x, w, targets, lse, reduction=reduction)
    sx.sync_status()
    _check_grads(dloss, x, w, targets, lse, dx, dw, reduction)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("t,h,v", [(1, 8, 1), (1, 64, 1000), (5, 16, 7), (64, 64, 256), (130, 72, 300), (257, 128, 513), (300, 200, 2049)])
def test_small(t, h, v, dtype, reduction):
    _both(t, h, v, dtype, reduction, seed=t + v)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("t,h,v", [(1, 1024, 50257), (37, 1024, 50257), (513, 512, 8192), (1030, 264, 5001), (700, 768, 30011), (2049, 256, 4097)])
def test_medium(t, h, v, dtype):
    _both(t, h, v, dtype, "mean", seed=v)


def test_several_pieces():
    _both(4096, 128, 65536, BF, "none", seed=5)


@pytest.mark.parametrize("t,h,v,dtype", [(2049, 136, 40000, BF), (8192, 64, 5000, F32), (3000, 72, 12001, F32), (100, 300, 20011, F32)])
def test_pieces_in_parts(t, h, v, dtype):
    """Pieces of the vocabulary whose product dx is cut over the vocabulary once more, the last piece in fewer or shorter parts."""
    _both(t, h, v, dtype, "mean", seed=v)


@pytest.mark.parametrize("t", [1, 15, 16, 17, 61, 127, 128, 129])
@pytest.mark.parametrize("h,v", [(64, 33), (200, 4736), (136, 40009), (1024, 20000)])
def test_few_tokens(t, h, v):
    _both(t, h, v, BF, "none" if t % 2 else "mean", seed=t)


@pytest.mark.parametrize("t,h,v", [(5, 1032, 300), (128, 2048, 5000), (1, 4096, 9001), (37, 8192, 3000), (130, 4104, 700), (300, 6144, 5001), (600, 8192, 3000)])
def test_long_products_round_in_segments(t, h, v):
    """An accumulator that rounds towards 0 loses half a unit in the last place of its running sum per instruction (16 k) on
    average, always the same way. A segment of 512 is 32 instructions; while its sum runs from 0 to s, that is at most
    1/2 2^-23 s (1 + ... + 32) / 32 = 9.8e-7 s, and all segments together 9.8e-7 of a logit; lse moves by the mean of that over
    its logits, which are no larger than it is (here: most of the mass is on the target's). One sum over 8192 loses 16 times as much.
    (Up to H = 2048 it is one sum, 3.9e-6 by this estimate, which takes every unit at its largest; it is held to 1e-6 too.)
    """
    x, w, targets = _inputs(t, h, v, BF, seed=h, sharp=3.0)
    loss, lse = sx.linear_cross_entropy(x, w, targets, reduction="none")
    sx.sync_status()
    _check_loss(x, w, targets, loss, lse, "none")
    ref = torch.logsumexp(x.double() @ w.double().t(), 1)
    assert float((lse.double() - ref).norm() / ref.norm()) < 1e-6
    d = torch.ones(t, device=DEV)
    _check_grads(d, x, w, targets, lse, *sx.linear_cross_entropy_backward(d, x, w, targets, lse, reduction="none"), "none")


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("t,h,v", [(1, 64, 33), (1, 512, 3000), (2, 256, 1000), (5, 1000, 5001), (33, 136, 700), (64, 512, 9000)])
def test_few_tokens_gradients_are_rounded_once(t, h, v, reduction):
    """G in two bf16 parts is off by 2^-17: beside it the results' own rounding is all there is. A value whose rounding G's error turns
    over (it lies within 2^-17 of a tie: one in 2^8) is off by a whole step instead of half, 3.7 times the mean square: under 1 %
    of the norm; the chains' bound of _check_grads is 2^-13 at these sizes at the most."""
    x, w, targets = _inputs(t, h, v, BF, seed=7 * t + v, ignored=0.0)
    _, lse = sx.linear_cross_entropy(x, w, targets)
    d = torch.full((t,) if reduction == "none" else (), 0.7, device=DEV)
    got = sx.linear_cross_entropy_backward(d, x, w, targets, lse, reduction=reduction)
    sx.sync_status()
    p = torch.exp(x.double() @ w.double().t() - lse.double()[:, None])
    p[torch.arange(t, device=DEV), targets] -= 1
    g = p * (d.double() if reduction == "none" else d.double() / t).reshape(-1, 1)
    for a, ref in zip(got, (g @ w.double(), g.t() @ x.double())):
        rounding = (ref.to(BF).double() - ref).norm()
        assert float((a.double() - ref).norm()) <= 1.02 * float(rounding) + 2.0 ** -13 * float(ref.norm())


@pytest.mark.parametrize("shape", [1, 2])
@pytest.mark.parametrize("t,h,v", [(40, 64, 700), (600, 200, 3001), (1100, 512, 9000)])
def test_both_tile_shapes(t, h, v, shape):
    with _capi.option("pair_mode", shape):
        _both(t, h, v, BF, "sum", seed=t)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("h", [1, 7, 33, 100, 515])
def test_hidden_sizes_that_do_not_align(h, dtype):
    _both(70, h, 401, dtype, "mean", seed=h)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("pad,shift", [(8, 0), (3, 0), (0, 1), (0, 8)])
def test_strides_and_alignment(pad, shift, dtype):
    t, h, v = 50, 128, 700
    x, w, targets = _inputs(t, h, v, dtype)
    def view(a):
        flat = torch.full((a.shape[0] * (h + pad) + shift,), float("nan"), device=DEV, dtype=dtype)
        r = flat[shift:].view(a.shape[0], h + pad)[:, :h]
        r.copy_(a)
        return r
    xv, wv = view(x), view(w)
    tv = torch.stack([targets, targets], 1)[:, 0]
    loss, lse = sx.linear_cross_entropy(xv, wv, tv)
    _check_loss(x, w, targets, loss, lse, "mean")
    d = torch.ones((), device=DEV)
    _check_grads(d, x, w, targets, lse, *sx.linear_cross_entropy_backward(d, xv, wv, tv, lse), "mean")
    wt = w.t().contiguous().t()
    assert torch.equal(sx.linear_cross_entropy(x, wt, targets)[1], sx.linear_cross_entropy(x, w, targets)[1])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_ignored_rows(dtype):
    x, w, targets = _inputs(40, 64, 500, dtype)
    targets[:] = -100
    loss, lse = sx.linear_cross_entropy(x, w, targets)
    assert bool(loss.isnan())  # the mean of nothing
    assert float(sx.linear_cross_entropy(x, w, targets, reduction="sum")[0]) == 0
    for red in ("mean", "sum", "none"):
        d = torch.ones(40 if red == "none" else (), device=DEV)
        dx, dw = sx.linear_cross_entropy_backward(d, x, w, targets, lse, reduction=red)
        assert not dx.any() and not dw.any()
    # another index, one that is a word of the vocabulary
    targets = torch.randint(0, 500, (40,), device=DEV)
    targets[::3] = 7
    loss, lse = sx.linear_cross_entropy(x, w, targets, ignore_index=7)
    _check_loss(x, w, targets, loss, lse, "mean", ignore=7)
    d = torch.ones((), device=DEV)
    _check_grads(d, x, w, targets, lse, *sx.linear_cross_entropy_backward(d, x, w, targets, lse, ignore_index=7), "mean", ignore=7)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("t,h,pad", [(40, 64, 0), (300, 100, 0), (257, 33, 3), (500, 128, 8)])
def test_ignored_rows_may_hold_anything(t, h, pad, dtype):
    """A padded batch whose padding went wrong upstream: the loss and the gradients are those of the rows that count."""
    x, w, targets = _inputs(t, h, 700, dtype)
    skip = targets == -100
    assert bool(skip.any())
    x[skip] = 0
    wide = torch.zeros(t, h + pad, dtype=dtype, device=DEV)
    bad = wide[:, :h]
    bad.copy_(x)
    bad[skip] = float("nan")
    bad[int(skip.nonzero()[0, 0]), ::2] = float("inf")
    d = torch.ones((), device=DEV)
    loss, lse = sx.linear_cross_entropy(bad, w, targets)
    want, lse0 = sx.linear_cross_entropy(x, w, targets)
    assert torch.equal(loss, want) and torch.equal(lse[~skip], lse0[~skip])
    got = sx.linear_cross_entropy_backward(d, bad, w, targets, lse)
    _check_grads(d, x, w, targets, lse0, *got, "mean")
    assert all(torch.equal(a, b) for a, b in zip(got, sx.linear_cross_entropy_backward(d, x, w, targets, lse0)))
    assert not got[0][skip].any()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_targets_out_of_range_are_seen(dtype):
    x, w, targets = _inputs(30, 64, 300, dtype, ignored=0.0)
    targets[4], targets[9] = 300, -1
    loss, lse = sx.linear_cross_entropy(x, w, targets, reduction="none")
    bad = torch.zeros(30, dtype=torch.bool, device=DEV)
    bad[4] = bad[9] = True
    assert torch.equal(loss.isnan(), bad)
    assert bool(sx.linear_cross_entropy(x, w, targets)[0].isnan())
    dx, dw = sx.linear_cross_entropy_backward(torch.ones(30, device=DEV), x, w, targets, lse, reduction="none")
    assert torch.equal(dx.isnan().all(1), bad) and bool(dw.isnan().all())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_no_tokens(dtype):
    x, w, targets = _inputs(4, 64, 300, dtype)
    x, targets = x[:0], targets[:0]
    assert bool(sx.linear_cross_entropy(x, w, targets)[0].isnan())
    assert float(sx.linear_cross_entropy(x, w, targets, reduction="sum")[0]) == 0
    loss, lse = sx.linear_cross_entropy(x, w, targets, reduction="none")
    assert loss.shape == lse.shape == (0,)
    dx, dw = sx.linear_cross_entropy_backward(torch.ones((), device=DEV), x, w, targets, lse)
    assert dx.shape == (0, 64) and dw.shape == (300, 64) and not dw.any()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_large_and_far_logits(dtype):
    """Logits of several hundreds: 2^x of a raw logit would overflow."""
    x, w, targets = _inputs(60, 64, 1000, dtype)
    x = x * 64
    loss, lse = sx.linear_cross_entropy(x, w, targets, reduction="none")
    _check_loss(x, w, targets, loss, lse, "none")
    assert float(lse.max()) > 200
    d = torch.ones(60, device=DEV)
    dx, dw = sx.linear_cross_entropy_backward(d, x, w, targets, lse, reduction="none")
    assert bool(dx.isfinite().all()) and bool(dw.isfinite().all())
    # every logit of a whole tile far below the row's largest
    w2 = w.clone()
    w2[: 600] = 0
    w2[:600, 0] = -300
    x2 = x.clone()
    x2[:, 0] = 300
    targets2 = torch.where(targets >= 0, targets % 400 + 600, targets)
    loss, lse = sx.linear_cross_entropy(x2, w2, targets2, reduction="none")
    _check_loss(x2, w2, targets2, loss, lse, "none")


@pytest.mark.parametrize("dtype", [BF, F32])
def test_values_that_are_not_finite_stay_in_their_row(dtype):
    x, w, targets = _inputs(300, 64, 1000, dtype, ignored=0.0)
    want, lse0 = sx.linear_cross_entropy(x, w, targets, reduction="none")
    x[3, 5] = float("nan")
    x[200, 0] = float("inf")
    loss, lse = sx.linear_cross_entropy(x, w, targets, reduction="none")
    good = torch.ones(300, dtype=torch.bool, device=DEV)
    good[3] = good[200] = False
    assert torch.equal(loss[good], want[good]) and torch.equal(lse[good], lse0[good])
    assert bool(loss[3].isnan()) and not bool(loss[200].isfinite())
    # a padded row with NaN in it has no loss
    targets[3] = targets[200] = -100
    loss, _ = sx.linear_cross_entropy(x, w, targets, reduction="mean")
    assert bool(loss.isfinite())
    # a word whose logits are all -inf has no probability
    x2, w2, targets2 = _inputs(20, 64, 300, dtype, seed=3, ignored=0.0)
    x2[:, 0] = 1
    w2[100:200] = 0
    w2[100:200, 0] = float("-inf")
    keep = torch.cat([w2[:100], w2[200:]])
    targets2 %= 100
    a, la = sx.linear_cross_entropy(x2, w2, targets2, reduction="none")
    if dtype == F32:  # as documented: the split of an infinity into tf32 parts has no value
        assert bool(la.isnan().all())
        w2[100:200, 0] = -1e30
        a, la = sx.linear_cross_entropy(x2, w2, targets2, reduction="none")
    _check_loss(x2, keep, targets2, a, la, "none")


def test_gradient_against_differences():
    """d loss / dx and dW by central differences of the definition in 64 bits: h^2 of the third derivative is under 1e-8."""
    x, w, targets = _inputs(6, 16, 50, F32)
    loss, lse = sx.linear_cross_entropy(x, w, targets)
    dx, dw = sx.linear_cross_entropy_backward(torch.ones((), device=DEV), x, w, targets, lse)

    def f(a, b):
        return float(torch.nn.functional.cross_entropy(a @ b.t(), targets, ignore_index=-100))

    xd, wd, h = x.double(), w.double(), 1e-4
    for i, j in ((0, 0), (2, 7), (5, 15)):
        e = torch.zeros_like(xd)
        e[i, j] = h
        assert abs((f(xd + e, wd) - f(xd - e, wd)) / (2 * h) - float(dx[i, j])) < 2e-6
    for i, j in ((0, 0), (int(targets.max()), 3), (49, 15)):
        e = torch.zeros_like(wd)
        e[i, j] = h
        assert abs((f(xd, wd + e) - f(xd, wd - e)) / (2 * h) - float(dw[i, j])) < 2e-6


@pytest.mark.parametrize("dtype", [BF, F32])
def test_same_bits_every_time_on_streams_and_in_graphs(dtype):
    x, w, targets = _inputs(600, 128, 3001, dtype)
    d = torch.ones((), device=DEV)
    def step(stream=None):
        loss, lse = sx.linear_cross_entropy(x, w, targets, stream=stream)
        return (loss, lse) + sx.linear_cross_entropy_backward(d, x, w, targets, lse, stream=stream)
    want = step()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for stream in (None, s.cuda_stream, None):
        got = step(stream)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    keep = x.clone()
    x.zero_()
    graph.replay()
    x.copy_(keep)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_two_streams_at_once():
    cases = [_inputs(900, 128, 4001, BF, seed=k) for k in range(2)]
    d = torch.ones((), device=DEV)
    def step(c):
        loss, lse = sx.linear_cross_entropy(*c)
        return (loss, lse) + sx.linear_cross_entropy_backward(d, *c, lse)
    want = [step(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(5):
        for k, c in enumerate(cases):
            with torch.cuda.stream(streams[k]):
                got[k].append(step(c))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(a, b) for one in got[k] for a, b in zip(want[k], one))


def test_a_long_queue_of_passes():
    x, w, targets = _inputs(3815, 1104, 26330, BF)
    want, lse = sx.linear_cross_entropy(x, w, targets, reduction="sum")
    torch.cuda.synchronize()
    got = [sx.linear_cross_entropy(x, w, targets, reduction="sum")[0] for _ in range(400)]
    sx.sync_status()
    assert all(torch.equal(v, want) for v in got)


def test_refusals():
    x, w, targets = _inputs(8, 64, 100, BF)
    loss, lse = sx.linear_cross_entropy(x, w, targets)
    one = torch.ones((), device=DEV)
    for call in (lambda: sx.linear_cross_entropy(x.half(), w.half(), targets), lambda: sx.linear_cross_entropy(x, w.float(), targets),
                 lambda: sx.linear_cross_entropy(x, w[:, :32], targets), lambda: sx.linear_cross_entropy(x, w, targets.int()),
                 lambda: sx.linear_cross_entropy(x, w, targets[:4]), lambda: sx.linear_cross_entropy(x, w, targets.cpu()),
                 lambda: sx.linear_cross_entropy(x, w, targets, reduction="max"), lambda: sx.linear_cross_entropy(x, w[:0], targets),
                 lambda: sx.linear_cross_entropy(x[:, :0], w[:, :0], targets), lambda: sx.linear_cross_entropy(x[None], w, targets),
                 lambda: sx.linear_cross_entropy(x, w, targets, ignore_index=1.5),
                 lambda: sx.linear_cross_entropy_backward(one, x, w, targets, lse[:4]),
                 lambda: sx.linear_cross_entropy_backward(one.double(), x, w, targets, lse),
                 lambda: sx.linear_cross_entropy_backward(one, x, w, targets, lse, reduction="none"),
                 lambda: sx.linear_cross_entropy_backward(lse, x, w, targets, lse)):
        with pytest.raises(ValueError):
            call()
