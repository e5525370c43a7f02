"""Loss and gradients where logits are added up in segments: masks, strides, graphs and streams.

Tolerances as derived in test_linear_cross_entropy_gpu, whose checks are used here.
"""
import pytest
import torch

import symplex_b200 as sx
from test_linear_cross_entropy_gpu import _check_grads, _check_loss, _inputs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16
SHAPES = [(1, 4096, 700), (40, 2056, 3001), (100, 5000, 1000), (300, 4104, 2001), (200, 520, 5001), (1100, 1104, 17000)]


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("t,h,v", SHAPES)
def test_loss_and_gradients(t, h, v, reduction):
    x, w, targets = _inputs(t, h, v, BF, seed=t)
    if t == 1:
        targets[:] = 5
    loss, lse = sx.linear_cross_entropy(x, w, targets, reduction=reduction)
    g = torch.Generator(device=DEV).manual_seed(t + 1)
    d = torch.randn(t, generator=g, device=DEV) if reduction == "none" else torch.rand((), generator=g, device=DEV) + 0.5
    got = sx.linear_cross_entropy_backward(d, x, w, targets, lse, reduction=reduction)
    sx.sync_status()
    _check_loss(x, w, targets, loss, lse, reduction)
    _check_grads(d, x, w, targets, lse, *got, reduction)


@pytest.mark.parametrize("pad,shift", [(8, 0), (3, 0), (0, 1)])
@pytest.mark.parametrize("t,h,v", SHAPES[1:5])
def test_strides_and_rows_that_do_not_count(t, h, v, pad, shift):
    x, w, targets = _inputs(t, h, v, BF, seed=t + pad)
    skip = targets == -100
    assert bool(skip.any())
    x[skip] = 0
    d = torch.ones((), device=DEV)
    want, lse0 = sx.linear_cross_entropy(x, w, targets)
    grads0 = sx.linear_cross_entropy_backward(d, x, w, targets, lse0)

    def view(a):
        flat = torch.full((a.shape[0] * (h + pad) + shift,), float("nan"), device=DEV, dtype=BF)
        r = flat[shift:].view(a.shape[0], h + pad)[:, :h]
        r.copy_(a)
        return r
    xv, wv = view(x), view(w)
    xv[skip] = float("nan")
    loss, lse = sx.linear_cross_entropy(xv, wv, targets)
    grads = sx.linear_cross_entropy_backward(d, xv, wv, targets, lse)
    sx.sync_status()
    assert torch.equal(loss, want) and torch.equal(lse[~skip], lse0[~skip])
    assert all(torch.equal(a, b) for a, b in zip(grads, grads0)) and not grads[0][skip].any()
    _check_grads(d, x, w, targets, lse0, *grads, "mean")


@pytest.mark.parametrize("t,h,v", SHAPES[1:4])
def test_targets_out_of_range_are_seen(t, h, v):
    x, w, targets = _inputs(t, h, v, BF, ignored=0.0)
    targets[4], targets[9] = v, -1
    loss, lse = sx.linear_cross_entropy(x, w, targets, reduction="none")
    bad = torch.zeros(t, dtype=torch.bool, device=DEV)
    bad[4] = bad[9] = True
    dx, dw = sx.linear_cross_entropy_backward(torch.ones(t, device=DEV), x, w, targets, lse, reduction="none")
    assert torch.equal(loss.isnan(), bad) and torch.equal(dx.isnan().all(1), bad) and bool(dw.isnan().all())


@pytest.mark.parametrize("t,h,v", SHAPES[1:5])
def test_same_bits_in_graphs_and_on_streams(t, h, v):
    x, w, targets = _inputs(t, h, v, BF)
    d = torch.ones((), device=DEV)

    def step(stream=None):
        loss, lse = sx.linear_cross_entropy(x, w, targets, stream=stream)
        return (loss, lse) + sx.linear_cross_entropy_backward(d, x, w, targets, lse, stream=stream)
    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = step(side.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step())
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    sx.sync_status()
    assert all(torch.equal(a, b) for got in outs for a, b in zip(want, got))
