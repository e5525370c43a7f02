"""A model's output end as a program runs it: norm, loss of the head, its gradients and the norm's; norm and the 4-bit head
for single tokens. Held to 64-bit arithmetic and captured into graphs.

Bounds, u = 2^-24, on relative Frobenius norms. float32: the norm's result is off by under 16 u of |y|, a logit by at most
dl = (2 H + 96) u sum|y w|; p and with it every gradient moves by at most 2 dl of its own size, the products add chains of
(2 n + 128) u over n = V or T terms. At H = 256, V = 1500, sum|y w| < 40 that is under 2e-3 + 4e-4. bfloat16 is checked stage
by stage from what the stage before it wrote, so that only the stage's own roundings count: G and the result, half a step
(2^-8) each at the most and independent (as in the tests of the single operators).
"""
import math

import pytest
import torch

import symplex_b200 as sx

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
T, H, V = 333, 256, 1500


def _model(dtype, t=T, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(t, H, generator=g, device=DEV) * 2 + 0.5).to(dtype)
    gain = (1 + 0.2 * torch.randn(H, generator=g, device=DEV)).to(dtype)
    shift = (0.1 * torch.randn(H, generator=g, device=DEV)).to(dtype)
    head = (torch.randn(V, H, generator=g, device=DEV) / math.sqrt(H)).to(dtype)
    targets = torch.randint(0, V, (t,), generator=g, device=DEV)
    targets[::7] = -100
    return x, gain, shift, head, targets


def _train_step(x, gain, shift, head, targets, stream=None):
    y, mean, rstd = sx.layer_norm(x, gain, shift, return_stats=True, stream=stream)
    loss, lse = sx.linear_cross_entropy(y, head, targets, stream=stream)
    one = torch.ones((), device=DEV)
    dy, dhead = sx.linear_cross_entropy_backward(one, y, head, targets, lse, stream=stream)
    dx, dgain, dshift = sx.layer_norm_backward(dy, x, mean, rstd, gain, stream=stream)
    return dict(y=y, loss=loss, dy=dy, dhead=dhead, dx=dx, dgain=dgain, dshift=dshift)


def _exact(x, gain, shift, head, targets, y=None, dy=None):
    """The same in 64 bits; later stages from y and dy where they are given."""
    xd, gd, sd, hd = (a.double().requires_grad_() for a in (x, gain, shift, head))
    yd = torch.nn.functional.layer_norm(xd, (H,), gd, sd, 1e-5)
    yin = (yd if y is None else y.double()).detach().requires_grad_()
    loss = torch.nn.functional.cross_entropy(yin @ hd.t(), targets, ignore_index=-100)
    dyd, dhead = torch.autograd.grad(loss, (yin, hd))
    dx, dgain, dshift = torch.autograd.grad(yd, (xd, gd, sd), dyd if dy is None else dy.double())
    return dict(y=yd.detach(), loss=loss.detach(), dy=dyd, dhead=dhead, dx=dx, dgain=dgain, dshift=dshift)


def _off(a, b):
    return float((a.double() - b).norm() / b.norm())


def test_a_training_step_in_32_bits():
    got, ref = _train_step(*_model(F32)), _exact(*_model(F32))
    sx.sync_status()
    for k in ref:
        assert _off(got[k], ref[k]) < 2.4e-3, k


def test_a_training_step_in_bfloat16():
    m = _model(BF)
    got = _train_step(*m)
    sx.sync_status()
    ref = _exact(*m, y=got["y"], dy=got["dy"])
    assert _off(got["loss"], ref["loss"]) < 1e-4
    for k in ("y", "dy", "dhead", "dx", "dgain", "dshift"):
        assert _off(got[k], ref[k]) < 1.5 * 2.0 ** -8, k


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_training_step_captured_and_on_another_stream(dtype):
    m = _model(dtype)
    want = _train_step(*m)
    other = _train_step(*_model(dtype, seed=1))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    elsewhere = _train_step(*m, stream=s.cuda_stream)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _train_step(*m)
    for seed, ref in ((0, want), (1, other), (0, want)):
        for a, b in zip(m, _model(dtype, seed=seed)):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(got[k], ref[k]) for k in ref)
    assert all(torch.equal(elsewhere[k], want[k]) for k in want)


@pytest.mark.parametrize("tokens", [1, 3, 16])
@pytest.mark.parametrize("symmetric", [True, False])
def test_tokens_through_a_4_bit_head(tokens, symmetric):
    """Norm and head of a decoding step; the loss of the same rows under the weights that the codes stand for agrees with its logits."""
    x, gain, shift, head, targets = _model(BF, t=tokens)
    codes, scales, zeros = sx.int4_quantize(head, 64, symmetric=symmetric)
    q = torch.stack([codes & 15, codes >> 4], 2).reshape(V, H).double()
    z = 8.0 if zeros is None else zeros.double().repeat_interleave(64, 1)
    w = (q - z) * scales.double().repeat_interleave(64, 1)

    def step():
        y = sx.layer_norm(x, gain, shift)
        return y, sx.int4_matvec(y, codes, scales, zeros, group_size=64, out_dtype=F32)

    y, logits = step()
    ref = y.double() @ w.t()
    # exact products (bf16 x 4 bits x scale in fp32): chains of H steps and the scaling, in fp32
    bound = (2 * H + 128) * 2.0 ** -24 * (y.double().abs() @ ((q + z) * scales.double().repeat_interleave(64, 1).abs()).t())
    assert bool(((logits.double() - ref).abs() <= bound).all())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, again = step()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, logits)
    # w has at most 8 significant bits times a bf16 scale's 8: rounded to bf16 for the loss, half a step of each weight
    _, lse = sx.linear_cross_entropy(y, w.to(BF), targets)
    moved = (2.0 ** -8 + (2 * H + 64) * 2.0 ** -24) * (y.double().abs() @ w.abs().t()).max(1).values + 1e-4
    assert bool(((lse.double() - torch.logsumexp(logits.double(), 1)).abs() <= moved).all())


def _far(a, step):
    """``a`` as a view whose rows are ``step`` elements apart."""
    flat = torch.empty((a.shape[0] - 1) * step + a.shape[1], dtype=a.dtype, device=DEV)
    view = torch.as_strided(flat, a.shape, (step, 1))
    view.copy_(a)
    return view


@pytest.mark.parametrize("shift", [0, 3])
def test_rows_more_than_4_gb_apart(shift):
    """Offsets past 32 bits, in elements (1.5 * 2^30 apart, the third row beyond 2^31) and in bytes: the bits of rows that are
    equally aligned and close together."""
    def near(a):
        return _far(a, 2 * H + shift)

    def far(a):
        return _far(a, 3 * 2 ** 29 + shift)

    def same(a, b):
        a, b = (v if isinstance(v, tuple) else (v,) for v in (a, b))
        assert all(torch.equal(p, q) for p, q in zip(a, b))

    x, gain, shift_, head, targets = _model(BF, t=3)
    targets, head = targets % 3, head[:3]
    xn = near(x)
    stats = sx.layer_norm(xn, gain, shift_, return_stats=True)
    y, mean, rstd = stats
    xf = far(x)
    same(sx.layer_norm(xf, gain, shift_, return_stats=True), stats)
    same(sx.layer_norm_backward(y, xf, mean, rstd, gain), sx.layer_norm_backward(y, xn, mean, rstd, gain))
    del xf
    one = torch.ones((), device=DEV)
    for fx, fh in ((far, near), (near, far)):
        loss = sx.linear_cross_entropy(near(y), near(head), targets)
        yf, hf = fx(y), fh(head)
        same(sx.linear_cross_entropy(yf, hf, targets), loss)
        same(sx.linear_cross_entropy_backward(one, yf, hf, targets, loss[1]),
             sx.linear_cross_entropy_backward(one, near(y), near(head), targets, loss[1]))
        del yf, hf
    codes, scales, _ = sx.int4_quantize(near(head), 64)
    same(sx.int4_matvec(far(y), far(codes), scales, group_size=64), sx.int4_matvec(near(y), near(codes), scales, group_size=64))


def test_the_current_stream_by_its_handle():
    m = _model(BF)
    want = _train_step(*m)
    got = _train_step(*m, stream=torch.cuda.current_stream().cuda_stream)
    assert all(torch.equal(got[k], want[k]) for k in want)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_two_graphs_at_once(dtype):
    """Two captured steps, replayed side by side again and again: neither has the other's scratch."""
    models = [_model(dtype, seed=k) for k in (3, 4)]
    want = [_train_step(*m) for m in models]
    codes = [sx.int4_quantize(m[3], 64)[:2] for m in models]
    logits = [sx.int4_matvec(w["y"][:9].to(BF), *c, group_size=64) for w, c in zip(want, codes)]
    torch.cuda.synchronize()
    graphs, got = [], []
    for m, w, c in zip(models, want, codes):
        graph = torch.cuda.CUDAGraph()
        few = w["y"][:9].to(BF)
        with torch.cuda.graph(graph):
            got.append((_train_step(*m), sx.int4_matvec(few, *c, group_size=64), few))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for w, l, (g, l2, _) in zip(want, logits, got):
        assert all(torch.equal(g[k], w[k]) for k in w) and torch.equal(l, l2)
