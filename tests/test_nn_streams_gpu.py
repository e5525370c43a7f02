"""Operands that their owner drops while another stream has yet to read them."""
import pytest
import torch

import symplex_b200 as sx

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16
ROWS, COLS, WORDS = 600, 512, 3001


def _inputs():
    g = torch.Generator(device=DEV).manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    x, w, b = r(ROWS, COLS).to(BF), r(COLS).to(BF), r(COLS).to(BF)
    y, mean, rstd = sx.layer_norm(x, w, b, return_stats=True)
    head = (r(WORDS, COLS) / 20).to(BF)
    targets = torch.randint(0, WORDS, (ROWS,), generator=g, device=DEV)
    _, lse = sx.linear_cross_entropy(x, head, targets)
    codes, scales, zeros = sx.int4_quantize(head, 32, symmetric=False)
    return dict(x=x, w=w, b=b, dy=r(ROWS, COLS).to(BF), mean=mean, rstd=rstd, head=head, targets=targets, lse=lse,
                dloss=torch.ones((), device=DEV), codes=codes, scales=scales, zeros=zeros, few=x[:5].clone(), bias=r(WORDS))


CALLS = {
    "layer_norm": (("x", "w", "b"), lambda a, s: sx.layer_norm(a["x"], a["w"], a["b"], return_stats=True, stream=s)),
    "layer_norm_backward": (("dy", "x", "mean", "rstd", "w"),
                            lambda a, s: sx.layer_norm_backward(a["dy"], a["x"], a["mean"], a["rstd"], a["w"], stream=s)),
    "linear_cross_entropy": (("x", "head", "targets"), lambda a, s: sx.linear_cross_entropy(a["x"], a["head"], a["targets"], stream=s)),
    "linear_cross_entropy_backward": (("dloss", "x", "head", "targets", "lse"), lambda a, s: sx.linear_cross_entropy_backward(
        a["dloss"], a["x"], a["head"], a["targets"], a["lse"], stream=s)),
    "int4_quantize": (("head",), lambda a, s: sx.int4_quantize(a["head"], 32, symmetric=False, stream=s)),
    "int4_matvec": (("few", "codes", "scales", "zeros", "bias"), lambda a, s: (sx.int4_matvec(
        a["few"], a["codes"], a["scales"], a["zeros"], group_size=32, bias=a["bias"], stream=s),)),
}


@pytest.mark.parametrize("name", sorted(CALLS))
def test_operands_dropped_behind_a_call_on_another_stream(name):
    """The memory of a dropped operand is not handed out again before the stream that reads it has."""
    used, call = CALLS[name]
    keep = _inputs()
    want = call(keep, None)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    call(keep, side.cuda_stream)  # set-up and allocations of that stream
    torch.cuda.synchronize()
    mine = {k: keep[k].clone() for k in used}
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)  # about 50 ms of waiting
    got = call(mine, side.cuda_stream)
    sizes = [(v.shape, v.dtype, v.data_ptr()) for v in mine.values()]
    mine.clear()
    assert not side.query()  # the call has not run yet
    fill = [torch.empty(shape, dtype=dtype, device=DEV).view(torch.uint8).fill_(0x55) if shape else torch.full((), 9.0, device=DEV)
            for shape, dtype, _ in sizes for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    del fill


def test_an_output_dropped_behind_a_call_on_another_stream():
    """Nor that of an output of the caller's: what its next owner wrote stays."""
    keep = _inputs()
    side = torch.cuda.Stream()
    sx.layer_norm(keep["x"], out=torch.empty_like(keep["x"]), stream=side.cuda_stream)
    torch.cuda.synchronize()
    out = torch.empty_like(keep["x"])
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
    sx.layer_norm(keep["x"], out=out, stream=side.cuda_stream)
    del out
    assert not side.query()
    fill = [torch.full_like(keep["x"], 3.0) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(bool((f == 3.0).all()) for f in fill)


def test_in_a_capture_on_a_given_stream():
    """Operands may be named to the allocator during a capture too."""
    keep = _inputs()
    want = sx.layer_norm(keep["x"], keep["w"], keep["b"])
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        got = sx.layer_norm(keep["x"], keep["w"], keep["b"], stream=side.cuda_stream)
        main.wait_stream(side)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
