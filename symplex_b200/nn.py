"""Operators at a model's output end, on CUDA tensors: layer norm in front of the last product, the loss behind it
(softmax cross entropy of a linear head, logits never kept) and that product with 4-bit weights for a few tokens.

Like ``gemm`` they are asynchronous on ``stream`` (a raw handle; default: torch's current stream of the tensors' device)
and raise ``ValueError`` for arguments they do not take. Forward and backward passes are functions of their own; nothing
is recorded between them. What they allocate (results and scratch) comes from torch's allocator on the stream of the
call, so calls can be captured into CUDA graphs and run on several streams at once.
"""
from __future__ import annotations

import torch

from . import _capi
from ._capi import DT_BF16, DT_F32

__all__ = ["layer_norm", "layer_norm_backward"]

_DT = {torch.float32: DT_F32, torch.bfloat16: DT_BF16}


def _run(device, stream, fn):
    """``fn(raw_stream)`` with ``device`` current and, where a stream is given, torch's allocations on that stream."""
    if stream is None:
        if device.index == torch.cuda.current_device():
            return fn(torch.cuda.current_stream().cuda_stream)
        with torch.cuda.device(device):
            return fn(torch.cuda.current_stream().cuda_stream)
    with torch.cuda.device(device), torch.cuda.stream(torch.cuda.ExternalStream(stream, device)):
        return fn(stream)


def _rows(t):
    """``t`` as rows of its last dimension: (tensor to read, elements from one row to the next)."""
    if t.is_contiguous():
        return t, t.shape[-1]
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= t.shape[1]:
        return t, t.stride(0)
    return t.contiguous(), t.shape[-1]


def _ptr(t):
    return t.data_ptr() if t is not None else None


# ----------------------------------------------------------------------------- layer norm

def _norm_checks(who, x, *params):
    if not x.is_cuda or x.dtype not in _DT:
        raise ValueError(f"{who} takes float32 or bfloat16 CUDA tensors")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"{who} needs at least one value in the last dimension, got shape {tuple(x.shape)}")
    dtype = None
    for p in params:
        if p is None:
            continue
        if tuple(p.shape) != (x.shape[-1],) or p.device != x.device:
            raise ValueError(f"weight and bias must have shape ({x.shape[-1]},) on {x.device}")
        if p.dtype != x.dtype and p.dtype != torch.float32 or dtype not in (None, p.dtype):
            raise ValueError("weight and bias must both have the input's dtype or both be float32")
        dtype = p.dtype
    return dtype if dtype is not None else x.dtype


def layer_norm(x, weight=None, bias=None, *, eps=1e-5, out=None, return_stats=False, stream=None):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension (``symplex_b200_layer_norm``).

    ``x``: float32 or bfloat16 of any shape; a 2-D view with unit stride in its rows is read in place, other strides
    through a copy. ``weight`` and ``bias``: ``[cols]`` of ``x``'s dtype or float32, or None. ``out``: contiguous (or 2-D
    with unit stride in its rows), may be ``x``. Statistics are computed in 32 bits, the result is rounded once.
    Returns ``y``, or ``(y, mean, rstd)`` with ``return_stats`` (float32, shaped like ``x`` without its last dimension):
    what ``layer_norm_backward`` takes.
    """
    pdt = _norm_checks("layer_norm()", x, weight, bias)
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    if out is not None and (out.shape != x.shape or out.dtype != x.dtype or out.device != x.device or
                            not (out.is_contiguous() or (out.dim() == 2 and out.stride(1) == 1 and out.stride(0) >= out.shape[1]))):
        raise ValueError("out must match x in shape, dtype and device, with unit stride in its rows")

    def call(s):
        xr, ldx = _rows(x)
        y = out if out is not None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
        mean = rstd = None
        if return_stats:
            mean = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
            rstd = torch.empty_like(mean)
        w = weight.contiguous() if weight is not None else None
        b = bias.contiguous() if bias is not None else None
        cols = x.shape[-1]
        _capi.check(_capi.load().symplex_b200_layer_norm(
            xr.data_ptr(), _ptr(w), _ptr(b), y.data_ptr(), _ptr(mean), _ptr(rstd), x.numel() // cols, cols, ldx,
            cols if y.is_contiguous() else y.stride(0), _DT[x.dtype], _DT[pdt], eps, s))
        return (y, mean, rstd) if return_stats else y

    return _run(x.device, stream, call)


def layer_norm_backward(dy, x, mean, rstd, weight=None, *, param_grads=None, stream=None):
    """Gradients of ``layer_norm``: ``(dx, dweight, dbias)`` from the output's gradient, the input and the statistics of
    the forward pass (``symplex_b200_layer_norm_backward``).

    ``dweight`` and ``dbias`` have ``weight``'s dtype (``x``'s where there is no weight) and are None unless
    ``param_grads`` (default: whether ``weight`` is given). Their sums over rows are 32-bit, in a fixed order.
    """
    pdt = _norm_checks("layer_norm_backward()", x, weight)
    if dy.shape != x.shape or dy.dtype != x.dtype or dy.device != x.device:
        raise ValueError("dy must match x in shape, dtype and device")
    for t in (mean, rstd):
        if t.dtype != torch.float32 or t.shape != x.shape[:-1] or t.device != x.device:
            raise ValueError(f"mean and rstd must be float32 of shape {tuple(x.shape[:-1])} on {x.device}")
    if param_grads is None:
        param_grads = weight is not None

    def call(s):
        lib = _capi.load()
        (xr, ldx), (dyr, lddy) = _rows(x), _rows(dy)
        cols = x.shape[-1]
        rows = x.numel() // cols
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dw = db = ws = None
        size = 0
        if param_grads:
            dw = torch.empty(cols, dtype=pdt, device=x.device)
            db = torch.empty(cols, dtype=pdt, device=x.device)
            size = lib.symplex_b200_layer_norm_backward_workspace_bytes(rows, cols)
            ws = torch.empty(size, dtype=torch.uint8, device=x.device)
        w = weight.contiguous() if weight is not None else None
        m, r = mean.contiguous(), rstd.contiguous()
        _capi.check(lib.symplex_b200_layer_norm_backward(
            dyr.data_ptr(), xr.data_ptr(), m.data_ptr(), r.data_ptr(), _ptr(w), dx.data_ptr(), _ptr(dw), _ptr(db), rows, cols,
            lddy, ldx, cols, _DT[x.dtype], _DT[pdt], _ptr(ws), size, s))
        return dx, dw, db

    return _run(x.device, stream, call)
