"""Operators at a model's output end, on CUDA tensors: layer norm in front of the last product, the loss behind it
(softmax cross entropy of a linear head, logits never kept) and that product with 4-bit weights for a few tokens.

Like ``gemm`` they are asynchronous on ``stream`` (a raw handle; default: torch's current stream of the tensors' device)
and raise ``ValueError`` for arguments they do not take. Forward and backward passes are functions of their own; nothing
is recorded between them. What they allocate (results and scratch) comes from torch's allocator on the stream of the
call, so calls can be captured into CUDA graphs and run on several streams at once. On a ``stream`` that is not the current one the
operands are named to the allocator (``record_stream``) and may be dropped behind the call; that they are ready on that stream, and
that it is done before another one takes the results, is the caller's to see to.
"""
from __future__ import annotations

import functools

import torch

from . import _capi
from ._capi import ACTIVATIONS, DT_BF16, DT_F32, LOSS_REDUCTIONS

__all__ = ["layer_norm", "layer_norm_backward", "linear_cross_entropy", "linear_cross_entropy_backward",
           "int4_quantize", "int4_matvec"]

INT4_MAX_ROWS = 64

_DT = {torch.float32: DT_F32, torch.bfloat16: DT_BF16}


# The handle of torch's current stream; the object that torch.cuda.current_stream() makes for it costs 3 us a call.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _run(device, stream, fn, *operands):
    """``fn(raw_stream)`` with ``device`` current and, where a stream is given, torch's allocations on that stream and the ``operands``
    kept from being handed out again before it has read them."""
    if stream is None:
        if device.index == torch.cuda.current_device():
            return fn(_raw_stream(device.index))
        with torch.cuda.device(device):
            return fn(_raw_stream(device.index))
    other = stream != _raw_stream(device.index)
    s = torch.cuda.ExternalStream(stream, device)
    with torch.cuda.device(device), torch.cuda.stream(s):
        if other:
            for t in operands:
                if t is not None:
                    t.record_stream(s)
        return fn(stream)


def _rows(t):
    """``t`` as rows of its last dimension: (tensor to read, elements from one row to the next)."""
    if t.is_contiguous():
        return t, t.shape[-1]
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= t.shape[1]:
        return t, t.stride(0)
    return t.contiguous(), t.shape[-1]


def _like(t):
    """A contiguous tensor like ``t`` (``empty_like`` takes half the time of ``empty``, but keeps other strides)."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(query, *args):
    """A size query of the library, a function of its arguments alone."""
    return getattr(_capi.load(), query)(*args)


def _check(code):
    """Arguments that the library refuses are the caller's, like those refused here."""
    if code == _capi.ERR_INVALID:
        raise ValueError(_capi.last_error())
    _capi.check(code)


def _ptr(t):
    return t.data_ptr() if t is not None else None


# ----------------------------------------------------------------------------- layer norm

def _norm_checks(who, x, *params):
    """(columns, dtype of the parameters) of a norm over ``x``."""
    dtype, shape = x.dtype, x.shape
    if not x.is_cuda or dtype not in _DT:
        raise ValueError(f"{who} takes float32 or bfloat16 CUDA tensors")
    if not shape or shape[-1] == 0:
        raise ValueError(f"{who} needs at least one value in the last dimension, got shape {tuple(shape)}")
    cols, device, found = shape[-1], x.device, None
    for p in params:
        if p is None:
            continue
        if p.shape != (cols,) or p.device != device:
            raise ValueError(f"weight and bias must have shape ({cols},) on {device}")
        pdt = p.dtype
        if pdt != dtype and pdt != torch.float32 or found not in (None, pdt):
            raise ValueError("weight and bias must both have the input's dtype or both be float32")
        found = pdt
    return cols, found or dtype


def layer_norm(x, weight=None, bias=None, *, eps=1e-5, out=None, return_stats=False, stream=None):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension (``symplex_b200_layer_norm``).

    ``x``: float32 or bfloat16 of any shape; a 2-D view with unit stride in its rows is read in place, other strides
    through a copy. ``weight`` and ``bias``: ``[cols]`` of ``x``'s dtype or float32, or None. ``out``: contiguous (or 2-D
    with unit stride in its rows), may be ``x`` but not overlap it otherwise. Statistics are computed in 32 bits, the result is rounded once.
    Returns ``y``, or ``(y, mean, rstd)`` with ``return_stats`` (float32, shaped like ``x`` without its last dimension):
    what ``layer_norm_backward`` takes.
    """
    cols, pdt = _norm_checks("layer_norm()", x, weight, bias)
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    if out is not None and (out.shape != x.shape or out.dtype != x.dtype or out.device != x.device or
                            not (out.is_contiguous() or (out.dim() == 2 and out.stride(1) == 1 and out.stride(0) >= out.shape[1]))):
        raise ValueError("out must match x in shape, dtype and device, with unit stride in its rows")

    def call(s):
        xr, ldx = _rows(x)
        y = out if out is not None else _like(x)
        mean = rstd = None
        if return_stats:
            mean = x.new_empty(x.shape[:-1], dtype=torch.float32)
            rstd = torch.empty_like(mean)
        w = weight.contiguous() if weight is not None else None
        b = bias.contiguous() if bias is not None else None
        _check(_capi.load().symplex_b200_layer_norm(
            xr.data_ptr(), _ptr(w), _ptr(b), y.data_ptr(), _ptr(mean), _ptr(rstd), x.numel() // cols, cols, ldx,
            cols if out is None or y.is_contiguous() else y.stride(0), _DT[x.dtype], _DT[pdt], eps, s))
        return (y, mean, rstd) if return_stats else y

    return _run(x.device, stream, call, x, weight, bias, out)


def layer_norm_backward(dy, x, mean, rstd, weight=None, *, param_grads=None, stream=None):
    """Gradients of ``layer_norm``: ``(dx, dweight, dbias)`` from the output's gradient, the input and the statistics of
    the forward pass (``symplex_b200_layer_norm_backward``).

    ``dweight`` and ``dbias`` have ``weight``'s dtype (``x``'s where there is no weight) and are None unless
    ``param_grads`` (default: whether ``weight`` is given). Their sums over rows are 32-bit, in a fixed order.
    """
    cols, pdt = _norm_checks("layer_norm_backward()", x, weight)
    shape, device = x.shape, x.device
    if dy.shape != shape or dy.dtype != x.dtype or dy.device != device:
        raise ValueError("dy must match x in shape, dtype and device")
    for t in (mean, rstd):
        if t.dtype != torch.float32 or t.shape != shape[:-1] or t.device != device:
            raise ValueError(f"mean and rstd must be float32 of shape {tuple(shape[:-1])} on {device}")
    if param_grads is None:
        param_grads = weight is not None

    def call(s):
        lib = _capi.load()
        (xr, ldx), (dyr, lddy) = _rows(x), _rows(dy)
        rows = x.numel() // cols
        dx = _like(x)
        dw = db = ws = None
        size = 0
        if param_grads:
            dw = x.new_empty(cols, dtype=pdt)
            db = torch.empty_like(dw)
            size = _workspace_bytes("symplex_b200_layer_norm_backward_workspace_bytes", rows, cols)
            ws = x.new_empty(size, dtype=torch.uint8)
        w = weight.contiguous() if weight is not None else None
        m, r = mean.contiguous(), rstd.contiguous()
        _check(lib.symplex_b200_layer_norm_backward(
            dyr.data_ptr(), xr.data_ptr(), m.data_ptr(), r.data_ptr(), _ptr(w), dx.data_ptr(), _ptr(dw), _ptr(db), rows, cols,
            lddy, ldx, cols, _DT[x.dtype], _DT[pdt], _ptr(ws), size, s))
        return dx, dw, db

    return _run(device, stream, call, dy, x, mean, rstd, weight)


# ----------------------------------------------------------------------------- softmax cross entropy of a linear head

def _loss_checks(who, x, weight, targets, ignore_index, reduction):
    """(T, H, V) of a loss."""
    dtype, shape, device = x.dtype, x.shape, x.device
    if not x.is_cuda or dtype not in _DT or len(shape) != 2:
        raise ValueError(f"{who} takes a 2-D float32 or bfloat16 CUDA tensor")
    t, h = shape
    wshape = weight.shape
    if weight.dtype != dtype or len(wshape) != 2 or wshape[1] != h or weight.device != device:
        raise ValueError(f"weight must be {dtype} of shape [V, {h}] on {device}, got {weight.dtype} {tuple(wshape)}")
    v = wshape[0]
    if h == 0 or v == 0:
        raise ValueError("the hidden size and the vocabulary must not be empty")
    if targets.dtype != torch.int64 or targets.shape != (t,) or targets.device != device:
        raise ValueError(f"targets must be int64 of shape ({t},) on {device}")
    if reduction not in LOSS_REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(LOSS_REDUCTIONS)}, got {reduction!r}")
    if not isinstance(ignore_index, int) or not -2 ** 63 <= ignore_index < 2 ** 63:
        raise ValueError("ignore_index must be a 64-bit integer")
    return t, h, v


def linear_cross_entropy(x, weight, targets, *, ignore_index=-100, reduction="mean", stream=None):
    """Softmax cross entropy of the logits ``x @ weight.T``, which are never kept (``symplex_b200_linear_cross_entropy``).

    ``x``: float32 or bfloat16 ``[T, H]``; ``weight``: ``[V, H]`` of the same dtype (both may be views with unit stride in
    their rows); ``targets``: int64 ``[T]``, rows equal to ``ignore_index`` have no loss. ``reduction``: ``"mean"`` over the rows
    that count (NaN if none does), ``"sum"`` or ``"none"``. Returns ``(loss, lse)`` in float32: a 0-d tensor or ``[T]``, and the
    rows' log-sum-exp, which the backward pass takes. A target outside ``0..V-1`` gives its row the loss NaN;
    so does an infinity among float32 operands (their products are split into tf32 parts).
    """
    t, h, v = _loss_checks("linear_cross_entropy()", x, weight, targets, ignore_index, reduction)

    def call(s):
        lib = _capi.load()
        (xr, ldx), (w, ldw) = _rows(x), _rows(weight)
        lse = x.new_empty(t, dtype=torch.float32)
        loss = torch.empty_like(lse) if reduction == "none" else lse.new_empty(())
        size = _workspace_bytes("symplex_b200_linear_cross_entropy_workspace_bytes", xr.data_ptr() & 255, w.data_ptr() & 255, t, h, v, ldx,
                                ldw, _DT[x.dtype])  # of the pointers it looks at the alignment
        ws = x.new_empty(size, dtype=torch.uint8)
        tg = targets.contiguous()
        _check(lib.symplex_b200_linear_cross_entropy(
            xr.data_ptr(), w.data_ptr(), tg.data_ptr(), loss.data_ptr(), lse.data_ptr(), t, h, v, ldx, ldw, _DT[x.dtype], ignore_index,
            LOSS_REDUCTIONS[reduction], ws.data_ptr(), size, s))
        return loss, lse

    return _run(x.device, stream, call, x, weight, targets)


def linear_cross_entropy_backward(dloss, x, weight, targets, lse, *, ignore_index=-100, reduction="mean", stream=None):
    """Gradients ``(dx, dweight)`` of ``linear_cross_entropy`` (``symplex_b200_linear_cross_entropy_backward``).

    ``dloss``: float32, one value (``"mean"``, ``"sum"``) or ``[T]`` (``"none"``); ``lse`` from the forward pass over the same rows (both
    passes round a logit alike, which rows that are sure of their target depend on); the other arguments as there. The logits are computed again a piece of the vocabulary at a time. ``dx`` and ``dweight`` have the dtype of ``x``.
    Ignored rows of ``x`` may hold anything; they are taken as 0.
    """
    t, h, v = _loss_checks("linear_cross_entropy_backward()", x, weight, targets, ignore_index, reduction)
    if dloss.dtype != torch.float32 or dloss.device != x.device or \
            (dloss.shape != (t,) if reduction == "none" else dloss.numel() != 1):
        raise ValueError(f"dloss must be float32 on {x.device}: shape ({t},) for 'none', one value otherwise")
    if lse.dtype != torch.float32 or lse.shape != (t,) or lse.device != x.device:
        raise ValueError(f"lse must be float32 of shape ({t},) on {x.device}")

    def call(s):
        lib = _capi.load()
        (xr, ldx), (w, ldw) = _rows(x), _rows(weight)
        dx, dw = _like(x), _like(weight)
        size = _workspace_bytes("symplex_b200_linear_cross_entropy_backward_workspace_bytes", xr.data_ptr() & 255, w.data_ptr() & 255, t, h, v, ldx,
                                ldw, _DT[x.dtype])  # of the pointers it looks at the alignment
        ws = x.new_empty(size, dtype=torch.uint8)
        tg, ls, dl = targets.contiguous(), lse.contiguous(), dloss.contiguous()
        _check(lib.symplex_b200_linear_cross_entropy_backward(
            dl.data_ptr(), xr.data_ptr(), w.data_ptr(), tg.data_ptr(), ls.data_ptr(), dx.data_ptr(), dw.data_ptr(), t, h, v, ldx, ldw,
            _DT[x.dtype], ignore_index, LOSS_REDUCTIONS[reduction], ws.data_ptr(), size, s))
        return dx, dw

    return _run(x.device, stream, call, dloss, x, weight, targets, lse)


# ----------------------------------------------------------------------------- products with 4-bit weights

def _group_count(k, group_size, who):
    if not isinstance(group_size, int) or group_size <= 0 or group_size % 32:
        raise ValueError(f"{who}: group_size must be a positive multiple of 32, got {group_size!r}")
    return -(-k // group_size)


def int4_quantize(weight, group_size=128, *, symmetric=True, scale_dtype=torch.bfloat16, stream=None):
    """Lay out a ``[N, K]`` weight (float32 or bfloat16) in 4 bits: ``(codes, scales, zeros)`` for ``int4_matvec``.

    ``codes``: uint8 ``[N, ceil(K / 2)]``, the low half of a byte is the even k. ``scales``: ``scale_dtype``
    ``[N, ceil(K / group_size)]``. ``zeros``: None (symmetric: 8 everywhere, scale = max|w| / 7) or uint8 like ``scales``
    (scale = range / 15). A group with a weight that is not finite gets the scale NaN. (``symplex_b200_int4_quantize``)
    """
    if not weight.is_cuda or weight.dtype not in _DT or weight.dim() != 2:
        raise ValueError("int4_quantize() takes a 2-D float32 or bfloat16 CUDA tensor")
    if scale_dtype not in _DT:
        raise ValueError("scale_dtype must be float32 or bfloat16")
    n, k = weight.shape
    if k == 0:
        raise ValueError("K == 0 is not supported")
    groups = _group_count(k, group_size, "int4_quantize()")

    def call(s):
        w, ldw = _rows(weight)
        codes = torch.empty(n, (k + 1) // 2, dtype=torch.uint8, device=weight.device)
        scales = torch.empty(n, groups, dtype=scale_dtype, device=weight.device)
        zeros = None if symmetric else torch.empty(n, groups, dtype=torch.uint8, device=weight.device)
        _check(_capi.load().symplex_b200_int4_quantize(w.data_ptr(), codes.data_ptr(), scales.data_ptr(), _ptr(zeros), n, k,
                                                            group_size, ldw, _DT[weight.dtype], _DT[scale_dtype], s))
        return codes, scales, zeros

    return _run(weight.device, stream, call, weight)


def int4_matvec(x, codes, scales, zeros=None, *, group_size=128, bias=None, activation=None, out=None, out_dtype=None,
                stream=None):
    """``act(x @ W.T + bias)`` for a few rows of ``x`` (at most 64), ``W[n, k] = (codes[n, k] - zeros[n, k // group_size]) *
    scales[n, k // group_size]`` held as ``int4_quantize`` lays it out (``symplex_b200_int4_matvec``).

    ``x``: bfloat16 ``[K]`` or ``[M, K]``; ``zeros`` (0 to 15) None means 8 everywhere; ``bias``: float32 ``[N]``; ``activation`` as in
    ``gemm`` (the relu of NaN is NaN here). ``codes`` may be a view with unit stride in its rows. Returns ``[N]`` / ``[M, N]`` in ``out_dtype`` (bfloat16 or
    float32); ``out`` must not overlap an operand. More rows are passed in parts of at most 64 (``gemm`` takes
    no codes).
    """
    xshape, device = x.shape, x.device
    if not x.is_cuda or x.dtype != torch.bfloat16 or len(xshape) not in (1, 2):
        raise ValueError("int4_matvec() takes a 1-D or 2-D bfloat16 CUDA tensor")
    k = xshape[-1]
    m = xshape[0] if len(xshape) == 2 else 1
    if m > INT4_MAX_ROWS:
        raise ValueError(f"int4_matvec() takes at most {INT4_MAX_ROWS} rows a call, got {m}: pass them in parts")
    if k == 0:
        raise ValueError("K == 0 is not supported")
    groups = _group_count(k, group_size, "int4_matvec()")
    cshape = codes.shape
    if codes.dtype != torch.uint8 or len(cshape) != 2 or cshape[1] != (k + 1) // 2 or codes.device != device:
        raise ValueError(f"codes must be uint8 of shape [N, {(k + 1) // 2}] on {device}, got {codes.dtype} {tuple(cshape)}")
    n = cshape[0]
    if scales.dtype not in _DT or scales.shape != (n, groups) or scales.device != device:
        raise ValueError(f"scales must be float32 or bfloat16 of shape ({n}, {groups}) on {device}")
    if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != (n, groups) or zeros.device != device):
        raise ValueError(f"zeros must be uint8 of shape ({n}, {groups}) on {device}")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (n,) or bias.device != device):
        raise ValueError(f"bias must be float32 of shape ({n},) on {device}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}; expected one of {sorted(a for a in ACTIVATIONS if a)}")
    shape = (n,) if len(xshape) == 1 else (m, n)
    if out is not None:
        if out.shape != shape or out.dtype not in _DT or out.device != device or not out.is_contiguous() or \
                out_dtype not in (None, out.dtype):
            raise ValueError(f"out must be a contiguous float32 or bfloat16 tensor of shape {shape} on {device}")
        out_dtype = out.dtype
    elif out_dtype is None:
        out_dtype = torch.bfloat16
    elif out_dtype not in _DT:
        raise ValueError("out dtype must be float32 or bfloat16")

    def call(s):
        y = out if out is not None else x.new_empty(shape, dtype=out_dtype)
        (a, lda), (c, ldq) = _rows(x), _rows(codes)
        sc = scales.contiguous()
        z = zeros.contiguous() if zeros is not None else None
        b = bias.contiguous() if bias is not None else None
        _check(_capi.load().symplex_b200_int4_matvec(
            a.data_ptr(), c.data_ptr(), sc.data_ptr(), _ptr(z), _ptr(b), y.data_ptr(), m, n, k, group_size, lda, ldq, n,
            _DT[sc.dtype], _DT[out_dtype], ACTIVATIONS[activation], s))
        return y

    return _run(device, stream, call, x, codes, scales, zeros, bias, out)
