"""Cases of the operators at a model's output end: layer norm, the loss of a linear head, 4-bit matrix-vector products.

``listed()`` and ``draw(rng)`` name cases, ``prepare`` makes a case's inputs on the GPU, ``run`` is one pass through the
operator (elementary torch operations in 32 bits, or the framework's own entry point where ``own`` is set), ``exact`` is
the definition in 64 bits and ``work`` what a pass cannot do without.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_EB = {"bf16": 2, "fp32": 4}
IGNORE = -100


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # One token on its way to the head: what counts is the latency of the call.
        dict(name="norm_token", op="norm", rows=1, cols=4096, dtype="bf16", affine=True),
        # A training batch's activations.
        dict(name="norm_batch", op="norm", rows=8192, cols=4096, dtype="bf16", affine=True),
        # Backward pass of a small batch at an odd width in fp32.
        dict(name="norm_grad_odd", op="norm_grad", rows=777, cols=1003, dtype="fp32", affine=True),
        # Backward pass of a training batch.
        dict(name="norm_grad_batch", op="norm_grad", rows=8192, cols=4096, dtype="bf16", affine=True),
        # Scoring a handful of tokens against a ragged vocabulary: bound by reading the head's weights.
        dict(name="loss_few", op="loss", tokens=37, hidden=1024, vocab=50257, reduction="none", dtype="bf16"),
        # The loss of a training batch.
        dict(name="loss_batch", op="loss", tokens=8192, hidden=4096, vocab=65536, reduction="mean", dtype="bf16"),
        # A small model's training step in fp32.
        dict(name="loss_grad_fp32", op="loss_grad", tokens=509, hidden=512, vocab=8192, reduction="sum", dtype="fp32"),
        # A ragged packed batch over a ragged vocabulary.
        dict(name="loss_grad_odd", op="loss_grad", tokens=1999, hidden=768, vocab=50257, reduction="none", dtype="bf16"),
        # The gradient of a training batch.
        dict(name="loss_grad_batch", op="loss_grad", tokens=4096, hidden=4096, vocab=65536, reduction="mean", dtype="bf16"),
        # A square projection, one token.
        dict(name="int4_token", op="int4", tokens=1, n=4096, k=4096, group=128, zeros=False, dtype="bf16"),
        # A head over a ragged vocabulary, a few sequences at once, small groups.
        dict(name="int4_ragged", op="int4", tokens=5, n=50257, k=2048, group=32, zeros=True, dtype="bf16"),
        # A wide projection for a batch of sequences.
        dict(name="int4_wide", op="int4", tokens=16, n=28672, k=8192, group=64, zeros=True, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "loss", "loss_grad", "int4"])
    if op in ("norm", "norm_grad"):
        dtype = rng.choice(["bf16", "fp32"])
        cols = _log(rng, 16, 16384)
        if rng.random() < 0.5:
            cols = max(16, cols // 8 * 8)
        rows = _log(rng, 1, min(32768, (1 << 25) // cols))
        return dict(op=op, rows=rows, cols=cols, dtype=dtype, affine=rng.random() < 0.8)
    if op in ("loss", "loss_grad"):
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        hidden = 8 * _log(rng, 8, 1024 if dtype == "bf16" else 256)
        vocab = _log(rng, 1000, 131072 if dtype == "bf16" else 32768)
        most = (1 << 39) if dtype == "bf16" else (1 << 33)
        tokens = _log(rng, 1, max(2, min(8192, most // (hidden * vocab))))
        return dict(op=op, tokens=tokens, hidden=hidden, vocab=vocab, reduction=rng.choice(["mean", "sum", "none"]), dtype=dtype)
    group = rng.choice([32, 64, 128])
    return dict(op=op, tokens=rng.choice([1, 1, 2, 3, 4, 7, 8, 11, 16, 29]), n=_log(rng, 64, 65536), k=group * _log(rng, 4, 16384 // group),
                group=group, zeros=rng.random() < 0.5, dtype="bf16")


# ------------------------------------------------------------------------------------------------ inputs

def _count(targets):
    return (targets != IGNORE).sum()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = _DT[case["dtype"]]

    def randn(*shape, scale=1.0, shift=0.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)

    s = dict(case)
    if case["op"] in ("norm", "norm_grad"):
        rows, cols = case["rows"], case["cols"]
        # rows of different size and offset, as a residual stream has them
        x = torch.randn(rows, cols, generator=g, device="cuda")
        x = x * (0.5 + 2 * torch.rand(rows, 1, generator=g, device="cuda")) + torch.randn(rows, 1, generator=g, device="cuda")
        s["x"] = x.to(dt)
        s["weight"] = randn(cols, scale=0.1, shift=1.0) if case["affine"] else None
        s["bias"] = randn(cols, scale=0.1) if case["affine"] else None
        if case["op"] == "norm_grad":
            s["dy"] = randn(rows, cols, scale=1e-2)
            xf = s["x"].float()
            s["mean"] = xf.mean(1)
            s["rstd"] = torch.rsqrt((xf - s["mean"][:, None]).square().mean(1) + 1e-5)
    elif case["op"] in ("loss", "loss_grad"):
        t, h, v = case["tokens"], case["hidden"], case["vocab"]
        w = randn(v, h, scale=1.5 / math.sqrt(h))
        targets = torch.randint(0, v, (t,), generator=g, device="cuda")
        # some rows know their target, others do not
        x = torch.randn(t, h, generator=g, device="cuda") + 3 * torch.rand(t, 1, generator=g, device="cuda") * w[targets].float()
        if t > 4:  # padding and prompt tokens have no loss
            targets[torch.rand(t, generator=g, device="cuda") < 0.1] = IGNORE
        s.update(x=x.to(dt), weight=w, targets=targets)
        if case["op"] == "loss_grad":
            step = max(1, (1 << 28) // v)
            s["lse"] = torch.cat([torch.logsumexp(xc.float() @ w.float().t(), 1) for xc in s["x"].split(step)])
            if case["reduction"] == "none":
                s["dloss"] = torch.rand(t, generator=g, device="cuda") / t
            else:
                s["dloss"] = torch.rand((), generator=g, device="cuda") + 0.5
    else:
        m, n, k = case["tokens"], case["n"], case["k"]
        s["x"] = randn(m, k)
        s["codes"] = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
        s["scales"] = (0.002 + 0.01 * torch.rand(n, k // case["group"], generator=g, device="cuda")).to(dt)
        s["zeros"] = torch.randint(4, 12, (n, k // case["group"]), generator=g, device="cuda", dtype=torch.uint8) if case["zeros"] else None
    return s


# ------------------------------------------------------------------------------------------------ one pass

def _norm(s):
    if own:
        import symplex_b200 as sx
        return sx.layer_norm(s["x"], s["weight"], s["bias"], eps=1e-5, return_stats=True)
    x = s["x"].float()
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = 1.0 / torch.sqrt((d * d).mean(1) + 1e-5)
    y = d * rstd[:, None]
    if s["weight"] is not None:
        y = y * s["weight"].float() + s["bias"].float()
    return y.to(s["x"].dtype), mean, rstd


def _norm_grad(s):
    if own:
        import symplex_b200 as sx
        return sx.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["weight"])
    dy = s["dy"].float()
    xh = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
    g = dy * s["weight"].float() if s["weight"] is not None else dy
    dx = (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True)) * s["rstd"][:, None]
    dx = dx.to(s["x"].dtype)
    if s["weight"] is None:
        return dx, None, None
    return dx, (dy * xh).sum(0).to(s["weight"].dtype), dy.sum(0).to(s["weight"].dtype)


def _logits(s):
    return s["x"].float() @ s["weight"].float().t()


def _loss(s):
    if own:
        import symplex_b200 as sx
        return sx.linear_cross_entropy(s["x"], s["weight"], s["targets"], ignore_index=IGNORE, reduction=s["reduction"])
    logits = _logits(s)
    top = logits.max(1).values
    lse = top + (logits - top[:, None]).exp().sum(1).log()
    counted = s["targets"] != IGNORE
    at = torch.where(counted, s["targets"], 0)
    loss = torch.where(counted, lse - logits.gather(1, at[:, None])[:, 0], 0.0)
    if s["reduction"] == "mean":
        loss = loss.sum() / counted.sum()
    elif s["reduction"] == "sum":
        loss = loss.sum()
    return loss, lse


def _loss_grad(s):
    if own:
        import symplex_b200 as sx
        return sx.linear_cross_entropy_backward(s["dloss"], s["x"], s["weight"], s["targets"], s["lse"], ignore_index=IGNORE,
                                                reduction=s["reduction"])
    counted = s["targets"] != IGNORE
    at = torch.where(counted, s["targets"], 0)
    scale = s["dloss"] / counted.sum() if s["reduction"] == "mean" else s["dloss"]
    scale = torch.where(counted, scale, 0.0)
    grad = _logits(s).sub_(s["lse"][:, None]).exp_()
    grad.scatter_add_(1, at[:, None], torch.full_like(s["lse"], -1.0)[:, None])
    grad.mul_(scale[:, None])
    dx = (grad @ s["weight"].float()).to(s["x"].dtype)
    dw = (grad.t() @ s["x"].float()).to(s["weight"].dtype)
    return dx, dw


def _int4(s):
    if own:
        import symplex_b200 as sx
        return sx.int4_matvec(s["x"], s["codes"], s["scales"], s["zeros"], group_size=s["group"])
    n, half = s["codes"].shape
    codes = torch.stack([s["codes"] & 15, s["codes"] >> 4], 2).reshape(n, -1, s["group"]).float()
    zero = s["zeros"].float()[:, :, None] if s["zeros"] is not None else 8.0
    w = ((codes - zero) * s["scales"].float()[:, :, None]).reshape(n, 2 * half)
    return (s["x"].float() @ w.t()).to(s["x"].dtype)


_RUN = {"norm": _norm, "norm_grad": _norm_grad, "loss": _loss, "loss_grad": _loss_grad, "int4": _int4}


def run(state):
    return _RUN[state["op"]](state)


# ------------------------------------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    f = lambda t: None if t is None else t.double()  # noqa: E731
    if case["op"] == "norm":
        x = f(s["x"])
        var, mean = torch.var_mean(x, dim=1, unbiased=False)
        y = (x - mean[:, None]) / torch.sqrt(var[:, None] + 1e-5)
        if s["weight"] is not None:
            y = torch.addcmul(f(s["bias"])[None], y, f(s["weight"])[None])
        return y, mean, (var + 1e-5) ** -0.5
    if case["op"] == "norm_grad":
        x, dy, mean, rstd = f(s["x"]), f(s["dy"]), f(s["mean"])[:, None], f(s["rstd"])[:, None]
        xh = (x - mean) * rstd
        g = dy if s["weight"] is None else dy * f(s["weight"])
        c = case["cols"]
        dx = rstd / c * (c * g - g.sum(1, keepdim=True) - xh * torch.einsum("rc,rc->r", g, xh)[:, None])
        if s["weight"] is None:
            return dx, None, None
        return dx, torch.einsum("rc,rc->c", dy, xh), torch.einsum("rc->c", dy)
    if case["op"] in ("loss", "loss_grad"):
        w, targets = f(s["weight"]), s["targets"]
        counted = targets >= 0
        step = max(1, (1 << 27) // case["vocab"])
        losses, lses, dx, dw = [], [], [], torch.zeros_like(w)
        for r in range(0, case["tokens"], step):
            x, t, c = f(s["x"][r:r + step]), targets[r:r + step], counted[r:r + step]
            logits = torch.einsum("th,vh->tv", x, w)
            rows = torch.arange(len(t), device="cuda")
            if case["op"] == "loss":
                lse = torch.logsumexp(logits, 1)
                lses.append(lse)
                losses.append((lse - logits[rows, t.clamp(min=0)]) * c)
            else:
                g = torch.exp(logits - f(s["lse"][r:r + step])[:, None])
                g[rows, t.clamp(min=0)] -= 1
                d = f(s["dloss"])
                d = d[r:r + step] if case["reduction"] == "none" else (d / counted.sum() if case["reduction"] == "mean" else d)
                g *= (d * c)[:, None]
                dx.append(g @ w)
                dw += g.t() @ x
        if case["op"] == "loss_grad":
            return torch.cat(dx), dw
        loss = torch.cat(losses)
        if case["reduction"] != "none":
            loss = loss.sum() / (counted.sum() if case["reduction"] == "mean" else 1)
        return loss, torch.cat(lses)
    n, k = case["n"], case["k"]
    w = torch.empty(n, k, dtype=torch.float64, device="cuda")
    w[:, 0::2] = (s["codes"] % 16).double()
    w[:, 1::2] = (s["codes"] // 16).double()
    w -= f(s["zeros"]).repeat_interleave(case["group"], 1) if s["zeros"] is not None else 8
    w *= f(s["scales"]).repeat_interleave(case["group"], 1)
    return torch.einsum("mk,nk->mn", f(s["x"]), w)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without

def work(case):
    op, eb = case["op"], _EB[case["dtype"]]
    if op == "norm":
        r, c = case["rows"], case["cols"]
        return {"bytes": 2 * r * c * eb + 8 * r + (2 * c * eb if case["affine"] else 0), "flops": 8 * r * c}
    if op == "norm_grad":
        r, c = case["rows"], case["cols"]
        return {"bytes": 3 * r * c * eb + 8 * r + (3 * c * eb if case["affine"] else 0), "flops": 14 * r * c}
    if op in ("loss", "loss_grad"):
        t, h, v = case["tokens"], case["hidden"], case["vocab"]
        if op == "loss":
            return {"bytes": (t + v) * h * eb + 16 * t, "flops": 2 * t * h * v}
        # the logits are not kept, so the backward pass computes them again
        return {"bytes": 2 * (t + v) * h * eb + 12 * t, "flops": 6 * t * h * v}
    m, n, k = case["tokens"], case["n"], case["k"]
    groups = n * (k // case["group"])
    return {"bytes": n * k // 2 + groups * (eb + (1 if case["zeros"] else 0)) + (m * k + m * n) * eb, "flops": 2 * m * n * k}
