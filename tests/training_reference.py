"""64-bit restatements of the training operators and the error bounds the GPU tests use.

Bounds count roundings: a value held in a 16-bit type is off by at most half a step,
``finfo(t).eps / 2`` relative (plus half of the smallest subnormal); a k-term sum in fp32 by
k 2^-24 times the sum of magnitudes when its adds round to nearest, and by k 2^-23 when they
may truncate, as tensor-core accumulation may."""

from __future__ import annotations

import torch

U32 = 2.0 ** -24


def rounding(value: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Half a step of `dtype` at `value` (float64)."""
    info = torch.finfo(dtype)
    return value.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


# ---- LayerNorm ------------------------------------------------------------------


def layer_norm(x, gamma, beta, eps, residual=None):
    """(sum in x's type, y, mean, rstd) with y, mean, rstd in float64."""
    total = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    t = total.double()
    mean = t.mean(1, keepdim=True)
    rstd = ((t - mean).square().mean(1, keepdim=True) + eps).rsqrt()
    return total, (t - mean) * rstd * gamma.double() + beta.double(), mean, rstd


def layer_norm_bound(total, gamma, beta, y, mean, rstd):
    """|y - exact|: the mean is a fp32 sum whose longest chain has 8 (a thread's columns) + 5
    (its warp) + 16 (warps) adds, so it is off by 29 u mean|s|; h inherits that times rstd
    and, through the variance (the same chain and its own three roundings, halved by the
    square root), 20 u |h| more; then the products and the output's rounding."""
    t = total.double()
    shift = 32 * U32 * t.abs().mean(1, keepdim=True) * rstd
    h = (t - mean) * rstd
    # A shifted mean moves the variance by (shift of the mean)^2 only.
    off = (shift + (24 * U32 + shift.square()) * h.abs()) * gamma.double().abs() + 4 * U32 * beta.double().abs()
    return off + rounding(y.abs() + off, total.dtype)


def layer_norm_grads(dy, total, gamma, mean, rstd, dsum=None):
    t, d = total.double(), dy.double()
    h = (t - mean) * rstd
    w = d * gamma.double()
    dx = rstd * (w - w.mean(1, keepdim=True) - h * (w * h).mean(1, keepdim=True))
    return dx + (0 if dsum is None else dsum.double()), (d * h).sum(0), d.sum(0)


def layer_norm_grad_bounds(dy, total, gamma, mean, rstd, dx, dsum=None):
    """Bounds of dx, dgamma and dbeta: h is off by e = 32 u mean|s| rstd + 24 u |h| (above);
    the row means are chains of at most 29 adds; the column sums are sums over the rows in
    an order of at most rows adds."""
    t, d = total.double(), dy.double()
    rows = t.shape[0]
    h = (t - mean) * rstd
    e = 32 * U32 * t.abs().mean(1, keepdim=True) * rstd + 24 * U32 * h.abs()
    w = (d * gamma.double()).abs()
    m1 = 34 * U32 * w.mean(1, keepdim=True)
    wh_mean = (d * gamma.double() * h).mean(1, keepdim=True).abs()
    m2 = (w * e).mean(1, keepdim=True) + 36 * U32 * (w * h.abs()).mean(1, keepdim=True)
    inner = 4 * U32 * w + m1 + h.abs() * m2 + e * (wh_mean + m2) + 4 * U32 * (w.mean(1, keepdim=True) + h.abs() * wh_mean)
    off = rstd * inner + 24 * U32 * dx.abs()
    if dsum is not None:
        off = off + 2 * U32 * (dx.abs() + dsum.double().abs())
    return (off + rounding(dx.abs() + off, total.dtype),
            (d.abs() * e).sum(0) + (rows + 2) * U32 * (d * h).abs().sum(0), (rows + 2) * U32 * d.abs().sum(0))


# ---- vocabulary losses ---------------------------------------------------------------


def label_targets(labels, vocab, ignore_index):
    """Target matrix [n, vocab] and the rows that have one."""
    labels = labels.long()
    valid = (labels != ignore_index) & (labels >= 0) & (labels < vocab)
    t = torch.zeros((labels.shape[0], vocab), dtype=torch.float64, device=labels.device)
    t[valid.nonzero().squeeze(1), labels[valid]] = 1.0
    return t, valid, torch.zeros(labels.shape[0], dtype=torch.float64, device=labels.device)


def teacher_targets(tokens, logits, vocab, temperature):
    """Target matrix, the rows that have a target, and sum t log t per row."""
    tokens = tokens.long()
    keep = (tokens >= 0) & (tokens < vocab) & (logits.double() != -torch.inf)
    z = torch.where(keep, logits.double() / temperature, -torch.inf)
    valid = keep.any(1)
    z = torch.where(valid.unsqueeze(1), z, 0.0)
    p = torch.softmax(z, 1) * (keep & valid.unsqueeze(1))
    t = torch.zeros((tokens.shape[0], vocab), dtype=torch.float64, device=tokens.device)
    t.scatter_add_(1, torch.where(keep, tokens, 0), p)
    return t, valid, torch.special.xlogy(p, p).sum(1)


def vocab_loss(x, weight, targets, temperature=1.0):
    """(losses, lse, G per unit of dloss) in float64."""
    t, valid, entropy = targets
    z = x.double() @ weight.double().t() / temperature
    lse = torch.logsumexp(z, 1)
    dot = torch.where(t != 0, t * z, 0.0).sum(1)
    losses = torch.where(valid, temperature ** 2 * (entropy + t.sum(1) * lse - dot), 0.0)
    g = torch.where(valid.unsqueeze(1), temperature * ((z - lse.unsqueeze(1)).exp() - t), 0.0)
    return losses, lse, g


def logit_bound(x, weight, temperature=1.0):
    """[n]: the largest error of a row's z / T: a width-term tensor-core sum, the product with
    the rounded log2(e) / T and the exponent's base change."""
    d = x.shape[1]
    mag = (x.double().abs() @ weight.double().abs().t()).amax(1) / temperature
    return (d * 2 * U32 + 4 * U32) * mag


def loss_bounds(x, weight, targets, losses, lse, temperature=1.0, entries=1):
    """lse moves by at most the largest logit error; its sum has at most vocab adds but runs
    over at most 128-column slices (8 rounds of 4 adds) and their merge, so 2^-16 covers it
    with the exponentials' 2^-22; the loss adds the target's error and T^2 times the terms'
    own roundings (probabilities and their fp32 dot product over the entries)."""
    dz = logit_bound(x, weight, temperature)
    off_lse = dz + 2.0 ** -16 + 2 * U32 * lse.abs()
    mag = (x.double().abs() @ weight.double().abs().t()).amax(1) / temperature
    off = off_lse + dz + (entries + 8) * 4 * U32 * (mag + lse.abs()) + 2.0 ** -20
    return temperature ** 2 * off + 2 * U32 * losses.abs(), off_lse


def grad_bounds(x, weight, g, dloss, lse, dx, dweight, temperature=1.0, t=None, entries=1, parts=1):
    """G's error is p times the error of its exponent (the logit's, the given lse's rounding,
    the exponential's 2^-22), plus half a step of its 16-bit type, plus what the common scale
    2^13..2^14 over max |dloss T| flushes (2^-38 of that maximum); dx and dweight are sums of
    vocab or rows products of the tensor cores over it, rounded once.

    With two parts G's rounding is that of what its rounding left off.

    With the targets t given, p is g / T + t itself, also where it exceeds a target.  A teacher's
    probabilities are off by 64 u at most, those of equal tokens together: exponents at a
    distance D below the largest take three roundings, 3 u D, and the mean of D under t is at
    most log(256) < 5.6, in the entries and again in their sum (17 u each); the exponential
    is off by 4 u in both; the sum has 8 + 5 adds, the quotient and the sum of equals one
    rounding each: 17 + 17 + 8 + 13 + 2 = 57."""
    dtype = x.dtype
    eps = torch.finfo(dtype).eps
    gain = dloss.double().abs().unsqueeze(1)
    dz = (logit_bound(x, weight, temperature) * 2 + 2.0 ** -16 + 8 * U32 * lse.abs()).unsqueeze(1)
    p = (g.abs() + temperature)  # |g| = T |p - t| and t <= 1: p <= |g| / T + 1
    soft = torch.minimum(p, torch.full_like(p, temperature))
    # Tighter where there is no target: p is |g| itself.
    soft = torch.where(g >= 0, torch.minimum(soft, g.clamp(min=0) + torch.where(g > 0, 0.0, temperature)), soft)
    target = 4 * U32 * temperature
    if t is not None:
        soft = (g + temperature * t).clamp(min=0)
        target = temperature * (4 + 64 * (t > 0) * (entries > 1)) * U32
    big = (dloss.double().abs().max() * temperature) * 2.0 ** -38
    off_g = gain * (soft * (torch.expm1(dz) + 2.0 ** -20) + target) + gain * g.abs() * (eps / 2) ** parts + big
    full = gain * g.abs()
    w, a = weight.double().abs(), x.double().abs()
    vocab, rows = weight.shape[0], x.shape[0]
    off_dx = off_g @ w + (vocab + 160) * 2 * U32 * (full @ w)
    off_dw = off_g.t() @ a + (rows + 64) * 2 * U32 * (full.t() @ a)
    return off_dx + rounding(dx.abs() + off_dx, dtype), off_dw + rounding(dweight.abs() + off_dw, dtype)


def worst(actual: torch.Tensor, expected: torch.Tensor, bound: torch.Tensor) -> float:
    """The largest |actual - expected| as a share of its bound."""
    assert torch.isfinite(actual.double()).all(), "non-finite output"
    return float(((actual.double() - expected).abs() / bound.clamp(min=1e-300)).max()) if actual.numel() else 0.0
