"""Plain 64-bit definitions of the vocabulary operators, with the error that
their 32-bit sums may make beside each value."""
from __future__ import annotations

import math

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # half a step, relative


def dequant(codes, scales, zeros):
    b = codes.to(torch.int64)
    q = torch.stack([b % 16, b // 16], 2).double().reshape(codes.shape[0], -1)
    g = q.shape[1] // scales.shape[1]
    z = 8.0 if zeros is None else zeros.double().repeat_interleave(g, 1)
    return (q - z) * scales.double().repeat_interleave(g, 1)


def head(hidden, codes, scales, zeros, out_dtype, parts=9):
    """Logits and their tolerance.  The products are exact; a group's sum
    grows in steps of 16 columns (the tensor core's), the groups' sums and up
    to `parts` CTAs' parts are added one at a time: each addition is taken to
    lose two units of the last place of the sum of magnitudes (an accumulator
    that truncates loses one)."""
    w = dequant(codes, scales, zeros)
    h = hidden.double()
    ref = h @ w.t()
    groups = scales.shape[1]
    steps = w.shape[1] // groups // 16 + groups + parts + 2
    tol = (h.abs() @ w.abs().t()) * steps * 2.0 ** -22
    return ref, tol + ref.abs() * HALF[out_dtype]


# Relative error of a 32-bit sum of exponentials: the exponential itself
# (2^-21), the rounding of its argument and of log2(e) / T (2^-23 of the
# argument, whose mean under the distribution is at most log2 V <= 21), and
# some 130 additions in a row (a thread's vectors, the warp, the block, the
# cluster) at 2^-24: under 1.2e-5.
SUM = 1.2e-5


def rows(logits, ids, T):
    """(valid, lse, logp) in 64 bits; an empty row has -inf.  The maximum is
    taken off before anything is added: beside a maximum of 1e38 the logarithm
    of the sum would be lost in 64 bits too."""
    V = logits.shape[1]
    x = logits.double() / T
    valid = (ids >= 0) & (ids < V)
    m = x.amax(1)
    total = (x - torch.where(m == -math.inf, 0.0, m)[:, None]).exp().sum(1).log()
    lse = m + total
    lp = x.gather(1, ids.clamp(0, V - 1)[:, None])[:, 0] - m - total
    lp = torch.where(lse == -math.inf, -math.inf, lp)
    return valid, lse, torch.where(valid, lp, 0.0)


def grad(logits, ids, T, lse, g, dtype, rel=SUM):
    """g / T (onehot - softmax) and its tolerance: the probability's relative
    error `rel` plus 2^-22 of its logarithm (argument and factor), the
    rounding of g and of the subtraction at the id, and the output's."""
    V = logits.shape[1]
    x = logits.double() / T
    dead = (lse == -math.inf)[:, None]
    lp = torch.where(dead, -math.inf, x - torch.where(dead, 0.0, lse[:, None]))
    p = lp.exp()
    hot = torch.zeros_like(p)
    ok = (ids >= 0) & (ids < V)
    hot[torch.arange(len(ids), device=ids.device)[ok], ids[ok]] = 1.0
    gT = (torch.where(ok & (lse != -math.inf), g, 0.0) / T)[:, None]
    ref = gT * (hot - p)
    small = torch.where(p > 0, lp.clamp(min=-1000).abs() * 1.4427 * 2.0 ** -22, 0.0)
    tol = gT.abs() * (p * (rel + small) + (hot + p) * 2.0 ** -23) + ref.abs() * HALF[dtype] + 2.0 ** -125 * (1 + gT.abs())
    return ref, tol


def policy(logits, ids, old, adv, T, lo, hi, beta, ref, weights):
    """(loss, its tolerance, logp, d) where d is d(weights loss) / d logp and
    `d_tol` its own error through logp."""
    valid, lse, lp = rows(logits, ids, T)
    A = adv.double()
    dead = lse == -math.inf
    r = torch.ones_like(lp) if old is None else (lp - old.double()).exp()
    plain, cut = r * A, r.clamp(1 - lo, 1 + hi) * A
    loss = -torch.minimum(plain, cut)
    d = torch.where(plain <= cut, -plain, 0.0)
    tol = plain.abs()
    d_tol = plain.abs()
    if ref is not None and beta:
        q = ref.double() - lp
        loss = loss + beta * (q.exp() - q - 1)
        d = d + beta * (1 - q.exp())
        tol = tol + beta * (q.exp() + 1)
        d_tol = d_tol + beta * q.exp()
    d = torch.where(lp == -math.inf, 0.0, d)
    live = valid & ~dead
    w = 1.0 if weights is None else weights.double()
    loss = torch.where(live, loss, 0.0)
    d = torch.where(live, d * w, 0.0)
    err = SUM + 2.0 ** -23 * lp.abs().clamp(max=1e30)
    return loss, torch.where(live, tol * err, 0.0) + loss.abs() * 2.0 ** -23, lp, d, torch.where(live, d_tol * w * err, 0.0), lse


def embed_grad(ids, dout, V, scale, base, out_dtype):
    ok = (ids >= 0) & (ids < V)
    at = torch.where(ok, ids, V)
    ref = torch.zeros(V + 1, dout.shape[1], dtype=torch.float64, device=dout.device)
    mag = torch.zeros_like(ref)
    ref.index_add_(0, at, dout.double())
    mag.index_add_(0, at, dout.double().abs())
    count = torch.bincount(at, minlength=V + 1).double()[:V, None]
    ref, mag = ref[:V] * scale, mag[:V] * abs(scale)
    if base is not None:
        ref, mag = ref + base.double(), mag + base.double().abs()
    # one addition per token, the product and the base's
    return ref, mag * (count + 3) * 2.0 ** -24 + ref.abs() * HALF[out_dtype]
