"""Window attention in float64, with a bound for each output element of what
fp32 arithmetic and the roundings to the operands' type may change.

With u = 2^-24 and t the operands' half step (bf16 2^-8, fp32 2^-24):
a score is a sum of d products, off by (d + 3) u alpha sum |q||k|, and its
exponential by as much and by 4 u |s - m| + 4 u more (the argument's scaling
and rounding, v_exp_f32's ulp); `off` is the largest of a row's.  A probability
rounds once more to the operands' type (t) on its way into the second
product.  A sum of n terms is off by n u of the sum of its terms' sizes.
"""
import math

import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def visible(nq, nk, window, sinks):
    p = torch.arange(nq)[:, None] + nk - nq
    j = torch.arange(nk)[None]
    return (j <= p) & ((p - j < window) | (j < sinks))


def softmax(q, k, v, see, alpha, t):
    """(o, its bound, p, log_sum, its bound, off) of one head."""
    d, n = q.shape[1], max(1, see.shape[1])
    s = alpha * (q @ k.T)
    s = s.masked_fill(~see, -math.inf)
    size = abs(alpha) * (q.abs() @ k.abs().T)
    top = s.amax(1, keepdim=True) if s.shape[1] else torch.full(
        (len(s), 1), -math.inf, dtype=torch.float64)
    some = see.any(1, keepdim=True)
    top = torch.where(some, top, 0.0)
    e = torch.where(see, torch.exp(s - top), 0.0)
    total = e.sum(1, keepdim=True)
    p = torch.where(some, e / torch.where(some, total, 1.0), 0.0)
    off = torch.where(see, (d + 3) * U * size + 4 * U * (s - top).abs() +
                      4 * U, 0.0)
    # (the maximum that is taken off is off itself, by the same in all)
    off = off.amax(1, keepdim=True) if n and off.shape[1] else torch.zeros(
        (len(s), 1), dtype=torch.float64)
    o = p @ v
    bound = (2 * off + (n + 4) * U + t) * (p @ v.abs()) + t * o.abs()
    log_sum = torch.where(some, top + total.log(), -math.inf)[:, 0]
    log_bound = (off + (n + 4) * U)[:, 0] + 8 * U * torch.where(
        some[:, 0], log_sum.abs() + top[:, 0].abs(), 0.0)
    return o, bound, p, log_sum, log_bound, off


def gradients(q, k, v, do, see, alpha, t):
    """(dq, dk, dv) of one head and their bounds."""
    d, n, m = q.shape[1], max(1, see.shape[1]), max(1, see.shape[0])
    o, o_bound, p, log_sum, log_bound, off = softmax(q, k, v, see, alpha, t)
    dp = do @ v.T
    delta = (do * o).sum(1, keepdim=True)
    r = dp - delta
    ds = p * r
    # a probability comes again from the scores and the stored logarithm
    rel = 2 * off + log_bound[:, None] + 8 * U
    sizes = do.abs() @ v.abs().T + (do * o).abs().sum(1, keepdim=True)
    e = p * ((rel + t) * r.abs() + (1 + rel + t) * (
        (d + 4) * U * sizes + (do.abs() * o_bound).sum(1, keepdim=True)))
    a = abs(alpha)
    dq, dk, dv = alpha * ds @ k, alpha * ds.T @ q, p.T @ do
    dq_b = a * (e @ k.abs() + (n + 4) * U * (ds.abs() @ k.abs())) + t * dq.abs()
    dk_b = a * (e.T @ q.abs() + (m + 4) * U * (ds.abs().T @ q.abs()))
    dv_b = ((rel + t) * p).T @ do.abs() + (m + 4) * U * (p.T @ do.abs())
    return (dq, dk, dv), (dq_b, dk_b, dv_b)


def check(name, got, want, bound):
    got, want, bound = got.double().cpu(), want.double(), bound.double()
    assert got.shape == want.shape, name
    exact = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), \
        f"{name}: NaN in other places"
    both = exact & ~torch.isnan(want)
    assert torch.equal(got[both], want[both]), f"{name}: infinities differ"
    d = (got - want).abs()[~exact]
    # (1e-30: results below what bf16 and fp32 hold to full precision)
    bad = d > bound[~exact] + 1e-30
    if bad.any():
        ratio = (d / (bound[~exact] + 1e-30)).max()
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} "
                             f"values off, up to {ratio:.3g} of their bound")
