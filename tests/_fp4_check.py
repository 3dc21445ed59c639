"""A cache of 4-bit codes and attention against it in float64, from their
definitions.

With u = 2^-24: a score is a sum of `parts` d products that fp32 holds (a code
has two significant bits, a part of a query eight), off by (parts d + 3) u alpha
sum |q||k|, and its exponential by as much and by 4 u |s - m| + 4 u more.  A
probability is taken as bf16 parts, two to 2^-15 of it (bf16) or three to 2^-23
(fp32).  A product of 32 keys adds up to 33 terms, `parts` times, and joins and
raised maxima scale what is summed now and then: (parts + 1) n + 16 roundings of
u for n keys, in the sums of probabilities and of their values' products.
"""
import math

import torch

U = 2.0 ** -24
LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0],
                      dtype=torch.float64)


def quantise(x):
    """(codes [..., d / 2], scales [..., d / 32]) of x, one block at a time in
    float64: the least power of two that 7 times covers the block, the nearest
    of the eight sizes, the even code of two that are equally near."""
    blocks = x.double().unflatten(-1, (-1, 32))
    finite = torch.isfinite(blocks).all(-1)
    top = torch.where(finite[..., None], blocks, 0.0).abs().amax(-1)
    e = torch.full_like(top, -125.0)
    for k in range(-125, 125):
        e = torch.where(top > 7.0 * 2.0 ** k, k + 1.0, e)
    y = torch.where(finite[..., None], blocks, 0.0) / torch.exp2(e)[..., None]
    gap = (y.abs()[..., None] - LEVELS).abs()
    near = gap.amin(-1, keepdim=True)
    hits = gap == near
    even = torch.tensor([i % 2 == 0 for i in range(8)])
    both = hits.sum(-1, keepdim=True) == 2
    code = torch.where(both, hits & even, hits).to(torch.uint8).argmax(-1)
    code = (code + 8 * torch.signbit(y)).to(torch.uint8)
    code = torch.where(finite[..., None], code, 0).flatten(-2)
    scales = torch.where(finite, e + 127, 255.0).to(torch.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4, scales


def dequantise(codes, scales):
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    x = torch.cat([LEVELS, -LEVELS])[both].unflatten(-1, (-1, 32))
    factor = torch.exp2(scales.double() - 127)
    factor = torch.where(scales == 255, math.nan, factor)
    return (x * factor[..., None]).flatten(-2)


def attend(q, k, v, alpha, dtype):
    """(output, its bound) of rows q [m, d] that see all of k, v [n, d], in
    float64; n = 0 gives zeros."""
    d, n = q.shape[1], len(k)
    if n == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    bf16 = dtype == torch.bfloat16
    score_parts, parts, cut = (1, 2, 2.0 ** -15) if bf16 else (3, 3, 2.0 ** -23)
    s = alpha * (q @ k.T)
    size = abs(alpha) * (q.abs() @ k.abs().T)
    top = s.amax(1, keepdim=True)
    p = torch.softmax(s, 1)
    off = ((score_parts * d + 3) * U * size + 4 * U * (s - top).abs() +
           4 * U).amax(1, keepdim=True)
    o = p @ v
    sums = ((parts + 1) * n + 16) * U
    t = torch.finfo(dtype).eps / 2
    return o, (2 * off + 2 * sums + cut) * (p @ v.abs()) + t * o.abs()
