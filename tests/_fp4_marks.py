"""Caches of 4-bit codes whose values mark the tile of 32 keys that they lie in,
so that a tile which attention leaves out, takes twice or takes from another
sequence shows among any number of keys.

Key j of sequence i has one element of its value at 1, number (j / 32 + 3 i + 5
times its head) mod d, the others at zero: an output element is the probability
of the tiles that mark it, and every term of it is positive, so that its error
is relative to itself.  Scores are q0 a + q1 b: a, of the key's first element,
is the same for all tiles that mark one element and spreads over 24 (for the
maxima of parts), b is a key's own and moves its score by 3/8 at most.  All are
exact in fp32.

With u = 2^-24: the exponent's scale is off by 2 u of it, its argument by u, the
exponential by 2 u, and so for a part's maximum against another's, at most three
times on its way to the result: 6 S + 16 u in all for scores whose spread is S
powers of two.  A probability is cut to 2^-15 (bf16) or 2^-23.  A wave takes
every fourth tile of its workgroup's, no more than all of the sequence's T, each
`parts` times into a sum of 33 terms; a workgroup joins eight sums, and up to
T / 8 + 2 parts (a workgroup has 8 tiles or more of a split sequence) are joined
with 8 roundings each at most: 33 parts ceil(T / 4) + T + 64 roundings.
"""
import math

import torch

from _fp4_check import LEVELS, U

SIZES = torch.cat([LEVELS, -LEVELS])  # of a code
ONE = 127  # the scale byte of 1


def tile_codes(tile, d):
    """The code of a, for tiles that mark one element the same."""
    return (tile % d * 7) % 16


def key_codes(j):
    """The code of b."""
    return (j * 5 + j // 32) % 16


def queries(h):
    """(q0, q1) of each head, exact in bf16."""
    i = torch.arange(h)
    return (i % 5 - 2.0).double(), torch.where(i % 2 == 0, 1, -1).double() / 16


def build(dtype, lengths, page, h, hk, d, capacity, seed):
    """CPU operands as test_gpu_fp4_attention's `make` gives them; NaN in every
    row that holds no key."""
    gen = torch.Generator().manual_seed(seed)
    n = len(lengths)
    if page:
        need = [-(-m // page) for m in lengths]
        order = torch.randperm(sum(need) + 2, generator=gen)
        width = max(-(-capacity // page), max(need))
        table = torch.full((n, width), -7, dtype=torch.int32)
        at = 0
        for i, m in enumerate(need):
            table[i, :m] = order[at:at + m].to(torch.int32)
            at += m
        shape = (sum(need) + 2, page, hk)
    else:
        table, shape = None, (n, capacity, hk)
    caches = []
    for _ in "kv":
        caches.append([torch.zeros(*shape, d // 2, dtype=torch.uint8),
                       torch.full((*shape, d // 32), 255, dtype=torch.uint8)])
    for i, m in enumerate(lengths):
        j = torch.arange(m)
        at, slot = torch.full_like(j, i), j
        if page:
            at, slot = table[i].long()[j // page], j % page
        for codes, scales in caches:
            scales[at, slot] = ONE
        codes = caches[0][0]
        codes[at, slot, :, 0] = (tile_codes(j // 32, d) + 16 * key_codes(
            j)).to(torch.uint8)[:, None]
        codes = caches[1][0]
        for head in range(hk):
            c = (j // 32 + 3 * i + 5 * head) % d
            codes[at, slot, head, c // 2] = torch.where(
                c % 2 == 0, 0x02, 0x20).to(torch.uint8)
    q = torch.zeros(n, h, d, dtype=torch.float64)
    q[:, :, 0], q[:, :, 1] = queries(h)
    return {"lengths": torch.tensor(lengths, dtype=torch.int32),
            "table": table, "query": q.to(dtype), "key_cache": caches[0],
            "value_cache": caches[1]}


def weights(n, h, d, window, sinks):
    """[h, tiles]: the sums over each tile of exp(score - the largest), and how
    many of its keys are seen."""
    j = torch.arange(n)
    j = j[(j >= n - window) | (j < sinks)]
    q0, q1 = queries(h)
    s = (q0[:, None] * SIZES[tile_codes(j // 32, d)] +
         q1[:, None] * SIZES[key_codes(j)])
    p = torch.exp(s - s.amax(1, keepdim=True))
    w = torch.zeros(h, n // 32 + 1, dtype=torch.float64)
    return w.index_add_(1, j // 32, p), torch.bincount(
        j // 32, minlength=n // 32 + 1)


def outputs(w, i, hk, d):
    """[h, d] of sequence i from its tiles' weights."""
    h, tiles = w.shape
    group = h // hk
    p = w / w.sum(1, keepdim=True)
    out = torch.zeros(h, d, dtype=torch.float64)
    for head in range(hk):
        rows = slice(head * group, head * group + group)
        c = (torch.arange(tiles) + 3 * i + 5 * head) % d
        out[rows] = torch.zeros(group, d, dtype=torch.float64).index_add_(
            1, c, p[rows])
    return out


def relative_bound(tiles, dtype):
    bf16 = dtype == torch.bfloat16
    parts, cut = (2, 2.0 ** -15) if bf16 else (3, 2.0 ** -23)
    spread = 2 * (12.0 + 0.375) / math.log(2.0)
    roundings = 33 * parts * -(-tiles // 4) + tiles + 64
    return (2 * (roundings * U + (6 * spread + 16) * U + cut) +
            torch.finfo(dtype).eps / 2)


def expect(x, out, window, sinks):
    n, h, d = out.shape
    hk = x["key_cache"][0].shape[2]
    for i, m in enumerate(x["lengths"].tolist()):
        if m == 0:
            assert not out[i].any(), f"sequence {i}"
            continue
        w, seen = weights(m, h, d, window, sinks)
        want = outputs(w, i, hk, d)
        off = (out[i].double() - want).abs() / want.clamp(min=1e-30)
        most = relative_bound(int((seen > 0).sum()), out.dtype)
        assert (off <= most).all(), (
            f"sequence {i} of {m} keys: {int((off > most).sum())} of "
            f"{off.numel()} elements off, up to {float(off.max()):.3g} of "
            f"themselves, where {most:.3g} are due")


# sequences, their most keys, one's, room, page, window, sinks, heads, key heads:
# rows joined by a wave (more than 512 in all) and by a workgroup, of two parts
# and of more than either takes at once, heads behind the last full workgroup;
# sequences whole and divided, more of them than a wave's lanes and registers hold
CASES = [
    (64, 2600, 2600, 2600, 64, 10 ** 6, 0, 32, 8),
    (80, 300, 9000, 9100, 0, 10 ** 6, 0, 16, 2),
    (40, 700, 20000, 20000, 16, 10 ** 6, 0, 18, 1),
    (600, 300, 2500, 2600, 16, 10 ** 6, 0, 1, 1),
    (300, 900, 3000, 3000, 0, 2000, 700, 2, 1),
    (30, 3000, 3000, 3000, 24, 1000, 2000, 20, 1),
    (1, 40000, 40000, 40000, 0, 10 ** 6, 0, 3, 1),
    (4, 20000, 20000, 20000, 48, 16000, 5, 12, 4),
]


def lengths_of(case):
    """From 0 to the most, a fifth of them 0, and the one."""
    n, most, one = CASES[case][:3]
    gen = torch.Generator().manual_seed(case)
    x = torch.randint(0, most + 1, (n,), generator=gen)
    x[torch.rand(n, generator=gen) < 0.2] = 0
    x[n // 2] = one
    return x.tolist()
