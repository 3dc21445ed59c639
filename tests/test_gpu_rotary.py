"""Rotary positions on the GPU against extended precision, element by element.

With u = 2^-24: a cosine or sine is off by at most 4 u (the angle's rest within
a quarter turn rounds once, u pi / 4 of it at most, then about two roundings of
the series of sizes up to 1), a result (x, y) by 4 u (|x| + |y|) for both and
another u for its product and sum each, and half a step of its type.
"""
import math

import numpy as np
import pytest
import torch

import sparsewavecomp_amd as sw
from gpu_util import DEV, say

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
U = 2.0 ** -24


def turned(x, positions, frequencies, axes, interleaved, back=False):
    """x [tokens, heads, d] in float64, and what its elements may be off by but
    for the result's own rounding; angles in long double, whose 64 bits hold
    the products of positions and frequencies."""
    pairs = len(frequencies)
    p = positions.numpy().astype(np.longdouble)
    f = frequencies.numpy().astype(np.longdouble)
    angle = np.zeros((x.shape[0], pairs), dtype=np.longdouble)
    for i in range(pairs):
        axis = 0 if axes is None else int(axes[i])
        if 0 <= axis < len(p):
            angle[:, i] = p[axis] * f[i]
    cos = torch.from_numpy(np.cos(angle).astype(np.float64))[:, None]
    sin = torch.from_numpy(np.sin(angle).astype(np.float64))[:, None]
    if back:
        sin = -sin
    x = x.double()
    first = slice(0, 2 * pairs, 2) if interleaved else slice(0, pairs)
    second = slice(1, 2 * pairs, 2) if interleaved else slice(pairs, 2 * pairs)
    a, b = x[..., first], x[..., second]
    y, bound = x.clone(), torch.zeros_like(x)
    y[..., first], y[..., second] = a * cos - b * sin, a * sin + b * cos
    bound[..., first] = bound[..., second] = 6 * U * (a.abs() + b.abs())
    return y, bound


def check(name, got, want, bound):
    t = torch.finfo(got.dtype).eps / 2
    off = (got.double().cpu() - want).abs()
    bad = ~(off <= bound * (1 + t) + t * want.abs() + 1e-37)
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} off, "
                           f"up to {float(off.max()):.3g}")


def make(dtype, tokens, axes, h, hk, d, pairs, seed=0, far=5000):
    gen = torch.Generator().manual_seed(seed)
    positions = torch.randint(-far, far + 1, (axes, tokens), generator=gen,
                              dtype=torch.int64).to(torch.int32)
    frequencies = (10000.0 ** (-torch.arange(pairs).double() / pairs)).float()
    pair_axes = None if axes == 1 else torch.randint(
        0, axes, (pairs,), generator=gen, dtype=torch.int32)
    q = torch.randn(tokens, h, d, generator=gen).to(DTYPES[dtype])
    k = torch.randn(tokens, hk, d, generator=gen).to(DTYPES[dtype])
    return positions, frequencies, pair_axes, q, k


def on_gpu(*x):
    return [None if y is None else y.to(DEV) for y in x]


# tokens, axes, heads, key heads, d, pairs: one token; few and many heads;
# tokens that end inside a workgroup's; odd pairs; a part of a head; one pair
CASES = [
    (1, 1, 1, 1, 8, 4),
    (1, 3, 4, 2, 128, 64),
    (7, 2, 3, 1, 40, 20),
    (33, 1, 2, 2, 64, 32),
    (64, 1, 32, 8, 128, 64),
    (65, 3, 12, 4, 96, 40),
    (19, 2, 5, 1, 80, 1),
    (10, 1, 3, 3, 24, 7),
    (5, 2, 6, 6, 80, 16),
    (300, 1, 1, 1, 8, 3),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_rotary(dev, dtype, interleaved, case):
    say(f"rotary {dtype} {interleaved} {case}")
    p, f, ax, q, k = make(dtype, *case, seed=sum(case))
    pg, fg, ag, qg, kg = on_gpu(p, f, ax, q, k)
    for back in (False, True):
        call = sw.rotary_backward if back else sw.rotary
        qo, ko = torch.full_like(qg, 7.0), torch.full_like(kg, 7.0)
        got = call(pg, fg, ag, qg, kg, qo, ko, interleaved)
        torch.cuda.synchronize()
        assert got[0] is qo and got[1] is ko
        for name, x, y in (("query", q, qo), ("key", k, ko)):
            check(name, y, *turned(x, p, f, ax, interleaved, back))
            rest = 2 * len(f)
            assert torch.equal(y[..., rest:].cpu(), x[..., rest:])
    # in place, and without keys
    alone = torch.empty_like(qg)
    sw.rotary(pg, fg, ag, qg, None, alone, None, interleaved)
    sw.rotary(pg, fg, ag, qg, kg, qg, kg, interleaved)
    torch.cuda.synchronize()
    assert torch.equal(alone, qg)
    check("key in place", kg, *turned(k, p, f, ax, interleaved))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,pairs", [(80, 10), (96, 35), (64, 6), (128, 52),
                                     (128, 2), (8, 2), (104, 52), (120, 59)])
def test_pieces_of_every_width(dev, dtype, interleaved, d, pairs):
    """Pairs that make whole pieces of 16, 8, 4 and 2 bytes."""
    say(f"rotary pieces {dtype} {interleaved} {d} {pairs}")
    p, f, ax, q, k = make(dtype, 45, 2, 3, 2, d, pairs, seed=d + pairs)
    pg, fg, ag, qg, kg = on_gpu(p, f, ax, q, k)
    qo, ko = torch.full_like(qg, 7.0), torch.full_like(kg, 7.0)
    sw.rotary(pg, fg, ag, qg, kg, qo, ko, interleaved)
    check("query", qo, *turned(q, p, f, ax, interleaved))
    check("key", ko, *turned(k, p, f, ax, interleaved))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,pairs", [(40, 5), (40, 20), (96, 25), (128, 1),
                                     (8, 3), (16, 7), (72, 33), (128, 63)])
def test_pieces_that_leave_some_over(dev, dtype, interleaved, d, pairs):
    """What whole pieces leave over of the pairs and of what is copied, within
    rows of more than the heads, in place too; copied elements keep their bits."""
    say(f"rotary rest {dtype} {interleaved} {d} {pairs}")
    p, f, ax, q, k = make(dtype, 333, 3, 3, 1, d, pairs, seed=d + pairs)
    word = torch.int16 if dtype == "bf16" else torch.int32
    odd = torch.tensor([-0.0, math.nan, math.inf, -math.inf], dtype=q.dtype)
    for x in (q, k):
        n = min(4, d - 2 * pairs)
        x[5::7, :, 2 * pairs:2 * pairs + n] = odd[:n]
    pg, fg, ag, qg, kg = on_gpu(p, f, ax, q, k)
    wide = torch.full((333, 4, d + 8), 7.0, dtype=q.dtype, device=qg.device)
    qo, ko = wide[:, :3, :d], torch.full_like(kg, 7.0)
    sw.rotary(pg, fg, ag, qg, kg, qo, ko, interleaved)
    for name, x, y in (("query", q, qo), ("key", k, ko)):
        some = slice(0, 2 * pairs)
        want, bound = turned(x.clone().nan_to_num(0.0, 0.0, 0.0), p, f, ax,
                             interleaved)
        check(name, y[..., some], want[..., some], bound[..., some])
        assert torch.equal(y[..., 2 * pairs:].cpu().contiguous().view(word),
                           x[..., 2 * pairs:].contiguous().view(word))
    assert (wide[:, 3] == 7.0).all() and (wide[..., d:] == 7.0).all()
    sw.rotary(pg, fg, ag, qg, kg, qg, kg, interleaved)
    assert torch.equal(qg.view(word), qo.contiguous().view(word))
    assert torch.equal(kg.view(word), ko.view(word))


@pytest.mark.parametrize("far", [2 ** 20, 2 ** 31 - 1])
def test_far_positions(dev, far):
    """Whole turns by the million: the rest of the angle is right all the
    same."""
    say(f"rotary far {far}")
    p, f, ax, q, k = make("f32", 2000, 2, 1, 1, 64, 32, seed=3, far=far)
    pg, fg, ag, qg, kg = on_gpu(p, f, ax, q, k)
    sw.rotary(pg, fg, ag, qg, kg, qg, kg)
    check("query", qg, *turned(q, p, f, ax, False))
    check("key", kg, *turned(k, p, f, ax, False))


def test_quarter_turns(dev):
    """Angles next to multiples of a quarter turn, where cosine or sine is
    small: off by 2^-22 of the pair, not of the result."""
    say("rotary quarter turns")
    quarter = np.pi / 2
    p = torch.arange(-600, 600, dtype=torch.int32)[None]
    f = torch.tensor([quarter, quarter / 2, quarter * 3, quarter + 1e-6],
                     dtype=torch.float32)
    gen = torch.Generator().manual_seed(1)
    q = torch.randn(1200, 2, 8, generator=gen)
    pg, fg, qg = on_gpu(p, f, q)
    sw.rotary(pg, fg, None, qg, None, qg, None)
    check("query", qg, *turned(q, p, f, None, False))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients_against_differences(dev, dtype, interleaved):
    """The gradients along a direction are the differences of the float64 form
    along it: sum of gradient times direction = (L(x + h e) - L(x - h e)) / 2 h,
    L = sum of output times its gradient, which is linear in x."""
    say(f"rotary differences {dtype} {interleaved}")
    p, f, ax, q, k = make(dtype, 29, 2, 3, 2, 40, 12, seed=9)
    gen = torch.Generator().manual_seed(10)
    pg, fg, ag = on_gpu(p, f, ax)
    go = [torch.randn(x.shape, generator=gen).to(x.dtype) for x in (q, k)]
    grads = [torch.empty_like(x, device=DEV) for x in (q, k)]
    sw.rotary_backward(pg, fg, ag, *on_gpu(*go), *grads, interleaved)
    for x, g, dx in zip((q, k), go, grads):
        dx = dx.double().cpu()
        t = torch.finfo(x.dtype).eps / 2
        for _ in range(4):
            e = torch.randn(x.shape, generator=gen, dtype=torch.float64)
            loss = [float((turned(x.double() + s * e, p, f, ax,
                                  interleaved)[0] * g.double()).sum())
                    for s in (0.5, -0.5)]
            want, bound = turned(g, p, f, ax, interleaved, True)
            room = ((bound * (1 + t) + t * want.abs()) * e.abs()).sum()
            assert abs((dx * e).sum() - (loss[0] - loss[1])) <= \
                float(room) + 1e-9


def test_axes_that_are_not_there(dev):
    """Their pairs are copied, and nothing outside positions is read."""
    say("rotary axes outside")
    p, f, _, q, k = make("f32", 40, 2, 2, 1, 64, 32, seed=5)
    ax = torch.tensor([0, 1, -1, 2, 2 ** 31 - 1, -2 ** 31, 1, 0] * 4,
                      dtype=torch.int32)
    pg, fg, ag, qg, kg = on_gpu(p, f, ax, q, k)
    sw.rotary(pg, fg, ag, qg, kg, qg, kg)
    check("query", qg, *turned(q, p, f, ax, False))
    assert torch.equal(qg[..., 2].cpu(), q[..., 2])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_infinities_and_nan_stay_in_their_pair(dev, dtype):
    say(f"rotary inf {dtype}")
    p, f, ax, q, k = make(dtype, 20, 1, 2, 2, 64, 32, seed=6)
    pg, fg, qg, kg = on_gpu(p, f, q, k)
    want = torch.empty_like(qg)
    sw.rotary(pg, fg, None, qg, None, want, None)
    qg[3, 1, 5], qg[4, 0, 40], qg[5, 0, 63] = np.nan, np.inf, -np.inf
    got = torch.empty_like(qg)
    sw.rotary(pg, fg, None, qg, None, got, None)
    hit = torch.zeros(q.shape, dtype=torch.bool)
    hit[3, 1, [5, 37]] = hit[4, 0, [8, 40]] = hit[5, 0, [31, 63]] = True
    assert not torch.isfinite(got.cpu()[hit]).any()
    assert torch.equal(got.cpu()[~hit], want.cpu()[~hit])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_strides(dev, dtype):
    """Queries and keys as slices of one projection's output, outputs with heads
    before tokens; what lies between is left alone."""
    say(f"rotary strides {dtype}")
    p, f, ax, q, k = make(dtype, 37, 3, 4, 2, 64, 24, seed=7)
    pg, fg, ag, qg, kg = on_gpu(p, f, ax, q, k)
    want = sw.rotary(pg, fg, ag, qg, kg, torch.empty_like(qg),
                     torch.empty_like(kg))
    both = torch.cat([qg, kg, torch.full_like(kg, 5.0)], 1)
    qo = torch.full((4, 50, 64), 7.0, dtype=q.dtype, device=DEV)
    ko = torch.full((37, 9, 64), 7.0, dtype=q.dtype, device=DEV)
    sw.rotary(pg, fg, ag, both[:, :4], both[:, 4:6],
              qo[:, :37].transpose(0, 1), ko[:, 3:5])
    assert torch.equal(qo[:, :37].transpose(0, 1), want[0])
    assert torch.equal(ko[:, 3:5], want[1])
    assert (qo[:, 37:] == 7).all() and (ko[:, :3] == 7).all()
    assert (ko[:, 5:] == 7).all()
    sw.rotary(pg, fg, ag, both[:, :4], both[:, 4:6], both[:, :4], both[:, 4:6])
    assert torch.equal(both[:, :4], want[0])
    assert torch.equal(both[:, 4:6], want[1]) and (both[:, 6:] == 5).all()


def test_past_four_gib(dev):
    """Tokens whose byte offsets pass 2^32."""
    say("rotary past 4 GiB")
    p, f, ax, q, k = make("bf16", 41, 1, 40, 1, 128, 64, seed=8)
    pg, fg, qg, kg = on_gpu(p, f, q, k)
    want = sw.rotary(pg, fg, None, qg, kg, torch.empty_like(qg),
                     torch.empty_like(kg))
    far = (5 << 30) // 2 // 39 // 8 * 8  # elements between heads
    store = torch.empty(far * 39 + 41 * 128, dtype=torch.bfloat16, device=DEV)
    wide = store.as_strided((41, 40, 128), (128, far, 1))
    wide.copy_(qg)
    sw.rotary(pg, fg, None, wide, kg, wide, kg)
    assert torch.equal(wide, want[0])


def test_many_heads(dev):
    """More units of a token than one pass of a workgroup takes."""
    say("rotary many heads")
    p, f, ax, q, k = make("bf16", 3, 1, 700, 100, 128, 64, seed=11)
    pg, fg, qg, kg = on_gpu(p, f, q, k)
    sw.rotary(pg, fg, None, qg, kg, qg, kg)
    check("query", qg, *turned(q, p, f, None, False))
    check("key", kg, *turned(k, p, f, None, False))


def test_repeats_streams_and_graphs(dev):
    say("rotary graph")
    p, f, ax, q, k = make("bf16", 130, 3, 8, 2, 128, 64, seed=12)
    pg, fg, ag, qg, kg = on_gpu(p, f, ax, q, k)
    want = [torch.empty_like(x) for x in (qg, kg)]
    got = [torch.zeros_like(x) for x in (qg, kg)]
    back = [torch.zeros_like(x) for x in (qg, kg)]
    sw.rotary(pg, fg, ag, qg, kg, *want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    sw.rotary(pg, fg, ag, qg, kg, *got, stream=side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sw.rotary(pg, fg, ag, qg, kg, *got)
        sw.rotary_backward(pg, fg, ag, *got, *back)
    for i in range(3):
        pg += 17
        sw.rotary(pg, fg, ag, qg, kg, *want)
        eager = sw.rotary_backward(pg, fg, ag, *want, torch.empty_like(qg),
                                   torch.empty_like(kg))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        assert all(torch.equal(a, b) for a, b in zip(eager, back))
