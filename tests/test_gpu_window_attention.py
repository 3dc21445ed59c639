"""Window attention on the GPU against float64, element by element within
bounds that the arithmetic gives (tests/_window_check.py)."""
import math

import pytest
import torch

import sparsewavecomp_amd as sw
from _window_check import check, gradients, half_step, softmax, visible
from gpu_util import DEV, say

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def offsets(lengths, start=0):
    out = [start]
    for n in lengths:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32)


def inputs(dtype, nq, nk, h, hk, d, seed=0, lead=0, tail=0):
    """CPU operands for sequences of nq[i] queries and nk[i] keys, `lead`
    tokens before the first and `tail` behind the last."""
    gen = torch.Generator().manual_seed(seed)
    def values(n, heads):
        return torch.randn(lead + n + tail, heads, d, generator=gen).to(
            DTYPES[dtype])
    return (offsets(nq, lead), offsets(nk, lead), values(sum(nq), h),
            values(sum(nk), hk), values(sum(nk), hk))


def forward(qo, ko, q, k, v, alpha, window, sinks, fill=7.0):
    out = torch.full(q.shape, fill, dtype=q.dtype, device=DEV)
    lse = torch.full((q.shape[1], q.shape[0]), fill, device=DEV)
    got = sw.window_attention(qo.to(DEV), ko.to(DEV), q.to(DEV), k.to(DEV),
                              v.to(DEV), out, lse, alpha, window, sinks)
    torch.cuda.synchronize()
    assert got is out
    return out.cpu(), lse.cpu()


def expect(qo, ko, q, k, v, out, lse, alpha, window, sinks, fill=7.0,
           heads=None):
    """Every head's results, or those of `heads`."""
    t = half_step(q.dtype)
    g = q.shape[1] // k.shape[1]
    qd, kd, vd = q.double(), k.double(), v.double()
    inside = torch.zeros(q.shape[0], dtype=torch.bool)
    for i in range(len(qo) - 1):
        a, b, c, e = int(qo[i]), int(qo[i + 1]), int(ko[i]), int(ko[i + 1])
        inside[a:b] = True
        see = visible(b - a, e - c, window, sinks)
        for h in heads or range(q.shape[1]):
            o, ob, _, l, lb, _ = softmax(qd[a:b, h], kd[c:e, h // g],
                                         vd[c:e, h // g], see, alpha, t)
            check(f"output of sequence {i}, head {h}", out[a:b, h], o, ob)
            check(f"log_sum of sequence {i}, head {h}", lse[h, a:b], l, lb)
    assert torch.equal(out[~inside], torch.full_like(out[~inside], fill))
    assert torch.equal(lse[:, ~inside], torch.full_like(lse[:, ~inside], fill))


# (queries, keys), window, sinks: one token; a window of one; a window that
# starts inside a tile; sinks that touch it, lie apart and fill more than a
# tile; rows that see nothing (more queries than keys); empty sequences;
# keys before the queries; tile borders at 32, 64 and 128 from both sides
CASES = [
    (([1], [1]), 1, 0),
    (([1], [1]), 4096, 4),
    (([5], [5]), 1, 0),
    (([130], [130]), 1, 1),
    (([33, 0, 127, 1, 129], [33, 0, 127, 1, 129]), 40, 3),
    (([300], [300]), 64, 0),
    (([257], [257]), 31, 100),
    (([400], [400]), 100, 4),
    (([400], [400]), 33, 65),
    (([10, 200], [3, 150]), 50, 2),
    (([7], [0]), 50, 2),
    (([1, 20, 64], [500, 333, 64]), 128, 16),
    (([128, 64], [256, 192]), 128, 0),
    (([500], [500]), 2 ** 31 + 5, 0),
    (([500], [500]), 10, 2 ** 40),
    (([2] * 150, [2] * 150), 2, 0),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_forward(dev, dtype, case):
    (nq, nk), window, sinks = CASES[case]
    say(f"window forward {dtype} {CASES[case]}")
    x = inputs(dtype, nq, nk, 2, 1, 64, seed=case)
    out, lse = forward(*x, 0.125, window, sinks)
    expect(*x, out, lse, 0.125, window, sinks)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_forward_many_heads(dev, dtype, case):
    """The same with so many heads that a workgroup takes 128 rows, whose keys
    are not shared out among its waves."""
    (nq, nk), window, sinks = CASES[case]
    say(f"window forward many heads {dtype} {CASES[case]}")
    x = inputs(dtype, nq, nk, 288, 144, 64, seed=case)
    out, lse = forward(*x, 0.125, window, sinks)
    expect(*x, out, lse, 0.125, window, sinks, heads=[0, 131, 287])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("h,hk,d", [(1, 1, 8), (3, 3, 24), (6, 2, 64),
                                    (4, 1, 72), (2, 2, 96), (8, 2, 128),
                                    (5, 1, 128), (290, 145, 128)])
def test_forward_heads(dev, dtype, h, hk, d):
    say(f"window forward heads {dtype} {h} {hk} {d}")
    x = inputs(dtype, [70, 131], [90, 131], h, hk, d, seed=d + h)
    out, lse = forward(*x, 1 / math.sqrt(d), 48, 5)
    expect(*x, out, lse, 1 / math.sqrt(d), 48, 5,
           heads=None if h < 10 else [0, 3, h - 1])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_forward_leaves_other_tokens(dev, dtype):
    say(f"window forward lead and tail {dtype}")
    x = inputs(dtype, [40, 3, 150], [40, 9, 150], 2, 2, 64, seed=3, lead=13,
               tail=200)
    out, lse = forward(*x, 0.2, 30, 2)
    expect(*x, out, lse, 0.2, 30, 2)


@pytest.mark.parametrize("alpha", [-0.3, 0.0, 4.0])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_forward_alpha(dev, dtype, alpha):
    say(f"window forward alpha {dtype} {alpha}")
    x = inputs(dtype, [200], [200], 2, 1, 64, seed=5)
    out, lse = forward(*x, alpha, 70, 2)
    expect(*x, out, lse, alpha, 70, 2)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_forward_strides(dev, dtype):
    """Slices of one projection's output, heads before tokens, and one key
    head shared by a stride of zero."""
    say(f"window forward strides {dtype}")
    gen = torch.Generator().manual_seed(11)
    t, h, d = 150, 4, 64
    packed = torch.randn(t, 3 * h, d, generator=gen).to(DTYPES[dtype]).to(DEV)
    q, k, v = packed[:, :h], packed[:, h:2 * h], packed[:, 2 * h:]
    qo = offsets([t]).to(DEV)
    plain = torch.empty(t, h, d, dtype=q.dtype, device=DEV)
    sw.window_attention(qo, qo, q.contiguous(), k.contiguous(), v.contiguous(),
                        plain, None, 0.125, 40, 3)
    wide = torch.full((h, t, d), 7.0, dtype=q.dtype, device=DEV)
    sw.window_attention(qo, qo, q, k, v, wide.transpose(0, 1), None, 0.125,
                        40, 3)
    assert torch.equal(wide.transpose(0, 1), plain)
    one_k, one_v = k[:, :1].expand(-1, h, -1), v[:, :1].expand(-1, h, -1)
    shared = torch.empty_like(plain)
    sw.window_attention(qo, qo, q, one_k, one_v, shared, None, 0.125, 40, 3)
    sw.window_attention(qo, qo, q, k[:, :1], v[:, :1], plain, None, 0.125, 40, 3)
    assert torch.equal(shared, plain)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("at", [0, 60, 100, 199])
@pytest.mark.parametrize("heads", [2, 288])
def test_forward_keeps_what_is_masked_apart(dev, dtype, bad, at, heads):
    """An infinity or NaN of one key and value reaches the queries that see
    it, and no others."""
    say(f"window forward {bad} at {at} {dtype} {heads}")
    qo, ko, q, k, v = inputs(dtype, [200], [200], heads, heads, 64, seed=at)
    window, sinks = 50, 2
    sees = visible(200, 200, window, sinks)[:, at]
    clean, clean_lse = forward(qo, ko, q, k, v, 0.125, window, sinks)
    for what in ("value", "key"):
        kk, vv = k.clone(), v.clone()
        (vv if what == "value" else kk)[at, 1, 5] = bad
        out, lse = forward(qo, ko, q, kk, vv, 0.125, window, sinks)
        others = [i for i in range(heads) if i != 1]
        assert torch.equal(out[:, others], clean[:, others])
        assert torch.equal(lse[others], clean_lse[others])
        x, y = out[~sees, 1].float(), clean[~sees, 1].float()
        assert torch.isfinite(x).all()
        # (a repeated pass may add up in another order)
        if not sees.all():
            assert (x - y).abs().max() <= 4 * half_step(q.dtype) * y.abs().max()
        assert torch.isfinite(lse[1][~sees]).all()
        if what == "value":
            hit = out[sees, 1, 5].float()
            assert torch.isnan(hit).all() if math.isnan(bad) else \
                (hit == bad).all()
            rest = torch.cat([out[sees, 1, :5], out[sees, 1, 6:]], 1)
            assert torch.isfinite(rest).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("what", ["key", "value"])
@pytest.mark.parametrize("heads", [2, 288])
def test_forward_keeps_a_first_key_apart_that_is_no_sink(dev, dtype, bad, what,
                                                         heads):
    """The first key without sinks: the rows past the window do not see it, and
    keep the results of clean operands."""
    say(f"window forward {bad} at the first key {dtype} {heads} {what}")
    qo, ko, q, k, v = inputs(dtype, [200], [200], heads, heads, 64, seed=9)
    clean, clean_lse = forward(qo, ko, q, k, v, 0.125, 50, 0)
    (v if what == "value" else k)[0, 1, 5] = bad
    out, lse = forward(qo, ko, q, k, v, 0.125, 50, 0)
    apart = ~visible(200, 200, 50, 0)[:, 0]
    assert int(apart.sum()) == 150
    x, y = out[apart, 1].float(), clean[apart, 1].float()
    assert torch.isfinite(x).all()
    # (a repeated pass may add up in another order)
    assert (x - y).abs().max() <= 4 * half_step(q.dtype) * y.abs().max()
    x, y = lse[1][apart], clean_lse[1][apart]
    assert (x - y).abs().max() <= 8 * half_step(torch.float32) * y.abs().max()
    hit = out[~apart, 1, 5].float()
    if what == "key" and bad == math.inf:
        # a score of inf, or of -inf, which leaves the key out: NaN, but for the
        # rows of a negative element, of which the first sees no other key
        nan = q[~apart, 1, 5] > 0
        nan[0] = True
        assert torch.equal(torch.isnan(hit), nan)
    else:
        assert torch.isnan(hit).all() if math.isnan(bad) else \
            (hit == bad).all()
    out[:, 1], clean[:, 1], lse[1], clean_lse[1] = 0, 0, 0, 0
    assert torch.equal(out, clean) and torch.equal(lse, clean_lse)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,d", [(2, 64), (288, 64), (2, 128), (288, 128)])
@pytest.mark.parametrize("alpha,size", [(0.125, 3.0e38), (4.0, 3.0e38),
                                        (0.0, 3.0e38), (0.0, 8.0e36)])
def test_forward_of_large_values(dev, dtype, heads, d, alpha, size):
    """Values whose weighted mean is finite while a sum of them is not, in one
    head and sequence; the others keep their bits."""
    say(f"window forward large values {dtype} {heads} {d} {alpha} {size}")
    x = list(inputs(dtype, [200, 40], [230, 40], heads, heads, d, seed=21))
    clean, clean_lse = forward(*x, alpha, 60, 2)
    gen = torch.Generator().manual_seed(22)
    v = x[4].clone()
    v[:230, 1] = ((0.5 + torch.rand(230, d, generator=gen) / 2) * size).to(
        v.dtype)
    v[:230, 1, d // 2:] *= -1
    x[4] = v
    out, lse = forward(*x, alpha, 60, 2)
    assert torch.isfinite(out).all()
    expect(*x, out, lse, alpha, 60, 2, heads=[1])
    out[:200, 1], clean[:200, 1] = 0, 0
    lse[1, :200], clean_lse[1, :200] = 0, 0
    assert torch.equal(out, clean) and torch.equal(lse, clean_lse)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_forward_repeats_and_graph(dev, dtype):
    """The same bits again, on another stream, and from a captured graph that
    is replayed with eager work between."""
    say(f"window forward graph {dtype}")
    qo, ko, q, k, v = (x.to(DEV) for x in inputs(
        dtype, [100, 300], [100, 300], 4, 2, 128, seed=2))
    out = torch.empty_like(q)
    call = lambda o, **kw: sw.window_attention(qo, ko, q, k, v, o, None, 0.1,
                                               64, 4, **kw)
    call(out)
    side = torch.cuda.Stream()
    other = torch.empty_like(q)
    side.wait_stream(torch.cuda.current_stream())
    call(other, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(out, other)
    replayed = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(replayed)
    for i in range(3):
        q.mul_(1.5)
        call(out)
        replayed.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, replayed)


# ---- the backward pass ---------------------------------------------------------

def backward(qo, ko, q, k, v, do, alpha, window, sinks, fill=7.0):
    """Forward and backward as a training step makes them; the gradients."""
    dev = [x.to(DEV) for x in (qo, ko, q, k, v)]
    out = torch.full_like(dev[2], fill)
    lse = torch.full((q.shape[1], q.shape[0]), fill, device=DEV)
    sw.window_attention(*dev, out, lse, alpha, window, sinks)
    grads = [torch.full_like(x, fill) for x in dev[2:]]
    got = sw.window_attention_backward(*dev, out, lse, do.to(DEV), *grads,
                                       alpha, window, sinks)
    torch.cuda.synchronize()
    assert all(a is b for a, b in zip(got, grads))
    return [g.cpu() for g in grads]


def expect_gradients(qo, ko, q, k, v, do, grads, alpha, window, sinks,
                     fill=7.0, heads=None):
    """The gradients of every key head and its query heads, or of `heads`."""
    t = half_step(q.dtype)
    h, hk = q.shape[1], k.shape[1]
    g = h // hk
    qd, kd, vd, dod = (x.double() for x in (q, k, v, do))
    queries = torch.zeros(q.shape[0], dtype=torch.bool)
    keys = torch.zeros(k.shape[0], dtype=torch.bool)
    for i in range(len(qo) - 1):
        a, b, c, e = int(qo[i]), int(qo[i + 1]), int(ko[i]), int(ko[i + 1])
        queries[a:b], keys[c:e] = True, True
        see = visible(b - a, e - c, window, sinks)
        for j in heads or range(hk):
            total = [torch.zeros(e - c, q.shape[2], dtype=torch.float64)
                     for _ in range(4)]
            for x in range(j * g, j * g + g):
                (dq, *kv), (bound, *kv_bound) = gradients(
                    qd[a:b, x], kd[c:e, j], vd[c:e, j], dod[a:b, x], see,
                    alpha, t)
                check(f"dq of sequence {i}, head {x}", grads[0][a:b, x], dq,
                      bound)
                for n, y in enumerate(kv + kv_bound):
                    total[n] += y
            check(f"dk of sequence {i}, head {j}", grads[1][c:e, j], total[0],
                  total[2] + t * total[0].abs())
            check(f"dv of sequence {i}, head {j}", grads[2][c:e, j], total[1],
                  total[3] + t * total[1].abs())
    for x, inside in zip(grads, (queries, keys, keys)):
        assert torch.equal(x[~inside], torch.full_like(x[~inside], fill))


def output_gradient(x, seed=1):
    gen = torch.Generator().manual_seed(seed + 1000)
    return torch.randn(x[2].shape, generator=gen).to(x[2].dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_backward(dev, dtype, case):
    (nq, nk), window, sinks = CASES[case]
    say(f"window backward {dtype} {CASES[case]}")
    x = inputs(dtype, nq, nk, 2, 1, 64, seed=case)
    do = output_gradient(x)
    grads = backward(*x, do, 0.125, window, sinks)
    expect_gradients(*x, do, grads, 0.125, window, sinks)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_backward_many_heads(dev, dtype, case):
    """The same with so many heads that neither rows nor keys are split."""
    (nq, nk), window, sinks = CASES[case]
    say(f"window backward many heads {dtype} {CASES[case]}")
    x = inputs(dtype, nq, nk, 288, 144, 64, seed=case)
    do = output_gradient(x)
    grads = backward(*x, do, 0.125, window, sinks)
    expect_gradients(*x, do, grads, 0.125, window, sinks, heads=[0, 77, 143])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window,sinks", [(300, 0), (300, 3), (64, 40)])
def test_backward_parts(dev, dtype, window, sinks):
    """Few keys and many query heads on each: the tiles of their queries are
    split into parts, which end inside a head's tiles."""
    say(f"window backward parts {dtype} {window} {sinks}")
    x = inputs(dtype, [333, 0, 50], [350, 20, 50], 10, 1, 72, seed=12, lead=3,
               tail=5)
    need = sw.load_library().sw_window_attention_backward_workspace_bytes
    one, many = (need(3, 391, 428, h, 1, 72, window, 0,
                      4 if dtype == "f32" else 2) for h in (1, 10))
    assert many - 10 * one > 2 * 4 * 428 * 2 * 72
    do = output_gradient(x)
    grads = backward(*x, do, 0.2, window, sinks)
    expect_gradients(*x, do, grads, 0.2, window, sinks)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("sinks", [0, 3])
def test_backward_parts_of_the_last_tiles(dev, dtype, sinks):
    """More tiles of keys than run at once: the last ones alone are split,
    from the middle of a head on."""
    say(f"window backward parts of the last tiles {dtype} {sinks}")
    x = inputs(dtype, [1290, 10], [1290, 11], 104, 52, 72, seed=13, lead=2,
               tail=3)
    # 624 tiles, of which 512 are whole, 42 heads' and a part of the next's
    parts, elem = (2, 4) if dtype == "f32" else (3, 2)
    assert sw.load_library().sw_window_attention_backward_workspace_bytes(
        2, 1305, 1306, 104, 52, 72, 300, 0, elem) == 4 * (
            2 * 104 * 1305 + parts * 112 * 128 * 2 * 72)
    do = output_gradient(x)
    grads = backward(*x, do, 0.2, 300, sinks)
    expect_gradients(*x, do, grads, 0.2, 300, sinks, heads=[0, 42, 51])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("h,hk,d", [(1, 1, 8), (3, 3, 24), (6, 2, 64),
                                    (4, 1, 72), (2, 2, 96), (8, 2, 128),
                                    (5, 1, 128), (290, 145, 128)])
def test_backward_heads(dev, dtype, h, hk, d):
    say(f"window backward heads {dtype} {h} {hk} {d}")
    x = inputs(dtype, [70, 131], [90, 131], h, hk, d, seed=d + h)
    do = output_gradient(x)
    grads = backward(*x, do, 1 / math.sqrt(d), 48, 5)
    expect_gradients(*x, do, grads, 1 / math.sqrt(d), 48, 5,
                     heads=None if h < 10 else [0, 100, hk - 1])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window,sinks", [(100, 4), (40, 33), (700, 70)])
def test_backward_sinks_over_chunks(dev, dtype, d, window, sinks):
    """Sinks that queries of several chunks see from past the window, in
    sequences that start inside a chunk and one that has no such queries."""
    say(f"window backward sinks {dtype} {d} {window} {sinks}")
    x = inputs(dtype, [1500, 30, 1100], [1500, 30, 1200], 2, 1, d, seed=d,
               lead=5, tail=9)
    do = output_gradient(x)
    grads = backward(*x, do, 1 / math.sqrt(d), window, sinks)
    expect_gradients(*x, do, grads, 1 / math.sqrt(d), window, sinks)


SHORT_AND_LONG = [20] * 30 + [200] + [5] * 20 + [300, 170]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lengths,window,sinks,blocks,chunks", [
    (SHORT_AND_LONG, 64, 40, 42, 21 * 2),        # by long sequence
    (SHORT_AND_LONG, 64, 2 ** 40, 62, 5 * 42),   # by key and long sequence
    ([500, 0, 400], 10, 2 ** 40, 31, 10 * 29),   # by key and sequence
    ([700, 0, 3, 900], 10, 5, 4, 18),            # by sequence
])
def test_backward_far_sinks(dev, dtype, lengths, window, sinks, blocks, chunks):
    """Sinks that some sequences have past their windows and others have not,
    in each order of the blocks that their sums go to."""
    say(f"window backward far sinks {dtype} {len(lengths)} {window} {sinks}")
    queries = [n - n // 4 if n > 300 else n for n in lengths]
    x = inputs(dtype, queries, lengths, 2, 1, 72, seed=15, lead=3, tail=5)
    elem, tokens = x[2].element_size(), (len(x[2]), len(x[3]))
    need = sw.load_library().sw_window_attention_backward_workspace_bytes
    sizes = [need(len(lengths), *tokens, 2, 1, 72, window, n, elem)
             for n in (0, sinks)]
    assert sizes[1] - sizes[0] == 4 * 32 * 2 * 72 * (2 * blocks + chunks)
    do = output_gradient(x)
    grads = backward(*x, do, 0.2, window, sinks)
    expect_gradients(*x, do, grads, 0.2, window, sinks)


@pytest.mark.parametrize("n,length,h,hk,d,window,sinks", [
    (64, 256, 32, 8, 128, 1024, 2 ** 40),
    (8192, 32, 8, 8, 8, 1024, 64),
])
def test_backward_of_more_sinks_than_keys(dev, n, length, h, hk, d, window,
                                          sinks):
    """Many short sequences, which see all their keys, and sinks that only one
    long sequence has: what the forward pass takes the backward pass takes
    too, in scratch memory of about the gradients' size."""
    say(f"window backward many sinks {n} {length}")
    x = inputs("bf16", [length] * n + [1500], [length] * n + [1500], h, hk, d,
               seed=16)
    need = sw.load_library().sw_window_attention_backward_workspace_bytes
    tokens = n * length + 1500
    one = need(n + 1, tokens, tokens, h, hk, d, window, 0, 2)
    assert need(n + 1, tokens, tokens, h, hk, d, window, sinks, 2) - one <= \
        4 * hk * 2 * d * (2 * tokens + tokens // 4 + 8192)
    do = output_gradient(x)
    got = backward(*x, do, 0.3, window, sinks)
    plain = backward(*x, do, 0.3, window, 0)
    for a, b in zip(got, plain):
        assert torch.equal(a[:n * length], b[:n * length])
    a = n * length
    off = torch.tensor([0, 1500], dtype=torch.int32)
    expect_gradients(off, off, *(y[a:] for y in x[2:]), do[a:],
                     [y[a:] for y in got], 0.3, window, sinks,
                     heads=[0, hk - 1])


@pytest.mark.parametrize("alpha", [-0.3, 0.0])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_backward_alpha(dev, dtype, alpha):
    say(f"window backward alpha {dtype} {alpha}")
    x = inputs(dtype, [200], [200], 2, 1, 64, seed=5)
    do = output_gradient(x)
    grads = backward(*x, do, alpha, 70, 2)
    expect_gradients(*x, do, grads, alpha, 70, 2)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_alpha_below_the_normal_numbers(dev, dtype):
    """An alpha of 5e-39 scales scores of 1e37 as any other would."""
    say(f"window small alpha {dtype}")
    x = list(inputs(dtype, [200, 30], [200, 50], 2, 1, 64, seed=6))
    x[2], x[3] = x[2] * 1e18, x[3] * 1e18
    alpha = 5e-39
    out, lse = forward(*x, alpha, 70, 2)
    expect(*x, out, lse, alpha, 70, 2)
    do = output_gradient(x)
    grads = backward(*x, do, alpha, 70, 2)
    expect_gradients(*x, do, grads, alpha, 70, 2)


def test_backward_against_differences(dev):
    """Directional derivatives of sum(output * do), by central differences in
    fp32: the step 2^-6 leaves a cubic term of about 2^-12 of the derivative,
    and the sum's rounding, about 2^-20 of its terms' size, is divided by the
    step."""
    say("window backward differences")
    x = inputs("f32", [150], [170], 4, 2, 32, seed=8)
    do = output_gradient(x)
    alpha, window, sinks = 0.2, 40, 3
    grads = backward(*x, do, alpha, window, sinks)
    gen = torch.Generator().manual_seed(77)
    for n in range(3):
        way = torch.randn(x[2 + n].shape, generator=gen)
        way /= way.norm()
        step = 2.0 ** -6
        sides = []
        for sign in (1, -1):
            y = list(x)
            y[2 + n] = x[2 + n] + sign * step * way
            out, _ = forward(*y, alpha, window, sinks)
            sides.append((out.double() * do.double()).sum())
        slope = (sides[0] - sides[1]) / (2 * step)
        want = (grads[n].double() * way.double()).sum()
        size = grads[n].double().norm()
        assert abs(slope - want) <= 2.0 ** -10 * size


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_backward_strides(dev, dtype):
    """Gradients into the slices of a projection's gradient, of operands that
    are slices too, from a broadcast output gradient."""
    say(f"window backward strides {dtype}")
    gen = torch.Generator().manual_seed(11)
    t, h, d = 150, 4, 64
    packed = torch.randn(t, 3 * h, d, generator=gen).to(DTYPES[dtype]).to(DEV)
    q, k, v = packed[:, :h], packed[:, h:2 * h], packed[:, 2 * h:]
    do = torch.randn(t, 1, d, generator=gen).to(DTYPES[dtype]).to(DEV)
    do = do.expand(t, h, d)
    off = offsets([t]).to(DEV)
    out = torch.empty(h, t, d, dtype=q.dtype, device=DEV).transpose(0, 1)
    lse = torch.empty(h, t, device=DEV)
    sw.window_attention(off, off, q, k, v, out, lse, 0.125, 40, 3)
    full = torch.full_like(packed, 7.0)
    sw.window_attention_backward(
        off, off, q, k, v, out, lse, do, full[:, :h], full[:, h:2 * h],
        full[:, 2 * h:], 0.125, 40, 3)
    dense = [x.contiguous() for x in (q, k, v, out)]
    plain = [torch.empty_like(x) for x in dense[:3]]
    sw.window_attention_backward(off, off, *dense, lse, do.contiguous(),
                                 *plain, 0.125, 40, 3)
    assert torch.equal(full, torch.cat(plain, 1))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("what", ["query", "key", "value", "do"])
@pytest.mark.parametrize("heads", [1, 288])
def test_backward_keeps_what_is_masked_apart(dev, dtype, bad, what, heads):
    """An infinity or NaN at one token reaches the gradients of the tokens
    that it sees or that see it, and of those alone that share a query with
    them; the rest are those of clean operands."""
    say(f"window backward {bad} in {what} {dtype} {heads}")
    qo, ko, q, k, v = inputs(dtype, [260], [260], heads, heads, 64, seed=4)
    do = output_gradient((qo, ko, q, k, v))
    window, sinks, at = 40, 2, 101
    clean = backward(qo, ko, q, k, v, do, 0.125, window, sinks)
    y = {"query": q.clone(), "key": k.clone(), "value": v.clone(),
         "do": do.clone()}
    y[what][at, 0, 3] = bad
    got = backward(qo, ko, y["query"], y["key"], y["value"], y["do"], 0.125,
                   window, sinks)
    see = visible(260, 260, window, sinks)
    rows = torch.zeros(260, dtype=torch.bool)
    if what in ("query", "do"):
        rows[at] = True
    else:
        rows = see[:, at].clone()
    cols = see[rows].any(0)
    for n, (x, c) in enumerate(zip(got, clean)):
        assert torch.equal(x[:, 1:], c[:, 1:])
        free = ~rows if n == 0 else ~cols
        x, c = x[free, 0].float(), c[free, 0].float()
        assert torch.isfinite(x).all()
        # (a repeated pass may add up in another order)
        assert (x - c).abs().max() <= 8 * half_step(q.dtype) * c.abs().max()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_training_step_repeats_and_graphs(dev, dtype):
    """Forward and backward together: the same bits again, from a given
    workspace, on another stream, and from two captured graphs replayed in
    turn with eager work between."""
    say(f"window training step graph {dtype}")
    x = inputs(dtype, [100, 1300], [100, 1300], 4, 2, 128, seed=2)
    qo, ko, q, k, v = (y.to(DEV) for y in x)
    do = output_gradient(x).to(DEV)

    def buffers():
        return [torch.empty_like(q), torch.empty(4, 1400, device=DEV),
                torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)]

    def step(b, stream=None, **kw):
        sw.window_attention(qo, ko, q, k, v, b[0], b[1], 0.1, 64, 4,
                            stream=stream)
        sw.window_attention_backward(qo, ko, q, k, v, b[0], b[1], do, *b[2:],
                                     0.1, 64, 4, stream=stream, **kw)
    want, other = buffers(), buffers()
    step(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    step(other, stream=side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    need = sw.load_library().sw_window_attention_backward_workspace_bytes(
        2, 1400, 1400, 4, 2, 128, 64, 4, q.element_size())
    step(other, workspace=torch.full((need,), 255, dtype=torch.uint8,
                                     device=DEV))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graphs, held = [], []
    for _ in range(2):
        held.append(buffers())
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            step(held[-1])
    for i in range(3):
        q.mul_(1.25)
        step(want)
        for b in held:
            for y in b:
                y.zero_()
        graphs[i % 2].replay()
        graphs[1 - i % 2].replay()
        torch.cuda.synchronize()
        for b in held:
            assert all(torch.equal(a, c) for a, c in zip(want, b))


def test_backward_refuses_a_short_workspace(dev):
    x = inputs("f32", [10], [10], 1, 1, 64)
    qo, ko, q, k, v = (y.to(DEV) for y in x)
    lse = torch.zeros(1, 10, device=DEV)
    g = [torch.zeros_like(q) for _ in range(3)]
    with pytest.raises(sw.ShapeError, match="workspace must hold"):
        sw.window_attention_backward(
            qo, ko, q, k, v, q, lse, q, *g, 1.0, 4, 1,
            workspace=torch.zeros(16, dtype=torch.uint8, device=DEV))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_nothing_on_one_side(dev, dtype):
    """No queries at all: keys' gradients of zero.  No keys: zeros and -inf.
    No sequences: nothing is written."""
    say(f"window empty sides {dtype}")
    x = inputs(dtype, [0, 0], [5, 40], 2, 1, 64)
    for window, sinks in ((10, 3), (100, 0)):
        grads = backward(*x, torch.empty_like(x[2]), 0.1, window, sinks)
        assert all((g == 0).all() for g in grads)
    x = inputs(dtype, [5, 40], [0, 0], 2, 1, 64)
    out, lse = forward(*x, 0.1, 10, 3)
    assert (out == 0).all() and (lse == -math.inf).all()
    grads = backward(*x, output_gradient(x), 0.1, 10, 3)
    assert (grads[0] == 0).all()
    x = inputs(dtype, [5], [5], 2, 1, 64)
    none = torch.zeros(1, dtype=torch.int32)
    out, lse = forward(none, none, *x[2:], 0.1, 10, 3)
    assert (out == 7).all() and (lse == 7).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_offsets_outside_the_operands(dev, dtype):
    """Offsets that lead outside are clamped: sequences in place keep their
    results, and nothing outside the operands is touched."""
    say(f"window bad offsets {dtype}")
    x = inputs(dtype, [300, 200], [300, 200], 2, 1, 64, seed=3)
    do = output_gradient(x)
    good = backward(*x, do, 0.125, 64, 4)
    bad = torch.tensor([0, 300, 2 ** 31 - 1], dtype=torch.int32)
    got = backward(bad, bad, *x[2:], do, 0.125, 64, 4)
    assert all(torch.equal(a, b) for a, b in zip(good, got))
    for bad in ([-1000, 300, 500], [400, 100, 600], [-2 ** 31, 2 ** 31 - 1, 0]):
        bad = torch.tensor(bad, dtype=torch.int32)
        # rows of one projection, so that neighbours show what is written
        wide = torch.full((500, 6, 64), 7.0, dtype=x[2].dtype, device=DEV)
        wide[:, :2] = x[2].to(DEV)
        off = bad.to(DEV)
        lse = torch.full((2, 500), 7.0, device=DEV)
        k, v = x[3].to(DEV), x[4].to(DEV)
        sw.window_attention(off, off, wide[:, :2], k, v, wide[:, 2:4], lse,
                            0.125, 64, 4)
        g = torch.full((500, 5, 64), 7.0, dtype=x[2].dtype, device=DEV)
        sw.window_attention_backward(off, off, wide[:, :2], k, v,
                                     wide[:, 2:4], lse, do.to(DEV), g[:, :2],
                                     g[:, 2:3], g[:, 3:4], 0.125, 64, 4)
        torch.cuda.synchronize()
        assert (wide[:, 4:] == 7).all() and (g[:, 4:] == 7).all()
