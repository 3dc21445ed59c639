"""Attention of single queries against a cache of 4-bit codes, on the GPU
against float64, element by element within bounds that the arithmetic gives
(tests/_fp4_check.py)."""
import math
import threading

import pytest
import torch

import sparsewavecomp_amd as sw
from _fp4_check import attend, dequantise, quantise
from _window_check import check
from gpu_util import DEV, say

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def make(dtype, lengths, page, h, hk, d, seed=0, spare=2, capacity=None):
    """CPU operands: queries, the sequences' codes and scales, what they stand
    for, and a cache that holds them in pages of a random order, NaN in every
    row that holds no key."""
    gen = torch.Generator().manual_seed(seed)
    n = len(lengths)
    x = {"query": torch.randn(n, h, d, generator=gen).to(DTYPES[dtype]),
         "lengths": torch.tensor(lengths, dtype=torch.int32)}
    if page:
        need = [-(-m // page) for m in lengths]
        order = torch.randperm(sum(need) + spare, generator=gen)
        table = torch.full((n, max([1] + need)), -7, dtype=torch.int32)
        at = 0
        for i, m in enumerate(need):
            table[i, :m] = order[at:at + m].to(torch.int32)
            at += m
        shape = (sum(need) + spare, page, hk)
    else:
        table, shape = None, (n, capacity or max([1] + lengths), hk)
    x["table"] = table
    for name in ("key", "value"):
        codes = torch.randint(0, 256, (*shape, d // 2), generator=gen,
                              dtype=torch.int32).to(torch.uint8)
        scales = torch.full((*shape, d // 32), 255, dtype=torch.uint8)
        x[name + "_cache"], x[name + "s"] = [codes, scales], []
        for i, m in enumerate(lengths):
            put(x, name, i, torch.randn(m, hk, d, generator=gen))
    return x


def put(x, name, i, rows):
    """Sequence i's keys or values: its first len(rows) places."""
    codes, scales = quantise(rows)
    m = len(rows)
    if len(x[name + "s"]) == i:
        x[name + "s"].append(None)
    x[name + "s"][i] = dequantise(codes, scales)
    to = x[name + "_cache"]
    j = torch.arange(m)
    page, size = torch.full_like(j, i), to[0].shape[1]
    if x["table"] is not None:
        page, j = x["table"][i].long()[j // size], j % size
    to[0][page, j], to[1][page, j] = codes, scales


def head_major(y):
    return y.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)


def operands(x, place=head_major):
    table = None if x["table"] is None else x["table"].to(DEV)
    return [x["lengths"].to(DEV), table, x["query"].to(DEV),
            *(sw.Fp4Rows(*map(place, x[n])) for n in ("key_cache",
                                                      "value_cache"))]


def decode(x, alpha, window, sinks, fill=7.0, place=head_major, **kw):
    a = operands(x, place)
    out = torch.full_like(a[2], fill)
    got = sw.window_attention_decode_fp4(*a, out, alpha, window, sinks, **kw)
    torch.cuda.synchronize()
    assert got is out
    return out.cpu()


def expect(x, out, alpha, window, sinks=0, hidden=()):
    """`hidden`: (sequence, key) pairs that are not there."""
    hk = x["key_cache"][0].shape[2]
    g = out.shape[1] // hk
    for i, n in enumerate(x["lengths"].tolist()):
        j = torch.arange(n)
        see = (j >= n - window) | (j < sinks)
        for s, at in hidden:
            if s == i:
                see[at] = False
        for k in range(hk):
            rows = slice(k * g, k * g + g)
            o, bound = attend(x["query"][i, rows].double(),
                              x["keys"][i][see, k], x["values"][i][see, k],
                              alpha, out.dtype)
            check(f"sequence {i}, key head {k}", out[i, rows], o, bound)


# lengths, page (0: one run of memory), window, sinks: lengths of zero and one;
# chunks' and tiles' borders from both sides; pages that end inside a tile, of
# one key, of an odd number; sinks apart from the window, across a page's end
# and as many as the keys
CASES = [
    ([1], 0, 1, 0),
    ([0], 0, 5, 0),
    ([0, 1, 0], 16, 100, 4),
    ([15, 16, 17, 31, 32, 33, 127, 128, 129], 16, 1000, 0),
    ([255, 256, 257, 300], 0, 10 ** 12, 0),
    ([300, 40, 7], 24, 64, 5),
    ([300, 40, 7], 1, 33, 3),
    ([520, 513, 512], 64, 256, 4),
    ([520, 100], 100, 130, 128),
    ([2000, 3], 256, 1990, 9),
    ([2000, 1500], 0, 700, 900),
    ([40] * 70, 16, 30, 4),
    ([1023, 1024, 1025, 1151, 1153], 48, 4000, 0),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_decode(dev, dtype, d, case):
    lengths, page, window, sinks = CASES[case]
    say(f"fp4 decode {dtype} {d} {CASES[case]}")
    x = make(dtype, lengths, page, 4, 2, d, seed=case)
    expect(x, decode(x, 0.125, window, sinks), 0.125, window, sinks)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("h,hk,d", [
    (1, 1, 32), (3, 3, 96), (17, 1, 64), (32, 2, 96), (40, 1, 128),
    (8, 8, 128), (64, 8, 32), (6, 2, 32)])
def test_decode_heads(dev, dtype, h, hk, d):
    """Also more query heads on one key head than a part has rows."""
    say(f"fp4 decode heads {dtype} {h} {hk} {d}")
    for lengths, page in (([70, 5], 16), ([1500], 0)):
        x = make(dtype, lengths, page, h, hk, d, seed=d + h)
        expect(x, decode(x, 1 / math.sqrt(d), 1200, 5), 1 / math.sqrt(d),
               1200, 5)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_long(dev, dtype):
    """Many parts to join, and a capacity far past the lengths."""
    say(f"fp4 decode long {dtype}")
    x = make(dtype, [20000, 300, 9000], 0, 2, 1, 64, seed=1, capacity=25000)
    expect(x, decode(x, 0.125, 1 << 20, 0), 0.125, 1 << 20, 0)
    expect(x, decode(x, 0.125, 15000, 7), 0.125, 15000, 7)


def ragged(n, most, seed):
    """Lengths from 0 to `most`, a fifth of them 0."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randint(0, most + 1, (n,), generator=gen)
    x[torch.rand(n, generator=gen) < 0.2] = 0
    x[n // 2] = most
    return x.tolist()


# sequences, most keys, page, window, sinks, heads, key heads: more sequences than
# a wave has lanes, none in front or behind; windows and sinks whose tiles overlap;
# shares of less than a sequence and of many; more key heads than workgroups that
# run at once
SHARES = [
    (65, 700, 16, 10 ** 6, 0, 2, 1),
    (150, 900, 16, 600, 40, 4, 2),
    (300, 520, 0, 515, 3, 1, 1),
    (3, 6000, 64, 10 ** 6, 0, 12, 1),
    (7, 3000, 24, 1000, 2000, 20, 1),
    (2, 1500, 16, 10 ** 6, 0, 1100, 1100),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(SHARES)))
def test_shares_of_many_sequences(dev, dtype, case):
    n, most, page, window, sinks, h, hk = SHARES[case]
    say(f"fp4 shares {dtype} {SHARES[case]}")
    lengths = ragged(n, most, case)
    if case == 1:
        lengths[0] = lengths[-1] = 0
    x = make(dtype, lengths, page, h, hk, 32, seed=case, capacity=most)
    expect(x, decode(x, 0.2, window, sinks), 0.2, window, sinks)
    x["lengths"][:] = 0  # nothing is left to share
    got = decode(x, 0.2, window, sinks)
    assert torch.equal(got, torch.zeros_like(got))


# sequences, their most keys, one's, room, heads, key heads: rows joined by a wave
# and by a workgroup, of a part or two and of more than either takes at once, some
# behind the last full workgroup; more sequences than a wave's registers hold
JOINS = [
    (80, 300, 9000, 9100, 16, 2),
    (600, 60, 2500, 2600, 1, 1),
    (600, 300, 2500, 2600, 1, 1),
    (200, 500, 3000, 3000, 2, 1),
    (40, 700, 700, 5000, 17, 1),
    (1, 40000, 40000, 40000, 3, 1),
    (30, 9, 33000, 33000, 18, 1),
    (260, 1000, 1000, 4000, 3, 3),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(JOINS)))
def test_joins(dev, dtype, case):
    n, most, one, room, h, hk = JOINS[case]
    say(f"fp4 joins {dtype} {JOINS[case]}")
    lengths = ragged(n, most, case)
    lengths[n // 2] = one
    x = make(dtype, lengths, 0, h, hk, 32, seed=case, capacity=room)
    expect(x, decode(x, 0.2, 10 ** 6, 0), 0.2, 10 ** 6)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_more_sequences_than_are_shared(dev, dtype):
    """Past 4096 each has a workgroup to itself, whatever room it has."""
    say(f"fp4 4,200 sequences {dtype}")
    lengths = ragged(4200, 40, 5)
    lengths[17] = 800
    x = make(dtype, lengths, 16, 1, 1, 32, seed=7)
    expect(x, decode(x, 0.2, 10 ** 6, 0), 0.2, 10 ** 6, 0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_one_key_comes_back(dev, dtype):
    """One key's output is its value: bf16 its bits.  In fp32 the probability p
    is 2 to what the maximum's own rounding leaves, next to 1; its three parts
    hold it whole, so that the product v p, 1 / p and their product round, and in
    the join of parts as many again and the part's weight twice: 8 u."""
    say(f"fp4 one key {dtype}")
    x = make(dtype, [1, 700], 16, 4, 2, 128, seed=2)
    got = decode(x, 0.3, 1, 0)
    for i, n in enumerate((1, 700)):
        want = x["values"][i][n - 1].repeat_interleave(2, 0)
        if dtype == "bf16":
            assert torch.equal(got[i].double(), want)
        else:
            assert ((got[i].double() - want).abs() <=
                    8 * 2.0 ** -24 * want.abs()).all()


@pytest.mark.parametrize("alpha", [-0.3, 0.0, 4.0])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_alpha(dev, dtype, alpha):
    say(f"fp4 decode alpha {dtype} {alpha}")
    x = make(dtype, [200, 700], 32, 2, 1, 64, seed=5)
    expect(x, decode(x, alpha, 500, 2), alpha, 500, 2)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [2, 70])
def test_alpha_below_the_normal_numbers(dev, dtype, n):
    """An alpha of 5e-39 scales scores of 1e37 as any other would."""
    say(f"fp4 decode small alpha {dtype} {n}")
    lengths = [40, 700] + [9] * (n - 2)
    x = make(dtype, lengths, 32, 2, 1, 64, seed=5)
    x["query"] *= 2.0 ** 60
    for i in range(n):
        put(x, "key", i, x["keys"][i] * 2.0 ** 60)
    expect(x, decode(x, 5e-39, 500, 2), 5e-39, 500, 2)


@pytest.mark.parametrize("spread", [1.0, 30.0])
def test_fp32_queries_lose_nothing(dev, spread):
    """Queries whose 24 bits count: large parts that cancel against small ones
    within a score."""
    say(f"fp4 fp32 queries {spread}")
    x = make("f32", [300, 900], 16, 4, 2, 128, seed=6)
    gen = torch.Generator().manual_seed(1)
    x["query"] *= torch.exp2(
        spread * (torch.rand(x["query"].shape, generator=gen) - 0.5))
    expect(x, decode(x, 0.01, 2000, 0), 0.01, 2000, 0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bad", [-1, 10 ** 6, -2 ** 31])
def test_decode_pages_outside_the_cache(dev, dtype, bad):
    """Their keys are not there; a sequence without any other gets zeros."""
    say(f"fp4 decode bad page {dtype} {bad}")
    x = make(dtype, [100, 600, 40], 16, 4, 2, 64, seed=9)
    x["table"][0, 2] = bad
    x["table"][1, 30:] = bad
    hidden = [(0, j) for j in range(32, 48)] + [
        (1, j) for j in range(480, 600)]
    expect(x, decode(x, 0.125, 300, 50), 0.125, 300, 50, hidden)
    expect(x, decode(x, 0.125, 10 ** 6, 0), 0.125, 10 ** 6, 0, hidden)
    x["table"][:2] = bad
    for window in (50, 10 ** 6):
        got = decode(x, 0.125, window, 0)
        assert torch.equal(got[:2], torch.zeros_like(got[:2]))
        assert (got[2] != 0).any()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_lengths_past_the_table(dev, dtype):
    say(f"fp4 decode long lengths {dtype}")
    x = make(dtype, [96, 32], 16, 2, 1, 64, seed=2)
    out = decode(x, 0.125, 50, 2)
    x["lengths"] = torch.tensor([2 ** 31 - 1, 32], dtype=torch.int32)
    assert torch.equal(decode(x, 0.125, 50, 2), out)
    x["lengths"] = torch.tensor([-5, 32], dtype=torch.int32)
    got = decode(x, 0.125, 50, 2)
    assert torch.equal(got[0], torch.zeros_like(got[0]))
    assert torch.equal(got[1], out[1])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
def test_decode_strides(dev, dtype, d):
    """Rows of heads together, keys and values in one cache, scales that start
    anywhere, slices of queries."""
    say(f"fp4 decode strides {dtype} {d}")
    x = make(dtype, [100, 33], 16, 4, 2, d, seed=6)
    want = decode(x, 0.125, 60, 3)
    assert torch.equal(decode(x, 0.125, 60, 3, place=lambda y: y.to(DEV)), want)
    lengths, table, query, *_ = operands(x)
    codes = torch.stack([x["key_cache"][0], x["value_cache"][0]], 1).to(DEV)
    scales = torch.stack([x["key_cache"][1], x["value_cache"][1]], 3).to(DEV)
    odd = torch.empty(scales.numel() + 3, dtype=torch.uint8, device=DEV)[3:]
    scales = odd.copy_(scales.flatten()).view(scales.shape)
    assert scales.data_ptr() % 2 == 1
    rows = [sw.Fp4Rows(codes[:, i], scales[:, :, :, i]) for i in range(2)]
    wide = torch.zeros(2, 9, d, dtype=query.dtype, device=DEV)
    wide[:, 2:6] = query
    out = torch.full((4, 2, d), 7.0, dtype=query.dtype, device=DEV)
    sw.window_attention_decode_fp4(lengths, table, wide[:, 2:6], *rows,
                                   out.transpose(0, 1), 0.125, 60, 3)
    assert torch.equal(out.transpose(0, 1).cpu(), want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_past_four_gib(dev, dtype):
    """Rows of a cache whose byte offsets pass 2^32, codes and scales, by page
    strides over memory that no key lies in."""
    say(f"fp4 decode past 4 GiB {dtype}")
    x = make(dtype, [40, 50, 45], 16, 2, 1, 64, seed=3)
    pages = x["key_cache"][0].shape[0]
    far = (5 << 30) // (pages - 1) // 16 * 16
    want = decode(x, 0.125, 30, 2)
    rows = []
    for name in ("key_cache", "value_cache"):
        store = torch.empty(far * (pages - 1) + 16 * 34, device=DEV,
                            dtype=torch.uint8)
        codes = store.as_strided((pages, 16, 1, 32), (far, 32, 32, 1))
        scales = store.as_strided((pages, 16, 1, 2), (far, 2, 2, 1), 512)
        codes.copy_(x[name][0].to(DEV))
        scales.copy_(x[name][1].to(DEV))
        rows.append(sw.Fp4Rows(codes, scales))
    lengths, table, query, *_ = operands(x)
    out = torch.empty_like(query)
    sw.window_attention_decode_fp4(lengths, table, query, *rows, out, 0.125,
                                   30, 2)
    assert torch.equal(out.cpu(), want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_keeps_what_is_masked_apart(dev, dtype):
    """A NaN block of a hidden key changes nothing, of a key that is seen its
    head's rows, of a value its block's columns of them."""
    say(f"fp4 decode NaN {dtype}")
    x = make(dtype, [300, 310], 16, 4, 2, 64, seed=4)
    window, sinks = 40, 5
    want = decode(x, 0.125, window, sinks)
    page, slot = x["table"][0, 6], 3  # key 99 of sequence 0: hidden
    for name in ("key_cache", "value_cache"):
        x[name][1][page, slot] = 255
    assert torch.equal(decode(x, 0.125, window, sinks), want)
    page = x["table"][0, 18]  # key 291: seen
    x["value_cache"][1][page, slot, 0, 1] = 255
    got = decode(x, 0.125, window, sinks)
    assert torch.isnan(got[0, :2, 32:]).all()
    got[0, :2, 32:] = want[0, :2, 32:]
    assert torch.equal(got, want)
    x["key_cache"][1][page, slot, 1, 0] = 255
    got = decode(x, 0.125, window, sinks)
    assert torch.isnan(got[0, 2:]).all()
    assert torch.equal(got[1], want[1])
    assert torch.equal(got[0, :2, :32], want[0, :2, :32])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_decode_of_queries_that_are_not_finite(dev, dtype, bad):
    """They give NaN, in their own rows."""
    say(f"fp4 decode query {bad} {dtype}")
    x = make(dtype, [300, 900], 16, 4, 2, 64, seed=8)
    want = decode(x, 0.125, 10 ** 6, 0)
    x["query"][1, 2, 10] = bad
    got = decode(x, 0.125, 10 ** 6, 0)
    assert torch.isnan(got[1, 2]).all()
    got[1, 2] = want[1, 2]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("length", [30, 900])
def test_decode_scores_of_minus_infinity(dev, dtype, length):
    """Keys that are seen and all score -inf (a scale that no write leaves)
    give NaN, as the softmax does; one other key takes all."""
    say(f"fp4 -inf scores {dtype} {length}")
    x = make(dtype, [length], 0, 1, 1, 64, seed=1)
    x["query"][:] = 1.0
    codes, scales = x["key_cache"]
    codes[0, :, 0, :16], scales[0, :, 0, 0] = 0xFF, 254  # -6 times 2^127
    got = decode(x, 0.125, 10 ** 6, 0)
    assert torch.isnan(got).all()
    codes[0, length // 2, 0, :16] = 0
    got = decode(x, 0.125, 10 ** 6, 0)
    assert torch.equal(got[0, 0], x["values"][0][length // 2, 0].to(got.dtype))


# (what one wave, four waves of a part, and many parts add up passes fp32's
# range)
LARGE = [(0.125, 3.0e38), (4.0, 3.0e38), (0.0, 3.0e38), (0.0, 5.0e36),
         (0.0, 1.5e36)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("alpha,size", LARGE)
def test_decode_of_large_values(dev, dtype, d, alpha, size):
    """Values whose weighted mean is finite while a sum of them is not, in one
    sequence; the others keep their bits."""
    say(f"fp4 decode large values {dtype} {d} {alpha} {size}")
    gen = torch.Generator().manual_seed(32)
    for lengths, window, sinks in (([128, 130], 200, 0), ([2000, 300], 1900, 4),
                                   ([9000, 8000], 10 ** 6, 0)):
        x = make(dtype, lengths, 0, 4, 2, d, seed=31)
        clean = decode(x, alpha, window, sinks)
        v = (0.5 + torch.rand(x["values"][0].shape, generator=gen) / 2) * size
        v[..., d // 2:] *= -1
        put(x, "value", 0, v)
        got = decode(x, alpha, window, sinks)
        assert torch.isfinite(got).all()
        expect(x, got, alpha, window, sinks)
        assert torch.equal(got[1], clean[1])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_steps_repeat_and_graph(dev, dtype):
    """The same bits again, on another stream, from a given workspace, and from
    two captured graphs replayed in turn with lengths that grow."""
    say(f"fp4 step graph {dtype}")
    x = make(dtype, [600] * 40, 16, 4, 2, 128, seed=1)
    a = operands(x)
    a[0] -= 10

    def step(out, **kw):
        return sw.window_attention_decode_fp4(*a, out, 0.1, 590, 4, **kw)
    want, other = torch.empty_like(a[2]), torch.empty_like(a[2])
    step(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    step(other, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(want, other)
    need = sw.load_library().sw_window_attention_decode_fp4_workspace_bytes(
        40, 16, a[1].shape[1], 4, 2, 128, 590, 4)
    assert need > 0
    space = torch.full((need,), 255, dtype=torch.uint8, device=DEV)
    step(other.zero_(), workspace=space)
    torch.cuda.synchronize()
    assert torch.equal(want, other)
    with pytest.raises(sw.ShapeError, match="workspace must hold"):
        step(other, workspace=space[:-16])
    graphs, held = [], []
    for _ in range(2):
        held.append(torch.empty_like(a[2]))
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            step(held[-1])
    for i in range(4):
        a[0] += 1
        step(want)
        for y in held:
            y.zero_()
        graphs[i % 2].replay()
        graphs[1 - i % 2].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(want, y) for y in held)


def test_a_stream_that_is_not_torchs(dev):
    """Any object with a stream's handle will do where the caller gives the
    workspace; without one the call is refused."""
    class Handle:
        cuda_stream = torch.cuda.Stream().cuda_stream

    say("fp4 decode on a bare handle")
    x = make("f32", [1100], 0, 4, 2, 64, seed=5)
    a = operands(x)
    want, got = torch.empty_like(a[2]), torch.zeros_like(a[2])
    need = sw.load_library().sw_window_attention_decode_fp4_workspace_bytes(
        1, 1100, 1, 4, 2, 64, 1000, 4)
    assert need > 0
    space = torch.empty(need, dtype=torch.uint8, device=DEV)
    sw.window_attention_decode_fp4(*a, want, 0.1, 1000, 4)
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="needs a workspace"):
        sw.window_attention_decode_fp4(*a, got, 0.1, 1000, 4, stream=Handle)
    sw.window_attention_decode_fp4(*a, got, 0.1, 1000, 4, workspace=space,
                                   stream=Handle)
    torch.cuda.synchronize()
    assert torch.equal(want, got)


def test_scratch_while_another_thread_captures(dev):
    """A step takes its scratch memory also while another thread captures a
    graph, and leaves that capture alone."""
    say("fp4 decode while another thread captures")
    a = operands(make("f32", [3000], 0, 4, 2, 128, seed=4))
    want, got = torch.zeros_like(a[2]), torch.zeros_like(a[2])
    sw.window_attention_decode_fp4(*a, want, 0.1, 2500)
    x, y = torch.ones(1000, device=DEV), torch.empty(1000, device=DEV)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()  # the next scratch memory is a new allocation
    failed = []

    def other():
        try:
            with torch.cuda.stream(side):
                sw.window_attention_decode_fp4(*a, got, 0.1, 2500)
        except Exception as e:  # noqa: BLE001 (reported below)
            failed.append(e)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        torch.mul(x, 3.0, out=y)
        thread = threading.Thread(target=other)
        thread.start()
        thread.join(30)
    assert not thread.is_alive() and not failed, failed
    torch.cuda.synchronize()
    assert torch.equal(want, got)
    for _ in range(2):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert bool((y == 3.0).all())
