"""Attention of single queries against caches, and over a shared prefix, on
the GPU against float64, element by element within bounds that the arithmetic
gives (tests/_window_check.py)."""
import math
import threading

import pytest
import torch

import sparsewavecomp_amd as sw
from _window_check import check, half_step, softmax
from gpu_util import DEV, say

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def make(dtype, lengths, page, h, hk, d, seed=0, prefix=None, spare=2,
         capacity=None):
    """CPU operands: queries, the sequences' keys and values, and a cache that
    holds them, in pages of a random order with NaN in every row that holds no
    key."""
    gen = torch.Generator().manual_seed(seed)
    t = DTYPES[dtype]
    n = len(lengths)
    values = lambda *s: torch.randn(*s, generator=gen).to(t)
    x = {"query": values(n, h, d),
         "keys": [values(m, hk, d) for m in lengths],
         "values": [values(m, hk, d) for m in lengths],
         "lengths": torch.tensor(lengths, dtype=torch.int32)}
    if page:
        need = [-(-m // page) for m in lengths]
        order = torch.randperm(sum(need) + spare, generator=gen)
        width = max([1] + need)
        table = torch.full((n, width), -7, dtype=torch.int32)
        at = 0
        for i, m in enumerate(need):
            table[i, :m] = order[at:at + m].to(torch.int32)
            at += m
        shape = (sum(need) + spare, page, hk, d)
    else:
        table, shape = None, (n, capacity or max([1] + lengths), hk, d)
    x["table"] = table
    for name in ("key", "value"):
        cache = torch.full(shape, math.nan, dtype=t)
        for i, m in enumerate(lengths):
            for j in range(m):
                if page:
                    cache[table[i, j // page], j % page] = x[name + "s"][i][j]
                else:
                    cache[i, j] = x[name + "s"][i][j]
        x[name + "_cache"] = cache
    if prefix is not None:
        x["prefix_key"] = values(prefix, hk, d)
        x["prefix_value"] = values(prefix, hk, d)
    return x


def on_gpu(x, *names):
    return [None if x[n] is None else x[n].to(DEV) for n in names]


def decode(x, alpha, window, sinks, fill=7.0, **kw):
    a = on_gpu(x, "lengths", "table", "query", "key_cache", "value_cache")
    out = torch.full_like(a[2], fill)
    got = sw.window_attention_decode(*a, out, alpha, window, sinks, **kw)
    torch.cuda.synchronize()
    assert got is out
    return out.cpu()


def prefixed(x, alpha, fill=7.0, **kw):
    a = on_gpu(x, "lengths", "table", "query", "prefix_key", "prefix_value",
               "key_cache", "value_cache")
    out = torch.full_like(a[2], fill)
    got = sw.shared_prefix_attention(*a, out, alpha, **kw)
    torch.cuda.synchronize()
    assert got is out
    return out.cpu()


def expect(x, out, alpha, window=None, sinks=0, hidden=()):
    """`hidden`: (sequence, key) pairs that are not there."""
    t = half_step(out.dtype)
    g = out.shape[1] // x["key_cache"].shape[2]
    for i, n in enumerate(x["lengths"].tolist()):
        j = torch.arange(n)
        see = torch.ones(n, dtype=torch.bool) if window is None else \
            (j >= n - window) | (j < sinks)
        for s, at in hidden:
            if s == i:
                see[at] = False
        for h in range(out.shape[1]):
            k = x["keys"][i][see, h // g].double()
            v = x["values"][i][see, h // g].double()
            if window is None:
                k = torch.cat([x["prefix_key"][:, h // g].double(), k])
                v = torch.cat([x["prefix_value"][:, h // g].double(), v])
            o, bound, *_ = softmax(x["query"][i, h:h + 1].double(), k, v,
                                   torch.ones(1, len(k), dtype=torch.bool),
                                   alpha, t)
            check(f"sequence {i}, head {h}", out[i, h:h + 1], o, bound)


# lengths, page (0: one run of memory), window, sinks: lengths of zero and one;
# chunks' and tiles' borders from both sides; pages that end inside a tile, of
# one key, of an odd number; sinks apart from the window, across a page's end
# and as many as the keys
CASES = [
    ([1], 0, 1, 0),
    ([0], 0, 5, 0),
    ([0, 1, 0], 16, 100, 4),
    ([31, 32, 33, 127, 128, 129], 16, 1000, 0),
    ([255, 256, 257, 300], 0, 10 ** 12, 0),
    ([300, 40, 7], 24, 64, 5),
    ([300, 40, 7], 1, 33, 3),
    ([520, 513, 512], 64, 256, 4),
    ([520, 100], 100, 130, 128),
    ([2000, 3], 256, 1990, 9),
    ([2000, 1500], 0, 700, 900),
    ([40] * 70, 16, 30, 4),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_decode(dev, dtype, case):
    lengths, page, window, sinks = CASES[case]
    say(f"decode {dtype} {CASES[case]}")
    x = make(dtype, lengths, page, 4, 2, 64, seed=case)
    expect(x, decode(x, 0.125, window, sinks), 0.125, window, sinks)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("h,hk,d", [(1, 1, 8), (3, 3, 24), (17, 1, 72),
                                    (32, 2, 96), (40, 1, 128), (8, 8, 128)])
def test_decode_heads(dev, dtype, h, hk, d):
    """Also more query heads on one key head than a part has rows."""
    say(f"decode heads {dtype} {h} {hk} {d}")
    for lengths, page in (([70, 5], 16), ([1500], 0)):
        x = make(dtype, lengths, page, h, hk, d, seed=d + h)
        expect(x, decode(x, 1 / math.sqrt(d), 1200, 5), 1 / math.sqrt(d),
               1200, 5)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_long(dev, dtype):
    """Many parts to join, and a capacity far past the lengths."""
    say(f"decode long {dtype}")
    x = make(dtype, [20000, 300, 9000], 0, 2, 1, 64, seed=1, capacity=25000)
    expect(x, decode(x, 0.125, 1 << 20, 0), 0.125, 1 << 20, 0)
    expect(x, decode(x, 0.125, 15000, 7), 0.125, 15000, 7)


@pytest.mark.parametrize("alpha", [-0.3, 0.0, 4.0])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_alpha(dev, dtype, alpha):
    say(f"decode alpha {dtype} {alpha}")
    x = make(dtype, [200, 700], 32, 2, 1, 64, seed=5)
    expect(x, decode(x, alpha, 500, 2), alpha, 500, 2)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [2, 70])
def test_alpha_below_the_normal_numbers(dev, dtype, n):
    """An alpha of 5e-39 scales scores of 1e37 as any other would."""
    say(f"decode small alpha {dtype} {n}")
    x = make(dtype, [40, 700] + [9] * (n - 2), 32, 2, 1, 64, seed=5, prefix=90)
    x["query"] *= 1e18
    for name in ("key_cache", "prefix_key"):
        x[name] *= 1e18
    x["keys"] = [k * 1e18 for k in x["keys"]]
    expect(x, decode(x, 5e-39, 500, 2), 5e-39, 500, 2)
    expect(x, prefixed(x, 5e-39), 5e-39)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bad", [-1, 10 ** 6, -2 ** 31])
def test_decode_pages_outside_the_cache(dev, dtype, bad):
    """Their keys are not there; a sequence without any other gets zeros."""
    say(f"decode bad page {dtype} {bad}")
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
@pytest.mark.parametrize("length", [30, 900])
def test_decode_scores_of_minus_infinity(dev, dtype, length):
    """Keys that are seen and all score -inf give NaN, as the softmax does; one
    other key takes all."""
    say(f"decode -inf scores {dtype} {length}")
    x = make(dtype, [length], 0, 1, 1, 64, seed=1)
    x["query"][:] = 1.0
    x["key_cache"][0, :, 0, 0] = -math.inf
    got = decode(x, 0.125, 10 ** 6, 0)
    assert torch.isnan(got).all()
    x["key_cache"][0, length // 2, 0, 0] = 0.0
    got = decode(x, 0.125, 10 ** 6, 0)
    assert torch.equal(got[0, 0], x["value_cache"][0, length // 2, 0])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_lengths_past_the_table(dev, dtype):
    say(f"decode long lengths {dtype}")
    x = make(dtype, [96, 32], 16, 2, 1, 64, seed=2)
    out = decode(x, 0.125, 50, 2)
    x["lengths"] = torch.tensor([2 ** 31 - 1, 32], dtype=torch.int32)
    assert torch.equal(decode(x, 0.125, 50, 2), out)
    x["lengths"] = torch.tensor([-5, 32], dtype=torch.int32)
    got = decode(x, 0.125, 50, 2)
    assert torch.equal(got[0], torch.zeros_like(got[0]))
    assert torch.equal(got[1], out[1])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_strides(dev, dtype):
    """Heads before slots, keys and values in one cache, slices of queries."""
    say(f"decode strides {dtype}")
    x = make(dtype, [100, 33], 16, 4, 2, 64, seed=6)
    want = decode(x, 0.125, 60, 3)
    both = torch.stack([x["key_cache"], x["value_cache"]], 1)  # p, 2, s, h, d
    both = both.transpose(2, 3).contiguous().to(DEV)           # p, 2, h, s, d
    k, v = (both[:, i].transpose(1, 2) for i in range(2))
    wide = torch.zeros(2, 9, 64, dtype=k.dtype, device=DEV)
    wide[:, 2:6] = x["query"].to(DEV)
    out = torch.full((4, 2, 64), 7.0, dtype=k.dtype, device=DEV)
    sw.window_attention_decode(x["lengths"].to(DEV), x["table"].to(DEV),
                               wide[:, 2:6], k, v, out.transpose(0, 1), 0.125,
                               60, 3)
    assert torch.equal(out.transpose(0, 1).cpu(), want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_one_row_of_buffers_with_far_heads(dev, dtype):
    """A batch of one whose query and output are a token of buffers with heads
    before tokens, pages of one key and a prefix of one key laid out alike."""
    say(f"one row, far heads {dtype}")
    x = make(dtype, [5], 1, 4, 2, 64, seed=7, prefix=1)
    t, far = DTYPES[dtype], (1 << 23) // 64 + 10

    def apart(y):
        """y [1, heads, d] as a token of a buffer [heads, far, d]."""
        buf = torch.full((y.shape[1], far, 64), 7.0, dtype=t, device=DEV)
        buf[:, 100:101] = y.transpose(0, 1).to(DEV)
        return buf, buf[:, 100:101].transpose(0, 1)
    _, query = apart(x["query"])
    lengths, table = on_gpu(x, "lengths", "table")
    caches = on_gpu(x, "key_cache", "value_cache")
    # (pages, 1, heads, d) of (heads, pages, d)
    caches = [c.transpose(0, 2).contiguous().transpose(0, 2) for c in caches]
    buf, out = apart(torch.full((1, 4, 64), 7.0))
    sw.window_attention_decode(lengths, table, query, *caches, out, 0.125, 3, 1)
    assert torch.equal(out.cpu(), decode(x, 0.125, 3, 1))
    assert (buf[:, :100] == 7).all() and (buf[:, 101:] == 7).all()
    _, pk = apart(x["prefix_key"])
    _, pv = apart(x["prefix_value"])
    sw.shared_prefix_attention(lengths, table, query, pk, pv, *caches, out,
                               0.125)
    assert torch.equal(out.cpu(), prefixed(x, 0.125))
    # a prompt of one token, and its gradients into such buffers
    off = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    want = torch.empty(1, 4, 64, dtype=t, device=DEV)
    lse = torch.empty(4, 1, device=DEV)
    q, k, v = on_gpu(x, "query", "prefix_key", "prefix_value")
    sw.window_attention(off, off, q, k, v, want, None, 0.125, 3, 1)
    sw.window_attention(off, off, query, pk, pv, out, lse, 0.125, 3, 1)
    assert torch.equal(out, want)
    plain = [torch.empty_like(y) for y in (q, k, v)]
    sw.window_attention_backward(off, off, q, k, v, want, lse, q, *plain,
                                 0.125, 3, 1)
    grads = [apart(torch.zeros(y.shape))[1] for y in (q, k, v)]
    sw.window_attention_backward(off, off, query, pk, pv, out, lse, query,
                                 *grads, 0.125, 3, 1)
    assert all(torch.equal(a, b) for a, b in zip(grads, plain))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_past_four_gib(dev, dtype):
    """Rows of a cache whose byte offsets pass 2^32, by a page stride over
    memory that no key lies in."""
    say(f"decode past 4 GiB {dtype}")
    x = make(dtype, [40, 50, 45], 16, 2, 1, 64, seed=3)
    pages = x["key_cache"].shape[0]
    far = (5 << 30) // (pages - 1) // x["key_cache"].element_size() // 8 * 8
    want = decode(x, 0.125, 30, 2)
    caches = []
    for name in ("key_cache", "value_cache"):
        store = torch.empty(far * (pages - 1) + 16 * 64, device=DEV,
                            dtype=x[name].dtype)
        cache = store.as_strided((pages, 16, 1, 64), (far, 64, 64, 1))
        cache.copy_(x[name].to(DEV))
        caches.append(cache)
    out = torch.empty_like(x["query"], device=DEV)
    sw.window_attention_decode(*on_gpu(x, "lengths", "table", "query"),
                               *caches, out, 0.125, 30, 2)
    assert torch.equal(out.cpu(), want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_decode_keeps_what_is_masked_apart(dev, dtype, bad):
    say(f"decode {bad} {dtype}")
    x = make(dtype, [300, 310], 16, 2, 2, 64, seed=4)
    window, sinks = 40, 5
    want = decode(x, 0.125, window, sinks)
    page, slot = x["table"][0, 6], 3  # key 99 of sequence 0: hidden
    for name in ("key_cache", "value_cache"):
        x[name][page, slot] = bad
    assert torch.equal(decode(x, 0.125, window, sinks), want)
    page = x["table"][0, 18]
    x["value_cache"][page, slot, 0, 7] = bad  # key 291: seen
    got = decode(x, 0.125, window, sinks)
    hit = got[0, 0, 7]
    assert torch.isnan(hit) if math.isnan(bad) else hit == bad
    got[0, 0, 7] = want[0, 0, 7]
    assert torch.equal(got, want)


@pytest.mark.parametrize("lengths,page,window", [
    ([300, 40], 0, 500), ([2000, 1500, 0, 1], 64, 1700)])
@pytest.mark.parametrize("prefix", [None, 200])
def test_bf16_probabilities_keep_fifteen_bits(dev, lengths, page, window,
                                              prefix):
    """A probability goes into its product as its upper eight bits and as what
    they leave off, less than 2^-7 of it and rounded by at most 2^-8 of that:
    off by 2^-15 of itself.  So an output is off by half a step of its own and
    by 2^-15 of the sum of its terms' sizes, however much of them cancels."""
    say(f"bf16 probabilities {lengths} {page} {prefix}")
    t = half_step(torch.bfloat16)
    x = make("bf16", lengths, page, 4, 2, 64, seed=17, prefix=prefix)
    out = decode(x, 0.125, window, 0) if prefix is None else prefixed(x, 0.125)
    for i, n in enumerate(lengths):
        for h in range(4):
            k, v = (x[m][i][:, h // 2].double() for m in ("keys", "values"))
            if prefix is None:
                k, v = k[-window:], v[-window:]
            else:
                k, v = (torch.cat([x[m][:, h // 2].double(), y]) for m, y in (
                    ("prefix_key", k), ("prefix_value", v)))
            see = torch.ones(1, len(k), dtype=torch.bool)
            o, bound, p, *_ = softmax(x["query"][i, h:h + 1].double(), k, v,
                                      see, 0.125, t)
            bound += (2.0 ** -15 - t) * (p @ v.abs())
            check(f"sequence {i}, head {h}", out[i, h:h + 1], o, bound)


def large(y, size, seed):
    """Values of [.., heads, d] of one sign a column, between size / 2 and
    size."""
    gen = torch.Generator().manual_seed(seed)
    v = (0.5 + torch.rand(y.shape, generator=gen) / 2) * size
    v[..., y.shape[-1] // 2:] *= -1
    return v.to(y.dtype)


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
    say(f"decode large values {dtype} {d} {alpha} {size}")
    for lengths, window, sinks in (([128, 130], 200, 0), ([2000, 300], 1900, 4),
                                   ([9000, 8000], 10 ** 6, 0)):
        x = make(dtype, lengths, 0, 4, 2, d, seed=31)
        clean = decode(x, alpha, window, sinks)
        v = large(x["values"][0], size, 32)
        x["values"][0] = v
        x["value_cache"][0, :lengths[0]] = v
        got = decode(x, alpha, window, sinks)
        assert torch.isfinite(got).all()
        expect(x, got, alpha, window, sinks)
        assert torch.equal(got[1], clean[1])


# ---- a shared prefix -------------------------------------------------------------

# lengths, page, prefix, heads, key heads, d: one sequence; no keys of its own;
# an empty prefix; query rows on both sides of the kernels' rule and of their
# tiles; prefixes that end inside a tile and take several parts
PREFIX_CASES = [
    ([5], 0, 1, 1, 1, 64),
    ([0], 16, 100, 2, 1, 64),
    ([0, 3, 50], 16, 0, 4, 2, 64),
    ([0, 0], 16, 0, 4, 2, 64),
    ([10, 0, 33], 16, 63, 4, 2, 64),
    ([7] * 16, 0, 257, 8, 2, 96),
    ([7] * 17, 16, 700, 4, 1, 64),
    ([20] * 33, 24, 64, 4, 1, 128),
    ([1, 300, 20], 0, 1300, 96, 2, 128),
    ([1, 2] * 40, 16, 2100, 8, 2, 40),
    ([3] * 65, 16, 129, 2, 1, 8),
    ([1000, 2000], 256, 3000, 4, 2, 64),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(PREFIX_CASES)))
def test_prefix(dev, dtype, case):
    lengths, page, prefix, h, hk, d = PREFIX_CASES[case]
    say(f"prefix {dtype} {PREFIX_CASES[case]}")
    x = make(dtype, lengths, page, h, hk, d, seed=case, prefix=prefix)
    expect(x, prefixed(x, 1 / math.sqrt(d)), 1 / math.sqrt(d))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("alpha", [-0.3, 0.0])
def test_prefix_alpha(dev, dtype, alpha):
    say(f"prefix alpha {dtype} {alpha}")
    for n in (3, 40):
        x = make(dtype, [9] * n, 16, 2, 1, 64, seed=n, prefix=200)
        expect(x, prefixed(x, alpha), alpha)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("alpha,size", LARGE)
@pytest.mark.parametrize("n,d", [(3, 64), (40, 64), (3, 128), (40, 128)])
def test_prefix_of_large_values(dev, dtype, alpha, size, n, d):
    say(f"prefix large values {dtype} {alpha} {size} {n} {d}")
    x = make(dtype, [9] * n, 16, 4, 2, d, seed=n, prefix=1000)
    x["prefix_value"] = large(x["prefix_value"], size, 33)
    got = prefixed(x, alpha)
    assert torch.isfinite(got).all()
    expect(x, got, alpha)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prefix_strides(dev, dtype):
    say(f"prefix strides {dtype}")
    for n in (3, 40):
        x = make(dtype, [9] * n, 16, 4, 2, 64, seed=n, prefix=200)
        want = prefixed(x, 0.125)
        x["prefix_key"] = x["prefix_key"].transpose(0, 1).contiguous(
            ).transpose(0, 1)
        both = torch.cat([x["prefix_key"], x["prefix_value"]], 1).to(DEV)
        a = on_gpu(x, "lengths", "table", "query")
        out = torch.empty_like(a[2])
        sw.shared_prefix_attention(*a, both[:, :2], both[:, 2:],
                                   *on_gpu(x, "key_cache", "value_cache"),
                                   out, 0.125)
        assert torch.equal(out.cpu(), want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [3, 40])
def test_prefix_is_a_cache_of_its_own_keys(dev, dtype, n):
    """The prefix and the suffix as one cache give the same to rounding."""
    say(f"prefix against decode {dtype} {n}")
    x = make(dtype, [9] * n, 16, 2, 1, 64, seed=n, prefix=100)
    keys = [torch.cat([x["prefix_key"], k]) for k in x["keys"]]
    values = [torch.cat([x["prefix_value"], v]) for v in x["values"]]
    y = dict(x, keys=keys, values=values, table=None,
             lengths=torch.full((n,), 109, dtype=torch.int32),
             key_cache=torch.stack(keys), value_cache=torch.stack(values))
    expect(y, prefixed(x, 0.125), 0.125, 10 ** 6)
    expect(y, decode(y, 0.125, 10 ** 6, 0), 0.125, 10 ** 6)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_steps_repeat_and_graph(dev, dtype):
    """A token step as a server makes it, window layers and a shared prefix:
    the same bits again, on another stream, from a given workspace, and from
    two captured graphs replayed in turn with lengths that grow."""
    say(f"cache step graph {dtype}")
    x = make(dtype, [600] * 40, 16, 4, 2, 128, seed=1, prefix=1500)
    a = on_gpu(x, "lengths", "table", "query", "prefix_key", "prefix_value",
               "key_cache", "value_cache")
    a[0] -= 10

    def buffers():
        return [torch.empty_like(a[2]) for _ in range(2)]

    def step(b, workspaces=(None, None), **kw):
        sw.window_attention_decode(a[0], a[1], a[2], a[5], a[6], b[0], 0.1,
                                   590, 4, workspace=workspaces[0], **kw)
        sw.shared_prefix_attention(*a, b[1], 0.1, workspace=workspaces[1],
                                   **kw)
    want, other = buffers(), buffers()
    step(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    step(other, stream=side)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, other))
    lib = sw.load_library()
    width = a[1].shape[1]
    sizes = (lib.sw_window_attention_decode_workspace_bytes(
        40, 16, width, 4, 2, 128, 590, 4),
        lib.sw_shared_prefix_attention_workspace_bytes(
            40, 1500, 16, width, 4, 2, 128))
    assert sizes[0] > 0 and sizes[1] > 0
    step(other, [torch.full((n,), 255, dtype=torch.uint8, device=DEV)
                 for n in sizes])
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, other))
    graphs, held = [], []
    for _ in range(2):
        held.append(buffers())
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            step(held[-1])
    for i in range(4):
        a[0] += 1
        step(want)
        for b in held:
            for y in b:
                y.zero_()
        graphs[i % 2].replay()
        graphs[1 - i % 2].replay()
        torch.cuda.synchronize()
        for b in held:
            assert all(torch.equal(p, q) for p, q in zip(want, b))


def test_decode_goes_on_from_a_prompt(dev):
    """Window attention of a prompt, then tokens one by one against the cache
    of its keys: each step gives what the prompt pass gives at its place."""
    say("decode after prompt")
    gen = torch.Generator().manual_seed(21)
    t, h, hk, d, window, sinks = 180, 4, 2, 64, 50, 3
    q = torch.randn(t, h, d, generator=gen).to(DEV)
    k = torch.randn(t, hk, d, generator=gen).to(DEV)
    v = torch.randn(t, hk, d, generator=gen).to(DEV)
    off = torch.tensor([0, t], dtype=torch.int32, device=DEV)
    whole = torch.empty_like(q)
    sw.window_attention(off, off, q, k, v, whole, None, 0.125, window, sinks)
    table = torch.arange(8, -1, -1, dtype=torch.int32, device=DEV)[None]
    pages = [torch.zeros(9, 20, hk, d, device=DEV) for _ in range(2)]
    out = torch.empty(1, h, d, device=DEV)
    for n in range(1, t + 1):
        page, slot = 8 - (n - 1) // 20, (n - 1) % 20
        pages[0][page, slot], pages[1][page, slot] = k[n - 1], v[n - 1]
        if n % 13 and n < 170:
            continue
        sw.window_attention_decode(
            torch.tensor([n], dtype=torch.int32, device=DEV), table,
            q[n - 1:n], *pages, out, 0.125, window, sinks)
        # both within fp32 sums of the same at most 53 terms of size 1
        assert (out[0] - whole[n - 1]).abs().max() <= 256 * 2.0 ** -24 * 4


def test_scratch_while_another_thread_captures(dev):
    """A backward pass and a step take their scratch memory also when the
    allocator has to ask the driver for it while another thread captures a
    graph, and leave that capture alone."""
    gen = torch.Generator(device=DEV).manual_seed(4)
    t, h, hk, d = 3000, 4, 2, 128
    off = torch.tensor([0, t], dtype=torch.int32, device=DEV)
    q, go = (torch.randn(t, h, d, generator=gen, device=DEV) for _ in "qo")
    k, v = (torch.randn(t, hk, d, generator=gen, device=DEV) for _ in "kv")
    lse = torch.empty(h, t, device=DEV)
    out = sw.window_attention(off, off, q, k, v, torch.empty_like(q), lse,
                              0.1, 100, 4)
    n = off[1:]

    def calls(b):
        sw.window_attention_backward(off, off, q, k, v, out, lse, go, *b[:3],
                                     0.1, 100, 4)
        sw.window_attention_decode(n, None, q[:1], k[None], v[None], b[3], 0.1,
                                   2000)
    want, got = ([torch.zeros_like(x) for x in (q, k, v, q[:1])]
                 for _ in "ab")
    lib = sw.load_library()
    assert lib.sw_window_attention_backward_workspace_bytes(
        1, t, t, h, hk, d, 100, 4, 4) > 0
    assert lib.sw_window_attention_decode_workspace_bytes(
        1, t, 1, h, hk, d, 2000, 0) > 0
    say("window attention while another thread captures")
    calls(want)
    a, b = torch.ones(1000, device=DEV), torch.empty(1000, device=DEV)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()  # the next scratch memory is a new allocation
    failed = []

    def other():
        try:
            with torch.cuda.stream(side):
                calls(got)
        except Exception as e:  # noqa: BLE001 (reported below)
            failed.append(e)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        torch.mul(a, 3.0, out=b)
        thread = threading.Thread(target=other)
        thread.start()
        thread.join(30)
    assert not thread.is_alive() and not failed, failed
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    for _ in range(2):
        b.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert bool((b == 3.0).all())


def test_a_stream_that_is_not_torchs(dev):
    """Any object with a stream's handle will do where the caller gives the
    workspace; without one the call is refused."""
    class Handle:
        cuda_stream = torch.cuda.Stream().cuda_stream

    say("window attention on a bare handle")
    gen = torch.Generator(device=DEV).manual_seed(5)
    k, v = (torch.randn(1, 1100, 2, 64, generator=gen, device=DEV)
            for _ in "kv")
    q = torch.randn(1, 4, 64, generator=gen, device=DEV)
    n = torch.tensor([1100], dtype=torch.int32, device=DEV)
    want, got = torch.empty_like(q), torch.zeros_like(q)
    need = sw.load_library().sw_window_attention_decode_workspace_bytes(
        1, 1100, 1, 4, 2, 64, 1000, 4)
    assert need > 0
    space = torch.empty(need, dtype=torch.uint8, device=DEV)
    sw.window_attention_decode(n, None, q, k, v, want, 0.1, 1000, 4)
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="needs a workspace"):
        sw.window_attention_decode(n, None, q, k, v, got, 0.1, 1000, 4,
                                   stream=Handle)
    sw.window_attention_decode(n, None, q, k, v, got, 0.1, 1000, 4,
                               workspace=space, stream=Handle)
    torch.cuda.synchronize()
    assert torch.equal(want, got)
