"""Writing a cache of 4-bit codes and reading it back, on the GPU, bit for bit
against float64 (tests/_fp4_check.py), and the two together with rotary
positions and attention."""
import math

import pytest
import torch

import sparsewavecomp_amd as sw
from _fp4_check import attend, dequantise, quantise
from _window_check import check, half_step, softmax
from gpu_util import DEV, say

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def empty(pages, page, heads, d, fill=0xA5):
    """A cache on the CPU whose bytes all hold `fill`."""
    return [sw.Fp4Rows(torch.full((pages, page, heads, d // 2), fill,
                                  dtype=torch.uint8),
                       torch.full((pages, page, heads, d // 32), fill,
                                  dtype=torch.uint8)) for _ in "kv"]


def on_gpu(*x):
    return [None if y is None else y.to(DEV) for y in x]


def rows_on_gpu(cache, head_major=True):
    def move(y):
        if head_major:
            return y.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
        return y.to(DEV)
    return [sw.Fp4Rows(*map(move, c)) for c in cache]


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def offsets(counts):
    return i32(0, *torch.tensor(counts).cumsum(0).tolist())


def table_of(lengths, page, gen, spare=2):
    need = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(need) + spare, generator=gen)
    table = torch.full((len(lengths), max([1] + need)), -7, dtype=torch.int32)
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = order[at:at + m].to(torch.int32)
        at += m
    return table, sum(need) + spare


def values(gen, dtype, *shape):
    """Blocks of sizes from 2^-20 to 2^20, some elements on the border between
    two codes."""
    x = torch.randn(*shape, generator=gen)
    x[..., ::5] = torch.round(x[..., ::5] * 4) / 4
    size = torch.randint(-20, 21, (*shape[:-1], shape[-1] // 32),
                         generator=gen).double().exp2().float()
    return (x * size.repeat_interleave(32, -1)).to(DTYPES[dtype])


def written(cache, x, counts, lengths, table):
    """What the write makes of `cache`, place by place."""
    size, token = cache[0].codes.shape[1], 0
    cache = [sw.Fp4Rows(*(y.clone() for y in c)) for c in cache]
    room = size * (1 if table is None else table.shape[1])
    new = [quantise(y) for y in x]
    for i, (m, n) in enumerate(zip(counts, lengths)):
        for r in range(m):
            place = n - m + r
            if 0 <= place < room:
                page, slot = i, place
                if table is not None:
                    page, slot = int(table[i, place // size]), place % size
                if 0 <= page < len(cache[0].codes):
                    for c, y in zip(cache, new):
                        c.codes[page, slot] = y[0][token]
                        c.scales[page, slot] = y[1][token]
            token += 1
    return cache


def read_back(cache, counts, starts, table, heads, d, fill=None):
    """[tokens, heads, d] in float64; zeros where a place is not there."""
    size, out = cache[0].codes.shape[1], []
    room = size * (1 if table is None else table.shape[1])
    for c in cache:
        x = torch.zeros(sum(counts), heads, d, dtype=torch.float64)
        token = 0
        for i, m in enumerate(counts):
            for r in range(m):
                place = r + (0 if starts is None else starts[i])
                if 0 <= place < room:
                    page, slot = i, place
                    if table is not None:
                        page, slot = int(table[i, place // size]), place % size
                    if 0 <= page < len(c.codes):
                        x[token] = dequantise(c.codes[page, slot],
                                              c.scales[page, slot])
                token += 1
        out.append(x)
    return out


def same(got, want):
    for a, b in zip(got, want):
        assert torch.equal(a.codes.cpu(), b.codes)
        assert torch.equal(a.scales.cpu(), b.scales)


# tokens of each sequence, keys in the cache after them, page (0: one run),
# heads, d: one token; none; ends of pages and of a workgroup's tokens; more
# sequences than lanes, empty ones among them; odd heads
CASES = [
    ([1], [1], 0, 1, 32),
    ([1], [100], 16, 2, 64),
    ([0, 5, 0], [3, 5, 0], 16, 1, 64),
    ([17, 16, 15], [17, 40, 15], 16, 3, 96),
    ([40, 1, 23], [40, 77, 23], 1, 2, 64),
    ([100, 3], [200, 103], 24, 8, 128),
    ([1] * 70, list(range(1, 71)), 8, 2, 64),
    ([0] * 100 + [3] + [0] * 130 + [9, 0, 2], [5] * 231 + [9, 4, 2], 4, 1, 32),
    ([300, 31], [300, 31], 64, 1, 128),
    ([33] * 3, [33] * 3, 0, 10, 128),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_write_and_read(dev, dtype, case):
    counts, lengths, page, heads, d = CASES[case]
    say(f"fp4 write {dtype} {CASES[case]}")
    gen = torch.Generator().manual_seed(case)
    table, pages = (None, len(counts))
    if page:
        table, pages = table_of(lengths, page, gen)
    cache = empty(pages, page or max(lengths), heads, d)
    x = [values(gen, dtype, sum(counts), heads, d) for _ in "kv"]
    off, n = offsets(counts), i32(*lengths)
    want = written(cache, x, counts, lengths, table)
    for head_major in (True, False):
        rows = rows_on_gpu(cache, head_major)
        a = on_gpu(off, n, table, *x)
        assert sw.fp4_cache_write(*a, *rows) == tuple(rows)
        torch.cuda.synchronize()
        same(rows, want)
        # the written tokens back, then everything
        starts = [n - m for n, m in zip(lengths, counts)]
        for m, s in ((counts, starts), (lengths, None)):
            out = [torch.full((sum(m), heads, d), 7.0, dtype=DTYPES[dtype],
                              device=DEV) for _ in "kv"]
            got = sw.fp4_cache_read(
                offsets(m).to(DEV), None if s is None else i32(*s).to(DEV),
                a[2], *rows, *out)
            torch.cuda.synchronize()
            assert got[0] is out[0] and got[1] is out[1]
            for y, z in zip(out, read_back(want, m, s, table, heads, d)):
                assert torch.equal(y.cpu().double(), z)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_many_tokens(dev, dtype):
    """Enough for a workgroup to take several."""
    say(f"fp4 many tokens {dtype}")
    gen = torch.Generator().manual_seed(1)
    for heads, d, t in ((1, 128, 40000), (8, 128, 5000)):
        counts = [t // 2 + 1, 0, t // 3, 7, 13]
        lengths = [c + 100 for c in counts]
        table, pages = table_of(lengths, 16, gen)
        x = [values(gen, dtype, sum(counts), heads, d) for _ in "kv"]
        rows = rows_on_gpu(empty(pages, 16, heads, d))
        a = on_gpu(offsets(counts), i32(*lengths), table, *x)
        sw.fp4_cache_write(*a, *rows)
        out = [torch.empty_like(y) for y in a[3:]]
        sw.fp4_cache_read(a[0], a[1] - i32(*counts).to(DEV), a[2], *rows, *out)
        for y, z in zip(out, x):
            assert torch.equal(y.cpu().double(), dequantise(*quantise(z)))
        # rows that were there before are as they were
        for i, n in enumerate(counts):
            page, slot = int(table[i, 99 // 16]), 99 % 16
            assert (rows[0].codes[page, slot] == 0xA5).all()
            assert (rows[1].scales[page, slot] == 0xA5).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_every_border(dev, dtype):
    """Each border between two codes and its neighbours, in blocks of every
    scale, up to the largest and below the smallest."""
    say(f"fp4 borders {dtype}")
    t = DTYPES[dtype]
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    low = 1 - torch.finfo(t).eps / 2
    x = torch.cat([borders, borders * low, borders * (1 + torch.finfo(t).eps),
                   torch.tensor([0.0, 0.0, 6.0, 6.5])])  # 25
    tops = torch.tensor([7.0, 7.0 * low, 4.0, 3.5 * (1 + torch.finfo(t).eps)])
    blocks = []
    for e in list(range(-149, 126)) + [125]:
        for top in tops:
            b = torch.cat([x, x[:6], top[None]]) * torch.cat(
                [torch.ones(16), -torch.ones(16)])
            blocks.append(b.double() * 2.0 ** e)
    x = torch.stack(blocks)[:, None]
    big = torch.finfo(t).max
    x = x.clamp(-big, big).to(t)
    x[0] = 0.0
    x[1] = -0.0
    x[2, 0, 3] = big
    rows = rows_on_gpu(empty(1, len(x), 1, 32))
    a = on_gpu(i32(0, len(x)), i32(len(x)), x)
    sw.fp4_cache_write(a[0], a[1], None, a[2], a[2], *rows)
    torch.cuda.synchronize()
    want = quantise(x)
    for r in rows:
        assert torch.equal(r.codes[0].cpu(), want[0])
        assert torch.equal(r.scales[0].cpu(), want[1])
    out = [torch.empty_like(a[2]) for _ in "kv"]
    sw.fp4_cache_read(a[0], None, None, *rows, *out)
    y = dequantise(*want)
    assert torch.isfinite(y).all()
    for o in out:
        assert torch.equal(o.cpu().double(), y)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_infinities_and_nan_stay_in_their_block(dev, dtype):
    say(f"fp4 inf {dtype}")
    gen = torch.Generator().manual_seed(2)
    x = values(gen, dtype, 12, 2, 64)
    clean = dequantise(*quantise(x))
    x[2, 1, 40], x[3, 0, 0], x[4, 1, 31] = math.nan, math.inf, -math.inf
    rows = rows_on_gpu(empty(1, 12, 2, 64))
    a = on_gpu(i32(0, 12), i32(12), x)
    sw.fp4_cache_write(a[0], a[1], None, a[2], a[2], *rows)
    out = [torch.empty_like(a[2]) for _ in "kv"]
    sw.fp4_cache_read(a[0], None, None, *rows, *out)
    assert torch.equal(rows[0].scales[0].cpu(), quantise(x)[1])
    clean[2, 1, 32:] = clean[3, 0, :32] = clean[4, 1, :32] = math.nan
    for o in out:
        assert torch.equal(torch.isnan(o.cpu()), torch.isnan(clean))
        assert torch.equal(o.cpu().double().nan_to_num(), clean.nan_to_num())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_every_scale_byte_and_code_reads(dev, dtype):
    """Also those that a write never leaves: up to 2^127, and 2^-127."""
    say(f"fp4 every byte {dtype}")
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1).view(
        256, 1, 16, 16)[:, :, :, None].reshape(256, 16, 1, 16)
    scales = torch.arange(256, dtype=torch.uint8).view(256, 1, 1, 1).expand(
        256, 16, 1, 1).contiguous()
    rows = [sw.Fp4Rows(codes.to(DEV), scales.to(DEV))] * 2
    off = i32(*range(0, 257 * 16, 16)).to(DEV)
    out = [torch.empty(4096, 1, 32, dtype=DTYPES[dtype], device=DEV)
           for _ in "kv"]
    sw.fp4_cache_read(off, None, None, *rows, *out)
    want = dequantise(codes, scales).to(DTYPES[dtype]).view(4096, 1, 32)
    for o in out:
        assert torch.equal(torch.isnan(o.cpu()), torch.isnan(want))
        assert torch.equal(o.cpu().nan_to_num(7, 1e30, -1e30),
                           want.nan_to_num(7, 1e30, -1e30))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_places_that_are_not_there(dev, dtype):
    """Lengths shorter than the tokens, past the table's row and near the ends
    of 32 bits; pages outside the cache; tokens before, behind and between the
    sequences; offsets that fall.  What is there is written, nothing else."""
    say(f"fp4 places {dtype}")
    gen = torch.Generator().manual_seed(3)
    counts = [6, 8, 5, 7, 4, 4]
    lengths = [4, 40, -1, 33, 2 ** 31 - 1, -2 ** 31]
    table = torch.arange(12, dtype=torch.int32).view(6, 2)
    table[1, 1], table[3, 0] = 10 ** 6, -1
    x = [values(gen, dtype, 34, 2, 64) for _ in "kv"]
    cache = empty(12, 16, 2, 64)
    want = written(cache, x, counts, lengths, table)
    rows = rows_on_gpu(cache)
    a = on_gpu(offsets(counts), i32(*lengths), table, *x)
    sw.fp4_cache_write(*a, *rows)
    torch.cuda.synchronize()
    same(rows, want)
    starts = [-2, 30, -2 ** 31, 12, 2 ** 31 - 1, 3]
    out = [torch.full_like(y, 7.0) for y in a[3:]]
    sw.fp4_cache_read(a[0], i32(*starts).to(DEV), a[2], *rows, *out)
    for y, z in zip(out, read_back(want, counts, starts, table, 2, 64)):
        assert torch.equal(y.cpu().double(), z)
    # tokens 0 and 1 and from 30 on are in no sequence
    counts = [6, 8, 5, 7, 2, 0]
    off = offsets(counts) + 2
    out = [torch.full_like(y, 7.0) for y in a[3:]]
    sw.fp4_cache_read(off.to(DEV), None, a[2], *rows, *out)
    for y, z in zip(out, read_back(want, counts, None, table, 2, 64)):
        assert (y[:2] == 7).all() and (y[30:] == 7).all()
        assert torch.equal(y[2:30].cpu().double(), z)
    fresh = rows_on_gpu(cache)
    sw.fp4_cache_write(off.to(DEV), a[1], a[2], *a[3:], *fresh)
    torch.cuda.synchronize()
    same(fresh, written(cache, [y[2:30] for y in x], counts, lengths, table))
    # offsets that fall, and outside the tokens: something, but in bounds
    for bad in ([0, 30, 10, 34, 5, 20, 34], [-9, 3, 90, 1000, 2 ** 31 - 1, 7, 8],
                [2 ** 31 - 1] * 7, [-2 ** 31] * 7):
        b = i32(*bad).to(DEV)
        sw.fp4_cache_write(b, a[1], a[2], *a[3:], *rows)
        sw.fp4_cache_read(b, i32(*starts).to(DEV), a[2], *rows, *out)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_strides(dev, dtype):
    """Keys and values as slices of one projection's output; codes and scales
    of both in one allocation; outputs with heads before tokens."""
    say(f"fp4 strides {dtype}")
    gen = torch.Generator().manual_seed(4)
    counts, lengths = [20, 9], [30, 9]
    table, pages = table_of(lengths, 8, gen)
    x = [values(gen, dtype, 29, 2, 64) for _ in "kv"]
    cache = empty(pages, 8, 2, 64)
    want = written(cache, x, counts, lengths, table)
    # [pages, k or v, heads, 8 * 32 bytes of codes, then 8 * 2 of scales]
    store = torch.full((pages, 2, 2, 8 * 34), 0xA5, dtype=torch.uint8,
                       device=DEV)
    rows = [sw.Fp4Rows(
        store[:, i, :, :256].unflatten(-1, (8, 32)).transpose(1, 2),
        store[:, i, :, 256:].unflatten(-1, (8, 2)).transpose(1, 2))
        for i in range(2)]
    both = torch.cat([*x, x[0]], 1).to(DEV)
    a = on_gpu(offsets(counts), i32(*lengths), table)
    sw.fp4_cache_write(*a, both[:, :2], both[:, 2:4], *rows)
    torch.cuda.synchronize()
    same(rows, want)
    wide = torch.full((2, 2, 40, 64), 7.0, dtype=DTYPES[dtype], device=DEV)
    out = [wide[i, :, 5:34].transpose(0, 1) for i in range(2)]
    sw.fp4_cache_read(a[0], i32(10, 0).to(DEV), a[2], *rows, *out)
    for y, z in zip(out, read_back(want, counts, [10, 0], table, 2, 64)):
        assert torch.equal(y.cpu().double(), z)
    assert (wide[:, :, :5] == 7).all() and (wide[:, :, 34:] == 7).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_past_four_gib(dev, dtype):
    """Pages whose byte offsets pass 2^32, of codes and of scales."""
    say(f"fp4 past 4 GiB {dtype}")
    gen = torch.Generator().manual_seed(5)
    counts = lengths = [40, 33]
    table, pages = table_of(lengths, 16, gen)
    x = [values(gen, dtype, 73, 1, 64) for _ in "kv"]
    cache = empty(pages, 16, 1, 64)
    want = written(cache, x, counts, lengths, table)
    far = (5 << 30) // (pages - 1) // 16 * 16
    store = torch.empty(far * (pages - 1) + 16 * 40, dtype=torch.uint8,
                        device=DEV)
    wide = sw.Fp4Rows(store.as_strided((pages, 16, 1, 32), (far, 32, 32, 1)),
                      store.as_strided((pages, 16, 1, 2), (far, 2, 2, 1), 512))
    a = on_gpu(offsets(counts), i32(*lengths), table, *x)
    spare = rows_on_gpu(cache)
    for pair in ([wide, spare[1]], [spare[0], wide]):
        sw.fp4_cache_write(*a, *pair)
        out = [torch.empty_like(y) for y in a[3:]]
        sw.fp4_cache_read(a[0], None, a[2], *pair, *out)
        for y, z in zip(out, read_back(want, counts, None, table, 1, 64)):
            assert torch.equal(y.cpu().double(), z)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_past_four_gib_of_one_page(dev, dtype):
    """The last keys of a page of 2^20 rows that lie 8 KiB apart, codes and
    scales: written, read back and attended to."""
    say(f"fp4 far rows {dtype}")
    gen = torch.Generator().manual_seed(8)
    n, new, h, hk, d = 2 ** 20 - 3, 20, 4, 2, 64
    x = [values(gen, "f32", new, hk, d).clamp(-4, 4).to(DTYPES[dtype])
         for _ in "kv"]
    q = torch.randn(1, h, d, generator=gen).to(DTYPES[dtype])
    rows = []
    for _ in "kv":
        store = torch.empty(2 ** 33, dtype=torch.uint8, device=DEV)
        rows.append(sw.Fp4Rows(
            store.as_strided((1, 2 ** 20, hk, 32), (0, 8192, 32, 1)),
            store.as_strided((1, 2 ** 20, hk, 2), (0, 8192, 2, 1), 4096)))
    a = on_gpu(i32(0, new), i32(n), q, *x)
    sw.fp4_cache_write(a[0], a[1], None, *a[3:], *rows)
    out = [torch.empty_like(y) for y in a[3:]]
    sw.fp4_cache_read(a[0], a[1] - new, None, *rows, *out)
    held = [dequantise(*quantise(y)) for y in x]
    for y, z in zip(out, held):
        assert torch.equal(y.cpu().double(), z)
    got = torch.empty_like(a[2])
    sw.window_attention_decode_fp4(a[1], None, a[2], *rows, got, 0.125, new)
    for i in range(h):
        o, bound = attend(q[:, i].double(), held[0][:, i // 2],
                          held[1][:, i // 2], 0.125, DTYPES[dtype])
        check(f"head {i}", got[:, i], o, bound)


def test_repeats_streams_and_graphs(dev):
    """The same bytes on another stream and from a captured graph whose
    lengths grow."""
    say("fp4 write graph")
    gen = torch.Generator().manual_seed(6)
    counts, start = [1] * 20, [30 + i for i in range(20)]
    table, pages = table_of([n + 9 for n in start], 8, gen)
    cache = empty(pages, 8, 2, 128)
    a = on_gpu(offsets(counts), i32(*start), table,
               *[values(gen, "bf16", 20, 2, 128) for _ in "kv"])
    eager, graphed, side = (rows_on_gpu(cache) for _ in range(3))
    out = [torch.zeros_like(y) for y in a[3:]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sw.fp4_cache_write(*a, *graphed)
        sw.fp4_cache_read(a[0], a[1], a[2], *graphed, *out)
    other = torch.cuda.Stream()
    for _ in range(4):
        a[1] += 1
        a[3] *= -1.25
        torch.cuda.synchronize()
        sw.fp4_cache_write(*a, *side, stream=other)
        sw.fp4_cache_write(*a, *eager)
        want = sw.fp4_cache_read(a[0], a[1], a[2], *eager,
                                 *[torch.empty_like(y) for y in out])
        graph.replay()
        torch.cuda.synchronize()
        for x, y, z in zip(eager, graphed, side):
            for i in range(2):
                assert torch.equal(x[i], y[i]) and torch.equal(x[i], z[i])
        assert all(torch.equal(x, y) for x, y in zip(want, out))


def test_empty_cache(dev):
    keys = sw.fp4_cache(5, 16, 3, 96)
    assert keys.codes.shape == (5, 16, 3, 48)
    assert keys.scales.shape == (5, 16, 3, 3)
    assert keys.codes.is_cuda and not keys.codes.any()
    assert keys.codes.stride() == (3 * 16 * 48, 48, 16 * 48, 1)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_prompt_and_its_steps(dev, dtype):
    """As a server runs a layer: two prompts' queries and keys get their
    positions, the keys and values go into the cache and come back for the
    prompts' attention; then tokens one by one, each written and attended to."""
    say(f"fp4 layer {dtype}")
    t = DTYPES[dtype]
    gen = torch.Generator().manual_seed(7)
    prompts, steps, h, hk, d, window, sinks = [90, 37], 9, 4, 2, 64, 60, 3
    alpha = 0.125
    table, pages = table_of([n + steps for n in prompts], 16, gen)
    cache = [sw.fp4_cache(pages, 16, hk, d) for _ in "kv"]
    f = (10000.0 ** (-torch.arange(32).double() / 32)).float().to(DEV)
    tg = table.to(DEV)
    held = [[torch.zeros(0, hk, d, dtype=t)] * 2 for _ in prompts]

    def project(n):
        return on_gpu(*[torch.randn(n, m, d, generator=gen).to(t)
                        for m in (h, hk, hk)])

    def keep(k, v, counts):
        """The rounded keys and values as they are in the cache."""
        k, v = (dequantise(*quantise(y.cpu())).to(t) for y in (k, v))
        at = 0
        for i, m in enumerate(counts):
            held[i] = [torch.cat([x, y[at:at + m]])
                       for x, y in zip(held[i], (k, v))]
            at += m

    def expect(q, out, places, prompt):
        """Query rows at places[i] (sequence, place)."""
        for r, (i, p) in enumerate(places):
            j = torch.arange(p + 1)
            see = j[(j > p - window) | (j < sinks)]
            for x in range(h):
                a = (q[r, x:x + 1].cpu().double(),
                     held[i][0][see, x // 2].double(),
                     held[i][1][see, x // 2].double())
                if prompt:
                    o, bound, *_ = softmax(
                        *a, torch.ones(1, len(see), dtype=torch.bool), alpha,
                        half_step(t))
                else:
                    o, bound = attend(*a, alpha, t)
                check(f"sequence {i}, place {p}, head {x}", out[r, x:x + 1], o,
                      bound)

    q, k, v = project(sum(prompts))
    pos = torch.cat([torch.arange(n) for n in prompts]).to(torch.int32)
    sw.rotary(pos[None].to(DEV), f, None, q, k, q, k)
    off, n = offsets(prompts).to(DEV), i32(*prompts).to(DEV)
    sw.fp4_cache_write(off, n, tg, k, v, *cache)
    back = sw.fp4_cache_read(off, None, tg, *cache, torch.empty_like(k),
                             torch.empty_like(v))
    keep(k, v, prompts)
    for x, y in zip(back, zip(*held)):
        assert torch.equal(x.cpu(), torch.cat(y))
    out = torch.empty_like(q)
    sw.window_attention(off, off, q, *back, out, None, alpha, window, sinks)
    expect(q, out, [(i, p) for i, m in enumerate(prompts) for p in range(m)],
           True)
    for step in range(steps):
        q, k, v = project(2)
        sw.rotary(n[None], f, None, q, k, q, k)
        n += 1
        sw.fp4_cache_write(i32(0, 1, 2).to(DEV), n, tg, k, v, *cache)
        keep(k, v, [1, 1])
        out = torch.empty_like(q)
        sw.window_attention_decode_fp4(n, tg, q, *cache, out, alpha, window,
                                       sinks)
        expect(q, out, [(i, m + step) for i, m in enumerate(prompts)], False)
