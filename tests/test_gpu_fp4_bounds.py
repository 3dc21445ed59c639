"""What the 4-bit cache's write and read leave alone when their offsets make no
sense: falling, negative, past the tokens, at the ends of 32 bits."""
import pytest
import torch

import sparsewavecomp_amd as sw
from gpu_util import DEV, say
from test_gpu_fp4_cache import DTYPES, i32, read_back, values

pytestmark = pytest.mark.gpu

TOKENS, PAGES, PAGE, HEADS, D = 34, 12, 16, 2, 64
LENGTHS = [4, 40, -1, 33, 2 ** 31 - 1, -2 ** 31]
STARTS = [-2, 30, -2 ** 31, 12, 2 ** 31 - 1, 3]
BAD = [
    [0, 30, 10, 34, 5, 20, 34],
    [34, 28, 20, 13, 9, 4, 0],
    [-9, 3, 90, 1000, 2 ** 31 - 1, 7, 8],
    [-2 ** 31, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, -1, 0, 34],
    [2 ** 31 - 1] * 7,
    [-2 ** 31] * 7,
    [5, 5, 5, 5, 5, 5, 6],
]


def guarded(shape, dtype, fill, pad):
    """(all memory, a view of `shape` with `pad` elements on both sides)."""
    n = torch.Size(shape).numel()
    store = torch.full((n + 2 * pad,), fill, dtype=dtype, device=DEV)
    return store, store[pad:pad + n].view(shape)


def holders(off):
    """The sequences that hold each token."""
    return [[i for i in range(len(off) - 1) if off[i] <= t < off[i + 1]]
            for t in range(TOKENS)]


def page_slot(table, i, place):
    if not 0 <= place < PAGE * table.shape[1]:
        return None
    page = int(table[i, place // PAGE])
    return (page, place % PAGE) if 0 <= page < PAGES else None


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bad", range(len(BAD)))
def test_offsets_that_make_no_sense(dev, dtype, bad):
    """Rows of no token, tokens of no sequence and all memory around caches and
    outputs keep their bits; a token that is read is what one of the sequences
    that hold it has in its place."""
    off = BAD[bad]
    say(f"fp4 offsets {dtype} {off}")
    gen = torch.Generator().manual_seed(bad)
    table = torch.arange(12, dtype=torch.int32).view(6, 2)
    table[1, 1], table[3, 0] = 10 ** 6, -1
    held = holders(off)
    x = [values(gen, dtype, TOKENS, HEADS, D).to(DEV) for _ in "kv"]
    stores, rows = [], []
    for _ in "kv":
        parts = []
        for width in (D // 2, D // 32):
            store, view = guarded((PAGES, HEADS, PAGE, width), torch.uint8,
                                  0x5C, 4096)
            view.copy_(torch.randint(0, 250, view.shape, generator=gen))
            stores.append((store, store.clone()))
            parts.append(view.transpose(1, 2))
        rows.append(sw.Fp4Rows(*parts))
    where = i32(*off).to(DEV), i32(*LENGTHS).to(DEV), table.to(DEV)
    before = [[y.clone() for y in r] for r in rows]

    sw.fp4_cache_write(*where, *x, *rows)
    torch.cuda.synchronize()
    reached = torch.zeros(PAGES, PAGE, dtype=torch.bool)
    for t, sequences in enumerate(held):
        for i in sequences:
            at = page_slot(table, i, LENGTHS[i] - (off[i + 1] - t))
            if at:
                reached[at] = True
    for r, old in zip(rows, before):
        for y, z in zip(r, old):
            assert torch.equal(y.cpu()[~reached], z.cpu()[~reached])
            z.copy_(y)
    for store, old in stores:
        for side in (slice(0, 4096), slice(-4096, None)):
            assert torch.equal(store[side], old[side])

    outs, to = [], []
    for _ in "kv":
        store, view = guarded((TOKENS, HEADS, D), DTYPES[dtype], 7.0, 2048)
        outs.append(store)
        to.append(view)
    sw.fp4_cache_read(where[0], i32(*STARTS).to(DEV), where[2], *rows, *to)
    torch.cuda.synchronize()
    for store in outs:
        assert (store[:2048] == 7).all() and (store[-2048:] == 7).all()
    for r, old in zip(rows, before):
        assert all(torch.equal(y, z) for y, z in zip(r, old))
    cpu = [sw.Fp4Rows(*(y.cpu() for y in r)) for r in rows]
    for y, cache in zip(to, cpu):
        y = y.cpu().double()
        for t, sequences in enumerate(held):
            if not sequences:
                assert (y[t] == 7).all(), t
                continue
            may = [y[t] == 7]  # (a search of offsets that fall may miss it)
            for i in sequences:
                want, _ = read_back([cache, cache], [1],
                                    [STARTS[i] + t - off[i]], table[i:i + 1],
                                    HEADS, D)
                may.append(y[t] == want[0])
            assert any(m.all() for m in may), t
