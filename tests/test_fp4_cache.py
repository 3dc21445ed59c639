"""What the 4-bit cache's entry points refuse, before any launch, and the
arithmetic that they share with the host."""
import ctypes
import random

import pytest

import sparsewavecomp_amd as sw

A = 1 << 20  # an aligned address that no call here reaches
ROWS = [1024, 64, 32, 64, 4, 2]  # page 16, 2 heads of 64: codes, scales
MOVED = [128, 64, 128, 64] + ROWS * 2
STEP = [256, 64, 256, 64] + ROWS * 2
CACHE = dict(key_codes=A, key_scales=A, value_codes=A, value_scales=A)
SIZES = dict(pages=5, page_size=16, table_width=3)


def call(op, dt="_bf16", strides=None, **kw):
    if op == "decode":
        a = dict(key_lengths=A, page_table=A, query=A, **CACHE, output=A,
                 sequences=2, **SIZES, query_heads=4, key_heads=2, d=64,
                 strides=None, window=8, sinks=1, alpha=1.0, workspace=A,
                 workspace_bytes=1 << 30, stream=None)
        name = "sw_window_attention_decode_fp4"
    else:
        moved = dict(key=A, value=A)
        a = dict(token_offsets=A, per_sequence=A, page_table=A)
        a |= moved | CACHE if op == "write" else CACHE | moved
        a |= dict(sequences=2, tokens=7, **SIZES, key_heads=2, d=64,
                  strides=None, stream=None)
        name = "sw_fp4_cache_" + op
    assert set(kw) <= set(a)
    a.update(kw)
    if strides:
        a["strides"] = (ctypes.c_int64 * 16)(*strides)
    lib = sw.load_library()
    return getattr(lib, name + dt)(*a.values()), lib.sw_last_error().decode()


def changed(op, i, v):
    s = STEP if op == "decode" else MOVED
    return s[:i] + [v] + s[i + 1:]


@pytest.mark.parametrize("dt", ["_f32", "_bf16"])
@pytest.mark.parametrize("op", ["write", "read", "decode"])
@pytest.mark.parametrize("kw,code,needle", [
    (dict(sequences=-1), -2, "sequences"),
    (dict(sequences=2 ** 30 + 1), -2, "sequences"),
    (dict(page_size=0), -2, "pages"),
    (dict(page_size=1 << 16, table_width=1 << 15), -2, "2^30 keys"),
    (dict(table_width=0), -2, "pages"),
    (dict(pages=-1), -2, "pages"),
    (dict(page_table=None, pages=1), -2, "every sequence needs its page"),
    (dict(key_heads=0), -2, "key heads"),
    (dict(d=40), -2, "blocks of 32"),
    (dict(d=160), -2, "multiple of 8 up to 128"),
    (dict(page_table=A + 2), -3, "not aligned"),
    (dict(key_codes=None), -3, "key codes pointer is null"),
    (dict(value_scales=None), -3, "value scales pointer is null"),
    (dict(value_codes=A + 8), -3, "value codes must be 16-byte aligned"),
    (dict(strides=(4, -64)), -2, "key codes strides"),
    (dict(strides=(4, 2 ** 41)), -2, "key codes strides"),
    (dict(strides=(5, 16)), -2, "key codes strides"),
    (dict(strides=(5, 2 ** 24)), -2, "key codes strides"),
    (dict(strides=(6, 40)), -3, "key codes must be 16-byte aligned"),
    (dict(strides=(8, 1)), -2, "key scales strides"),
    (dict(strides=(9, -1)), -2, "key scales strides"),
    (dict(strides=(14, 1)), -2, "value scales strides"),
])
def test_refused(dt, op, kw, code, needle):
    if "strides" in kw:
        kw = dict(strides=changed(op, *kw["strides"]))
    rc, message = call(op, dt, **kw)
    assert rc == code and needle in message


@pytest.mark.parametrize("op,kw,code,needle", [
    ("write", dict(tokens=-1), -2, "tokens"),
    ("read", dict(tokens=2 ** 30 + 1), -2, "tokens"),
    ("write", dict(token_offsets=None), -3, "token offsets pointer"),
    ("read", dict(token_offsets=A + 1), -3, "not aligned"),
    ("write", dict(per_sequence=None), -3, "key lengths pointer is null"),
    ("read", dict(per_sequence=A + 3), -3, "not aligned"),
    ("write", dict(key=None), -3, "key pointer is null"),
    ("read", dict(value=A + 8), -3, "value must be 16-byte aligned"),
    ("read", dict(strides=changed("read", 1, 0)), -2, "key rows overlap"),
    # (what is written shares no memory: pages, rows or heads on each other)
    ("write", dict(strides=changed("write", 4, 0)), -2, "key rows overlap"),
    ("write", dict(strides=changed("write", 4, 1008)), -2, "key rows overlap"),
    ("write", dict(strides=changed("write", 6, 16)), -2, "key rows overlap"),
    ("write", dict(strides=changed("write", 9, 1)), -2, "key rows overlap"),
    ("write", dict(strides=changed("write", 13, 60)), -2, "value rows overlap"),
    ("write", dict(strides=changed("write", 13, 2 ** 40), pages=2 ** 25), -2,
     "value rows overlap"),
    ("decode", dict(sequences=(1 << 24) + 1), -2, "sequences"),
    ("decode", dict(query_heads=5), -2, "multiple of key heads"),
    ("decode", dict(key_lengths=None), -3, "key lengths pointer is null"),
    ("decode", dict(key_lengths=A + 1), -3, "not aligned"),
    ("decode", dict(query=None), -3, "query pointer is null"),
    ("decode", dict(output=A + 4), -3, "output must be 16-byte aligned"),
    ("decode", dict(strides=changed("decode", 3, 0)), -2, "output rows overlap"),
    ("decode", dict(window=0), -2, "window of at least 1"),
    ("decode", dict(sinks=-1), -2, "no negative sinks"),
    ("decode", dict(alpha=float("nan")), -3, "alpha must be finite"),
    ("decode", dict(alpha=3.0e38), -3, "alpha must be finite"),
    ("decode", dict(page_size=1 << 17, window=1 << 17, workspace=None), -3,
     "workspace of"),
    ("decode", dict(page_size=1 << 17, window=1 << 17, workspace=A + 8), -3,
     "workspace of"),
    ("decode", dict(page_size=1 << 17, window=1 << 17, workspace_bytes=15), -3,
     "workspace of"),
])
def test_one_refuses(op, kw, code, needle):
    rc, message = call(op, **kw)
    assert rc == code and needle in message


def test_nothing_to_do():
    for op in ("write", "read"):
        for kw in (dict(sequences=0), dict(tokens=0, key=None, value=None)):
            assert call(op, token_offsets=None, **kw)[0] == 0
    assert call("decode", sequences=0, key_lengths=None, query=None,
                output=None, workspace=None)[0] == 0


def test_decode_workspace():
    need = sw.load_library().sw_window_attention_decode_fp4_workspace_bytes
    assert need(2, 16, 3, 4, 2, 64, 8, 1) == 0
    assert need(0, 1 << 20, 3, 4, 2, 64, 1 << 20, 1) == 0
    assert need(2, 1 << 20, 3, 4, 2, 40, 1 << 20, 1) == 0  # refused
    assert need(1, 1 << 17, 1, 8, 2, 128, 1 << 20, 0) > 0
    # only what is seen counts
    assert need(1, 1 << 17, 1, 8, 2, 128, 200, 40) == 0


def test_mirror_refuses():
    import torch
    n = torch.zeros(2, dtype=torch.int32)
    off = torch.zeros(3, dtype=torch.int32)
    table = torch.zeros(2, 3, dtype=torch.int32)
    rows = sw.Fp4Rows(torch.zeros(5, 16, 2, 32, dtype=torch.uint8),
                      torch.zeros(5, 16, 2, 2, dtype=torch.uint8))
    k, q = torch.zeros(7, 2, 64), torch.zeros(2, 4, 64)

    def write(**kw):
        a = dict(token_offsets=off, key_lengths=n, page_table=table, key=k,
                 value=k, key_cache=rows, value_cache=rows)
        sw.fp4_cache_write(**{**a, **kw})

    def read(**kw):
        a = dict(token_offsets=off, starts=n, page_table=table, key=k, value=k,
                 key_cache=rows, value_cache=rows)
        sw.fp4_cache_read(**{**a, **kw})

    def decode(**kw):
        a = dict(key_lengths=n, page_table=table, query=q, key_cache=rows,
                 value_cache=rows, output=q, alpha=1.0, window=4)
        sw.window_attention_decode_fp4(**{**a, **kw})
    bad = (sw.Fp4Rows(rows.codes[:4], rows.scales[:4]),
           sw.Fp4Rows(rows.codes, rows.scales[:, :3]),
           sw.Fp4Rows(rows.codes, rows.scales[..., :1]),
           sw.Fp4Rows(rows.codes[..., :16], rows.scales),
           sw.Fp4Rows(rows.codes[0], rows.scales[0]))
    for f in (write, read, decode):
        with pytest.raises(ValueError, match="device tensor"):
            f()
        for c in bad:
            with pytest.raises(sw.ShapeError, match="key and value caches"):
                f(value_cache=c)
        with pytest.raises(sw.ShapeError, match="page_table"):
            f(page_table=table[0])
        with pytest.raises(sw.ShapeError, match="page_table"):
            f(page_table=table[:1])
    for f, name in ((write, "key_lengths"), (read, "starts"),
                    (decode, "key_lengths")):
        with pytest.raises(sw.ShapeError, match=name):
            f(**{name: n[:1]})
    with pytest.raises(sw.ShapeError, match="key_lengths"):
        write(key_lengths=None)
    for f in (write, read):
        with pytest.raises(sw.ShapeError, match="tokens, key_heads, d"):
            f(value=k[:3])
        with pytest.raises(TypeError, match="float32 or bfloat16"):
            f(key=k.half())
        with pytest.raises(sw.ShapeError, match="1-D tensor"):
            f(token_offsets=off[None])
    with pytest.raises(sw.ShapeError, match="query and output"):
        decode(output=q[:1])
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        decode(query=q.half())
    for d in (0, 16, 40, 160):
        with pytest.raises(sw.ShapeError, match="32, 64, 96 or 128"):
            sw.fp4_cache(1, 16, 2, d)


def test_division_by_a_factor():
    """The kernels divide n < 2^31 by d as n m / 2^(31 + s): m = 2^(31 + s) / d
    rounded up, s = log2 d rounded up."""
    rng = random.Random(1)
    for d in [2, 3, 5, 7, 24, 48, 63, 64, 65, 2 ** 30, 2 ** 30 - 1] + [
            rng.randrange(2, 1 << rng.randrange(2, 31)) for _ in range(2000)]:
        s = (d - 1).bit_length()
        m = -(-(1 << (31 + s)) // d)
        assert m < 1 << 32
        for n in (0, 1, d - 1, d, 2 ** 31 - 1, (2 ** 31 - 1) // d * d,
                  (2 ** 31 - 1) // d * d - 1, rng.randrange(1 << 31)):
            assert (n * m >> 32) >> (s - 1) == n // d
