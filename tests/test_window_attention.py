"""What the window attention entry points refuse, before any launch."""
import ctypes

import pytest

import sparsewavecomp_amd as sw

A = 1 << 20  # an aligned address that no call here reaches


def c_forward(strides=None, dt="_bf16", **kw):
    a = dict(query_offsets=A, key_offsets=A, query=A, key=A, value=A, output=A,
             log_sum=None, sequences=1, query_tokens=10, key_tokens=10,
             query_heads=4, key_heads=2, d=64, window=8, sinks=1, alpha=1.0)
    a.update(kw)
    s = (ctypes.c_int64 * 8)(*strides) if strides else None
    rc = getattr(sw.load_library(), "sw_window_attention" + dt)(
        a["query_offsets"], a["key_offsets"], a["query"], a["key"],
        a["value"], a["output"], a["log_sum"], a["sequences"],
        a["query_tokens"], a["key_tokens"], a["query_heads"], a["key_heads"],
        a["d"], s, a["window"], a["sinks"], a["alpha"], None)
    return rc, sw.load_library().sw_last_error().decode()


@pytest.mark.parametrize("kw,code,needle", [
    (dict(sequences=-1), -2, "sequences and tokens"),
    (dict(query_tokens=2 ** 31), -2, "sequences and tokens"),
    (dict(query_heads=3), -2, "multiple of key heads"),
    (dict(key_heads=0), -2, "multiple of key heads"),
    (dict(d=60), -2, "multiple of 8"),
    (dict(d=136), -2, "multiple of 8"),
    (dict(d=0), -2, "multiple of 8"),
    (dict(window=0), -2, "window of at least 1"),
    (dict(sinks=-1), -2, "no negative sinks"),
    (dict(alpha=float("nan")), -3, "alpha must be finite"),
    (dict(alpha=float("inf")), -3, "alpha must be finite"),
    (dict(query_offsets=None), -3, "offsets pointer is null"),
    (dict(key=None), -3, "key pointer is null"),
    (dict(output=None), -3, "output pointer is null"),
    (dict(value=A + 2), -3, "value must be 16-byte aligned"),
    (dict(log_sum=A + 2), -3, "not aligned"),
    (dict(strides=[256, 64, 128, 4, 128, 64, 256, 64]), -3, "key must be 16-byte"),
    (dict(strides=[32, 64, 128, 64, 128, 64, 256, 64]), -2, "query strides"),
    (dict(strides=[256, -64, 128, 64, 128, 64, 256, 64]), -2, "query strides"),
    (dict(strides=[1 << 23, 64, 128, 64, 128, 64, 256, 64]), -2, "2^23 bytes"),
    (dict(strides=[256, 64, 128, 64, 128, 64, 256, 0]), -2, "output rows overlap"),
    (dict(strides=[256, 64, 128, 64, 128, 64, 128, 64]), -2, "output rows overlap"),
    (dict(strides=[256, 64, 128, 64, 128, 64, 64, 320]), -2, "output rows overlap"),
])
@pytest.mark.parametrize("dt", ["_f32", "_bf16"])
def test_refused(dt, kw, code, needle):
    if dt == "_f32" and "strides" in kw and code == -3:
        kw = dict(kw, strides=[256, 64, 128, 2, 128, 64, 256, 64])
    rc, message = c_forward(dt=dt, **kw)
    assert rc == code and needle in message


def c_backward(strides=None, dt="_bf16", **kw):
    a = dict(query_offsets=A, key_offsets=A, query=A, key=A, value=A, output=A,
             log_sum=A, output_gradient=A, query_gradient=A, key_gradient=A,
             value_gradient=A, sequences=1, query_tokens=10, key_tokens=10,
             query_heads=4, key_heads=2, d=64, window=8, sinks=1, alpha=1.0,
             workspace=A, workspace_bytes=1 << 30)
    a.update(kw)
    v = list(a.values())
    s = (ctypes.c_int64 * 16)(*strides) if strides else None
    rc = getattr(sw.load_library(), "sw_window_attention_backward" + dt)(
        *v[:17], s, *v[17:], None)
    return rc, sw.load_library().sw_last_error().decode()


FULL = [256, 64, 128, 64, 128, 64, 256, 64, 256, 64, 256, 64, 128, 64, 128, 64]


@pytest.mark.parametrize("kw,code,needle", [
    (dict(d=12), -2, "multiple of 8"),
    (dict(window=-3), -2, "window of at least 1"),
    (dict(log_sum=None), -3, "log_sum pointer is null"),
    (dict(output_gradient=None), -3, "output gradient pointer is null"),
    (dict(key_gradient=None), -3, "key gradient pointer is null"),
    (dict(workspace=None), -3, "workspace of"),
    (dict(workspace=A + 8), -3, "workspace of"),
    (dict(workspace_bytes=100), -3, "workspace of"),
    (dict(strides=FULL[:10] + [256, 0] + FULL[12:]), -2, "query gradient rows overlap"),
    (dict(strides=FULL[:12] + [64, 64] + FULL[14:]), -2, "key gradient rows overlap"),
    (dict(strides=FULL[:14] + [120, 64]), -2, "value gradient rows overlap"),
])
@pytest.mark.parametrize("dt", ["_f32", "_bf16"])
def test_backward_refused(dt, kw, code, needle):
    rc, message = c_backward(dt=dt, **kw)
    assert rc == code and needle in message


def test_backward_workspace_rule():
    need = sw.load_library().sw_window_attention_backward_workspace_bytes
    # two numbers of each query and head
    assert need(1, 100, 100, 4, 2, 64, 100, 7, 2) == 2 * 4 * 100 * 4
    # sinks apart: those of the window, and of one chunk of 64 queries a
    # sequence more than whole ones, 32 rows each
    rows = 2 * 32 * 2 * 64
    assert need(3, 100, 100, 4, 2, 64, 99, 7, 2) == 2 * 4 * 100 * 4 + \
        4 * rows * (3 + 1 + 3)
    assert need(3, 5000, 100, 4, 2, 64, 99, 7, 2) == 2 * 4 * 5000 * 4 + \
        4 * rows * (3 + 78 + 3)
    assert need(3, 99000, 100, 4, 2, 64, 99, 7, 2) == 2 * 4 * 99000 * 4 + \
        4 * rows * (3 + 386 + 3)
    # parts of few keys: dk and dv of each, in tiles of 128 keys, one more for
    # each sequence and head than there can be whole ones
    tiles, row = 33 * 4, 4 * 2 * 128
    one = need(1, 4096, 4096, 8, 4, 128, 4096, 0, 2)
    assert one == 2 * 4 * 8 * 4096 + 3 * tiles * 128 * row
    assert need(1, 4096, 4096, 8, 4, 128, 4096, 0, 4) == \
        2 * 4 * 8 * 4096 + 2 * tiles * 128 * row
    assert need(1, 4096, 4096, 12, 12, 128, 4096, 0, 2) == 2 * 4 * 12 * 4096
    # those behind the last 512 tiles, but for the numbers without keys
    assert need(1, 17000, 17000, 16, 4, 128, 1024, 0, 2) == \
        2 * 4 * 16 * 17000 + 16 * (133 * 4 - 512) * 128 * row
    for n in (1, 6):
        assert need(n, 16384, 16384, 16, 4, 128, 1024, 0, 2) == \
            2 * 4 * 16 * 16384
    # many sinks: at most the size of bf16 keys apart from a chunk a sequence
    # and the window's
    n = 1 << 20
    for sinks in (64, 100, 1000, 5000):
        assert need(1, n, n, 1, 1, 128, 64, sinks, 2) <= 2 * 4 * n + \
            2 * 2 * n * 128 + 3 * 4 * 256 * (sinks + 31)
    assert need(1, 100, 100, 4, 3, 64, 100, 7, 2) == 0
    assert need(1, 100, 100, 4, 2, 64, 100, 7, 8) == 0


def test_backward_workspace_of_many_sequences():
    """The sinks' sums are bounded by the keys, however many sequences there
    are and however many sinks none of them has."""
    need = sw.load_library().sw_window_attention_backward_workspace_bytes

    def sums(n, tokens, sinks, window=1024):
        return need(n, tokens, tokens, 32, 8, 128, window, sinks, 2) - \
            need(n, tokens, tokens, 32, 8, 128, window, 0, 2)
    keys = 2 * 8 * 128  # bytes of a bf16 key of all heads
    fp32 = 4 * keys     # of its two sums
    # the window's and the first chunk's sums, at most a row a key of each, and
    # one row for four queries of the later chunks' (twice that for fewer sinks
    # than a block has)
    for n, tokens in ((1, 65536), (64, 16384), (64, 65536), (4096, 262144),
                      (8192, 262144), (100, 262144)):
        for sinks in (1, 4, 32, 64, 65, 1000, 4096, 65536, 2 ** 40):
            for window in (16, 1024, 16000):
                bound = fp32 * (2 * (tokens + 32 * min(n, tokens // window)) +
                                tokens // 4 + 1024)
                assert 0 < sums(n, tokens, sinks, window) <= bound
    # blocks of 32 sinks: by sequence,
    block = 32 * fp32
    assert sums(6, 16384, 4) == (2 * 6 + 64) * block
    # by the sequences that may hold more keys than the window, 255 here,
    assert sums(8192, 262144, 64) == (2 * 255 * 2 + 1024 * 2) * block
    # and by keys: 15360 / 32 and 15
    assert sums(64, 16384, 2 ** 40) == 2 * 495 * block
    assert sums(2, 16384, 2 ** 40) == 2 * 482 * block


@pytest.mark.parametrize("dt", ["_f32", "_bf16"])
@pytest.mark.parametrize("alpha", [3.0e38, -2.4e38])
def test_refuses_an_alpha_that_overflows(dt, alpha):
    """Scores are scaled by alpha log2 e, which has to be finite itself."""
    for call in (c_forward, c_backward):
        rc, message = call(dt=dt, alpha=alpha)
        assert rc == -3 and "alpha must be finite" in message


def test_nothing_to_do():
    assert c_backward(sequences=0, workspace=None)[0] == 0
    assert c_backward(query_tokens=0, key_tokens=0, workspace=None)[0] == 0
    assert c_forward(sequences=0, query_offsets=None, key_offsets=None)[0] == 0
    assert c_forward(query_tokens=0, query=None, output=None)[0] == 0


def test_mirror_refuses():
    import torch
    off = torch.zeros(2, dtype=torch.int32)
    q, k = torch.zeros(4, 4, 64), torch.zeros(4, 2, 64)

    def call(qo=off, ko=off, query=q, key=k, value=k, output=q, log_sum=None):
        sw.window_attention(qo, ko, query, key, value, output, log_sum, 1.0, 4)
    with pytest.raises(ValueError, match="device tensor"):
        call()
    with pytest.raises(sw.ShapeError, match="expected query"):
        call(value=k[:3])
    with pytest.raises(sw.ShapeError, match="expected query"):
        call(key=k[..., :32], value=k[..., :32])
    with pytest.raises(sw.ShapeError, match="same length"):
        call(ko=off[:1])
    with pytest.raises(sw.ShapeError, match="query's shape"):
        call(output=k)
    with pytest.raises(sw.ShapeError, match="log_sum"):
        call(log_sum=torch.zeros(4, 5))
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        call(query=q.half())

    def back(**kw):
        a = dict(query_offsets=off, key_offsets=off, query=q, key=k, value=k,
                 output=q, log_sum=torch.zeros(4, 4), output_gradient=q,
                 query_gradient=q, key_gradient=k, value_gradient=k,
                 alpha=1.0, window=4)
        sw.window_attention_backward(**{**a, **kw})
    with pytest.raises(ValueError, match="device tensor"):
        back()
    with pytest.raises(sw.ShapeError, match="output_gradient must"):
        back(output_gradient=k)
    with pytest.raises(sw.ShapeError, match="value_gradient must"):
        back(value_gradient=q)
    with pytest.raises(sw.ShapeError, match="log_sum"):
        back(log_sum=torch.zeros(4, 3))


def test_strides_of_one_row():
    """A single token of a buffer whose heads lie far apart: its row stride is
    not used, and what the mirror passes for it is no reason to refuse."""
    import torch
    buf = torch.zeros(4, 1 << 17, 64, dtype=torch.bfloat16)
    assert buf.stride(0) * 2 > 1 << 23
    one = buf[:, 7:8].transpose(0, 1)
    for heads in (4, 1):
        _, strides = sw._heads(torch.bfloat16, -1, one[:, :heads], "query",
                               one[:, :2], "key", one[:, :2], "value",
                               one[:, :heads], "output")
        rc, message = c_forward(strides, query_tokens=1, key_tokens=1,
                                query_heads=heads, key_heads=min(heads, 2),
                                query_offsets=A + 1)
        # (refused for the offsets alone, behind the checks of all strides)
        assert rc == -3 and "not aligned" in message
    page = torch.zeros(3, 8, dtype=torch.bfloat16).as_strided(
        (1, 2, 1, 8), (5, 8, 8, 1))
    assert list(sw._heads(torch.bfloat16, -1, page, "key_cache", one,
                          "query")[1]) == [0, 8, 8, 64, 1 << 23]


def test_assembly_names_what_it_changes():
    """Every written-out statement that sets m0 lists it as changed, so that
    the compiler carries no value of its own across."""
    import glob
    import os
    import re
    sources = glob.glob(os.path.join(os.path.dirname(sw.__file__), "csrc", "*"))
    found = 0
    for path in sources:
        with open(path) as f:
            text = f.read()
        for m in re.finditer(r"\basm volatile\((.*?)\);", text, re.S):
            if re.search(r"\bm0,", m[1]):
                found += 1
                assert '"m0"' in m[1].rsplit(":", 1)[1], (path, m[0])
    assert found >= 2
