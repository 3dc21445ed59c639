"""What the cache attention entry points refuse, before any launch."""
import ctypes

import pytest

import sparsewavecomp_amd as sw

A = 1 << 20  # an aligned address that no call here reaches
PACKED = [256, 64, 256, 64, 2048, 128, 64, 2048, 128, 64, 128, 64, 128, 64]


def call(prefix, dt="_bf16", strides=None, **kw):
    a = dict(key_lengths=A, page_table=A, query=A)
    if prefix:
        a.update(prefix_key=A, prefix_value=A)
    a.update(key_cache=A, value_cache=A, output=A, sequences=2)
    if prefix:
        a.update(prefix_tokens=7)
    a.update(pages=5, page_size=16, table_width=3, query_heads=4, key_heads=2,
             d=64, strides=None)
    if not prefix:
        a.update(window=8, sinks=1)
    a.update(alpha=1.0, workspace=A, workspace_bytes=1 << 30, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    if strides:
        a["strides"] = (ctypes.c_int64 * 14)(*strides)
    name = "sw_shared_prefix_attention" if prefix else \
        "sw_window_attention_decode"
    rc = getattr(sw.load_library(), name + dt)(*a.values())
    return rc, sw.load_library().sw_last_error().decode()


def changed(i, v):
    return PACKED[:i] + [v] + PACKED[i + 1:]


@pytest.mark.parametrize("kw,code,needle", [
    (dict(sequences=-1), -2, "sequences"),
    (dict(sequences=(1 << 24) + 1), -2, "sequences"),
    (dict(page_size=0), -2, "pages"),
    (dict(page_size=1 << 16, table_width=1 << 15), -2, "2^30 keys"),
    (dict(table_width=0), -2, "pages"),
    (dict(pages=-1), -2, "pages"),
    (dict(page_table=None, pages=1), -2, "every sequence needs its page"),
    (dict(query_heads=5), -2, "multiple of key heads"),
    (dict(d=20), -2, "multiple of 8"),
    (dict(alpha=float("inf")), -3, "alpha must be finite"),
    (dict(key_lengths=None), -3, "key lengths pointer is null"),
    (dict(key_lengths=A + 1), -3, "not aligned"),
    (dict(page_table=A + 2), -3, "not aligned"),
    (dict(query=None), -3, "query pointer is null"),
    (dict(output=A + 4), -3, "output must be 16-byte aligned"),
    (dict(key_cache=None), -3, "key cache pointer is null"),
    (dict(value_cache=A + 8), -3, "value cache must be 16-byte aligned"),
    (dict(strides=changed(4, -64)), -2, "key cache page stride"),
    (dict(strides=changed(7, 2 ** 41)), -2, "value cache page stride"),
    (dict(strides=changed(7, 2050)), -3, "value cache must be 16-byte aligned"),
    (dict(strides=changed(5, 32)), -2, "key cache strides"),
    (dict(strides=changed(6, 2 ** 60)), -2, "key cache strides"),
    (dict(strides=changed(3, 0)), -2, "output rows overlap"),
])
@pytest.mark.parametrize("prefix", [False, True])
@pytest.mark.parametrize("dt", ["_f32", "_bf16"])
def test_refused(dt, prefix, kw, code, needle):
    rc, message = call(prefix, dt, **kw)
    assert rc == code and needle in message


@pytest.mark.parametrize("kw,code,needle", [
    (dict(window=0), -2, "window of at least 1"),
    (dict(sinks=-1), -2, "no negative sinks"),
])
def test_decode_refused(kw, code, needle):
    rc, message = call(False, **kw)
    assert rc == code and needle in message


@pytest.mark.parametrize("kw,code,needle", [
    (dict(prefix_tokens=-1), -2, "prefix"),
    (dict(prefix_tokens=2 ** 31), -2, "prefix"),
    (dict(prefix_key=None), -3, "prefix key pointer is null"),
    (dict(prefix_value=A + 2), -3, "prefix value must be 16-byte"),
    (dict(strides=changed(10, 32)), -2, "prefix key strides"),
    (dict(workspace=None), -3, "workspace of"),
    (dict(workspace=A + 8), -3, "workspace of"),
    (dict(workspace_bytes=15), -3, "workspace of"),
])
def test_prefix_refused(kw, code, needle):
    rc, message = call(True, **kw)
    assert rc == code and needle in message


@pytest.mark.parametrize("prefix", [False, True])
@pytest.mark.parametrize("dt", ["_f32", "_bf16"])
@pytest.mark.parametrize("alpha", [3.0e38, -2.4e38])
def test_refuses_an_alpha_that_overflows(dt, prefix, alpha):
    rc, message = call(prefix, dt, alpha=alpha)
    assert rc == -3 and "alpha must be finite" in message


def test_decode_workspace():
    need = sw.load_library().sw_window_attention_decode_workspace_bytes
    # few keys: one workgroup for each, nothing to join
    assert need(2, 16, 3, 4, 2, 64, 8, 1) == 0
    assert need(0, 1 << 20, 3, 4, 2, 64, 1 << 20, 1) == 0
    assert need(2, 16, 3, 4, 3, 64, 8, 1) == 0
    long = need(1, 1 << 17, 1, 8, 2, 128, 1 << 20, 0)
    assert long > 0
    # only what is seen counts
    assert need(1, 1 << 17, 1, 8, 2, 128, 200, 40) == 0
    rc, message = call(False, page_size=1 << 17, window=1 << 17,
                       workspace=None)
    assert rc == -3 and "workspace of" in message


def test_nothing_to_do():
    for prefix in (False, True):
        assert call(prefix, sequences=0, key_lengths=None, query=None,
                    output=None, workspace=None)[0] == 0


def test_mirror_refuses():
    import torch
    n = torch.zeros(2, dtype=torch.int32)
    q, c = torch.zeros(2, 4, 64), torch.zeros(5, 16, 2, 64)
    table = torch.zeros(2, 3, dtype=torch.int32)

    def decode(**kw):
        a = dict(key_lengths=n, page_table=table, query=q, key_cache=c,
                 value_cache=c, output=q, alpha=1.0, window=4)
        sw.window_attention_decode(**{**a, **kw})

    def prefix(**kw):
        a = dict(key_lengths=n, page_table=table, query=q,
                 prefix_key=c[0], prefix_value=c[0], key_cache=c,
                 value_cache=c, output=q, alpha=1.0)
        sw.shared_prefix_attention(**{**a, **kw})
    for f in (decode, prefix):
        with pytest.raises(ValueError, match="device tensor"):
            f()
        with pytest.raises(sw.ShapeError, match="query and output"):
            f(output=q[:1])
        with pytest.raises(sw.ShapeError, match="key and value caches"):
            f(value_cache=c[:1])
        with pytest.raises(sw.ShapeError, match="key_lengths"):
            f(key_lengths=n[:1])
        with pytest.raises(sw.ShapeError, match="page_table"):
            f(page_table=table[0])
        with pytest.raises(TypeError, match="float32 or bfloat16"):
            f(query=q.half())
    with pytest.raises(sw.ShapeError, match="prefix key and value"):
        prefix(prefix_value=c[1, :3])
