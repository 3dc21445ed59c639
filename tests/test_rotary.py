"""What the rotary entry points refuse, before any launch."""
import ctypes

import pytest

import sparsewavecomp_amd as sw

A = 1 << 20  # an aligned address that no call here reaches
PACKED = [256, 64, 128, 64, 256, 64, 128, 64]


def call(name="sw_rotary_bf16", strides=None, **kw):
    a = dict(positions=A, frequencies=A, pair_axes=A, query=A, key=2 * A,
             query_output=3 * A, key_output=4 * A, tokens=3, axes=2,
             query_heads=4, key_heads=2, d=64, pairs=32, interleaved=0,
             strides=None, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    if strides:
        a["strides"] = (ctypes.c_int64 * 8)(*strides)
    lib = sw.load_library()
    return getattr(lib, name)(*a.values()), lib.sw_last_error().decode()


def changed(i, v):
    return PACKED[:i] + [v] + PACKED[i + 1:]


@pytest.mark.parametrize("name", [
    "sw_rotary_f32", "sw_rotary_bf16", "sw_rotary_backward_f32",
    "sw_rotary_backward_bf16"])
@pytest.mark.parametrize("kw,code,needle", [
    (dict(tokens=-1), -2, "tokens"),
    (dict(tokens=2 ** 30 + 1), -2, "tokens"),
    (dict(axes=0), -2, "axes"),
    (dict(axes=65537), -2, "axes"),
    (dict(query_heads=0), -2, "query heads"),
    (dict(key_heads=-1), -2, "key heads"),
    (dict(key_heads=65537), -2, "key heads"),
    (dict(d=20), -2, "multiple of 8"),
    (dict(d=136), -2, "multiple of 8"),
    (dict(pairs=0), -2, "pairs"),
    (dict(pairs=33), -2, "pairs"),
    (dict(positions=None), -3, "positions pointer is null"),
    (dict(frequencies=None), -3, "frequencies pointer is null"),
    (dict(pair_axes=A + 2), -3, "not aligned"),
    (dict(query=None), -3, "query pointer is null"),
    (dict(key=None), -3, "key pointer is null"),
    (dict(query_output=3 * A + 4), -3, "must be 16-byte aligned"),
    (dict(strides=changed(0, 32)), -2, "query strides"),
    (dict(strides=changed(3, 2 ** 60)), -2, "key strides"),
    (dict(strides=changed(5, 0)), -2, "rows overlap"),
    (dict(strides=changed(6, 2 ** 24)), -2, "strides"),
    (dict(query_output=A, strides=changed(4, 512)), -3, "in place"),
    (dict(key_output=2 * A, strides=[256, 64, 128, 64, 256, 64, 64, 192]), -3,
     "in place"),
])
def test_refused(name, kw, code, needle):
    rc, message = call(name, **kw)
    assert rc == code and needle in message


def test_nothing_to_do():
    assert call(tokens=0, positions=None, frequencies=None, query=None,
                key=None, query_output=None, key_output=None)[0] == 0


def test_mirror_refuses():
    import torch
    p = torch.zeros(2, 5, dtype=torch.int32)
    f, ax = torch.zeros(32), torch.zeros(32, dtype=torch.int32)
    q, k = torch.zeros(5, 4, 64), torch.zeros(5, 2, 64)

    def forward(**kw):
        a = dict(positions=p, frequencies=f, pair_axes=ax, query=q, key=k,
                 query_output=q, key_output=k)
        sw.rotary(**{**a, **kw})

    with pytest.raises(ValueError, match="device tensor"):
        forward()
    for kw, match in ((dict(query_output=q[:4]), "query_output"),
                      (dict(key=None), "key_output"),
                      (dict(key=k[:3], key_output=k[:3]), "key"),
                      (dict(positions=p[0]), "positions"),
                      (dict(positions=p[:, :4]), "positions"),
                      (dict(frequencies=f[None]), "frequencies"),
                      (dict(pair_axes=ax[:3]), "pair_axes")):
        with pytest.raises(sw.ShapeError, match=match):
            forward(**kw)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        forward(query=q.half(), query_output=q.half())
    with pytest.raises(sw.ShapeError, match="query_gradient"):
        sw.rotary_backward(p, f, ax, q, k, q[1:], k)
