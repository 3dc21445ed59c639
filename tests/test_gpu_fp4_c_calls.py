"""The 4-bit cache's write, read and token step called as a C program does, on
strides that it fills itself."""
import ctypes

import pytest
import torch

import sparsewavecomp_amd as sw
from gpu_util import DEV, say

pytestmark = pytest.mark.gpu

# page, token and head stride, in bytes, of codes and of scales: pages of 64
# places that hold the rows of one of 8 heads of 128 together
ROWS = [8 * 64 * 64, 64, 64 * 64, 8 * 64 * 4, 4, 64 * 4]
MOVED = [8 * 128, 128, 8 * 128, 128, *ROWS, *ROWS]
STEP = [32 * 128, 128, 32 * 128, 128, *ROWS, *ROWS]


def test_c_calls(dev):
    say("fp4 C calls")
    lib, gen = sw.load_library(), torch.Generator().manual_seed(1)
    moved, step = ((ctypes.c_int64 * 16)(*x) for x in (MOVED, STEP))
    lengths, width = [700, 90, 1], 11
    off = torch.tensor([0, 700, 790, 791], dtype=torch.int32, device=DEV)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    table = torch.arange(3 * width, dtype=torch.int32, device=DEV).view(3, -1)
    k, v = (torch.randn(791, 8, 128, generator=gen).bfloat16().to(DEV)
            for _ in "kv")
    q = torch.randn(3, 32, 128, generator=gen).bfloat16().to(DEV)
    rows = [sw.fp4_cache(3 * width, 64, 8, 128, DEV) for _ in "kv"]
    cache = [y.data_ptr() for r in rows for y in r]
    back = [torch.zeros_like(k) for _ in "kv"]
    out = torch.zeros_like(q)
    sizes = (3 * width, 64, width)
    need = lib.sw_window_attention_decode_fp4_workspace_bytes(
        3, 64, width, 32, 8, 128, 10 ** 6, 0)
    assert need > 0
    space = torch.empty(need, dtype=torch.uint8, device=DEV)
    at, handle = sw._place(None)
    for rc in (
            lib.sw_fp4_cache_write_bf16(
                off.data_ptr(), n.data_ptr(), table.data_ptr(), k.data_ptr(),
                v.data_ptr(), *cache, 3, 791, *sizes, 8, 128, moved, handle),
            lib.sw_fp4_cache_read_bf16(
                off.data_ptr(), None, table.data_ptr(), *cache,
                *(y.data_ptr() for y in back), 3, 791, *sizes, 8, 128, moved,
                handle),
            lib.sw_window_attention_decode_fp4_bf16(
                n.data_ptr(), table.data_ptr(), q.data_ptr(), *cache,
                out.data_ptr(), 3, *sizes, 32, 8, 128, step, 10 ** 6, 0, 0.0884,
                space.data_ptr(), need, handle)):
        assert rc == 0, lib.sw_last_error()
    torch.cuda.synchronize()
    mirror = [sw.fp4_cache(3 * width, 64, 8, 128, DEV) for _ in "kv"]
    want = [torch.zeros_like(k) for _ in "kv"]
    sw.fp4_cache_write(off, n, table, k, v, *mirror)
    sw.fp4_cache_read(off, None, table, *mirror, *want)
    for a, b in zip(back, want):
        assert torch.equal(a, b) and a.any()
    for a, b in zip(rows, mirror):
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    got = torch.zeros_like(q)
    sw.window_attention_decode_fp4(n, table, q, *mirror, got, 0.0884, 10 ** 6)
    assert torch.equal(out, got) and out.any()
