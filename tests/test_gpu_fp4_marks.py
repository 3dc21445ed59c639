"""Attention against a cache of 4-bit codes over many parts, on values that mark
their tile (tests/_fp4_marks.py): heads of every size, rows joined by a wave and
by a workgroup."""
import pytest

import sparsewavecomp_amd as sw
from _fp4_marks import CASES, build, expect, lengths_of
from gpu_util import say
from test_gpu_fp4_attention import DTYPES, decode, make, put
from test_gpu_fp4_attention import expect as expect_random

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_every_tile_counts_once(dev, dtype, d, case):
    n, _, _, room, page, window, sinks, h, hk = CASES[case]
    say(f"fp4 marks {dtype} {d} {CASES[case]}")
    x = build(DTYPES[dtype], lengths_of(case), page, h, hk, d, room, case)
    expect(x, decode(x, 1.0, window, sinks), window, sinks)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
def test_random_values_joined_by_waves(dev, dtype, d):
    """More than 512 rows, sequences of two parts to a dozen."""
    say(f"fp4 joins of more than 512 rows {dtype} {d}")
    lengths = [3000, 0, 700, 1, 2500, 600] + [100] * 60
    x = make(dtype, lengths, 16, 8, 1, d, seed=d)
    expect_random(x, decode(x, 0.1, 10 ** 6, 0), 0.1, 10 ** 6)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_alpha_below_the_normal_numbers_in_parts(dev, dtype):
    """As test_gpu_fp4_attention has it for one part: 602 keys that are seen, of
    70 sequences of 8 heads."""
    say(f"fp4 decode small alpha in parts {dtype}")
    lengths = [40, 700] + [9] * 68
    assert sw.load_library().sw_window_attention_decode_fp4_workspace_bytes(
        70, 32, 22, 8, 1, 64, 600, 2) > 0
    x = make(dtype, lengths, 32, 8, 1, 64, seed=5)
    x["query"] *= 2.0 ** 60
    for i in range(70):
        put(x, "key", i, x["keys"][i] * 2.0 ** 60)
    expect_random(x, decode(x, 5e-39, 600, 2), 5e-39, 600, 2)
