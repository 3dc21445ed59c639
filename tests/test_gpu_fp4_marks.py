"""Attention against a cache of 4-bit codes over many parts, on values that mark
their tile (tests/_fp4_marks.py): heads of every size, rows joined by a wave and
by a workgroup."""
import pytest

from _fp4_marks import CASES, build, expect, lengths_of
from gpu_util import say
from test_gpu_fp4_attention import DTYPES, decode

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_every_tile_counts_once(dev, dtype, d, case):
    n, _, _, room, page, window, sinks, h, hk = CASES[case]
    say(f"fp4 marks {dtype} {d} {CASES[case]}")
    x = build(DTYPES[dtype], lengths_of(case), page, h, hk, d, room, case)
    expect(x, decode(x, 1.0, window, sinks), window, sinks)
