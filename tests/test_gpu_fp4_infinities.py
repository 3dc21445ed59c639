"""Attention against a cache of 4-bit codes whose values pass the types' range:
scale bytes of 253 and 254, which no write leaves."""
import math

import pytest
import torch

from gpu_util import say
from test_gpu_fp4_attention import decode, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("h,hk,d", [(8, 1, 32), (4, 2, 64), (8, 1, 128),
                                    (16, 1, 64), (24, 1, 128), (3, 1, 96)])
def test_infinite_values(dev, dtype, h, hk, d):
    """4 and 6 times 2^126, and 2 and more times 2^127, are infinite: so is the
    sum of what is seen, in those elements of their head's rows alone, whatever
    the number of query heads that share it."""
    say(f"fp4 infinite values {dtype} {h} {hk} {d}")
    g, signs = h // hk, torch.tensor([-math.inf, math.inf]).repeat(8)
    for lengths in ([300, 40], [900, 520]):
        x = make(dtype, lengths, 0, h, hk, d, seed=h + d)
        want = decode(x, 0.125, 10 ** 6, 0)
        codes, scales = x["value_cache"]
        kept = codes.clone(), scales.clone()
        for key, byte, code in ((3, 253, 0x7E), (20, 254, 0x4C),
                                (lengths[0] - 1, 254, 0x7D)):
            # half of the row's first block, the other half of it zero: -4 and
            # 6 times 2^126, -2 and 2, -3 and 6 times 2^127
            codes[0, key, 0, :16] = 0
            codes[0, key, 0, :8] = code
            scales[0, key, 0, 0] = byte
            got = decode(x, 0.125, 10 ** 6, 0)
            assert torch.equal(got[0, :g, :16].float(), signs.expand(g, 16)), (
                key, byte)
            got[0, :g, :32] = want[0, :g, :32]
            assert torch.equal(got, want), (key, byte)
            codes.copy_(kept[0])
            scales.copy_(kept[1])
        # an infinity of either sign
        for key, code in ((3, 0x77), (21, 0xFF)):
            codes[0, key, 0, :16], scales[0, key, 0, 0] = code, 254
        got = decode(x, 0.125, 10 ** 6, 0)
        assert torch.isnan(got[0, :g, :32]).all()
        got[0, :g, :32] = want[0, :g, :32]
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("h", [8, 16])
def test_the_largest_finite_values(dev, dtype, h):
    """One key: 3 times 2^126 and 3/2 times 2^127 come back as they are."""
    say(f"fp4 largest finite values {dtype} {h}")
    x = make(dtype, [1], 0, h, 1, 64, seed=h)
    codes, scales = x["value_cache"]
    for byte, code, size in ((253, 0xD5, 3 * 2.0 ** 126),
                             (254, 0xB3, 1.5 * 2.0 ** 127)):
        codes[0, 0, 0], scales[0, 0, 0] = code, byte
        got = decode(x, 0.125, 10 ** 6, 0).double()
        want = torch.tensor([size, -size], dtype=torch.float64).repeat(32)
        # fp32: a weight, a sum and their product round (bf16 hides them)
        off = 0.0 if dtype == "bf16" else 8 * 2.0 ** -24
        assert ((got - want).abs() <= off * size).all()
