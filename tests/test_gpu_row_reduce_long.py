"""Row reductions of rows that a whole wave takes, whose last windows reach into
the next rows: those hold NaN here, and the last rows end with the array."""
import pytest
import torch

import sparsewavecomp_amd as sw
from tests import gpu_util as G

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("many", [0, 40000])
@pytest.mark.parametrize("last", [2049, 4095, 4096, 4097, 7001])
def test_long_rows_beside_nan(dev, dt, many, last):
    """`many` rows of one entry in front: fewer lanes a row, and so several long
    rows in a wave."""
    G.say(f"long rows beside NaN {dt} {many} {last}")
    lens = torch.tensor([1] * many + [2049, 3, 2500, 2, 1, 2051, 5000, 1, 3000,
                                      2, 9000, 1, 4096, 1, last])
    long = lens > 1000
    ro = torch.zeros(len(lens) + 1, dtype=torch.int64)
    ro[1:] = lens.cumsum(0)
    g = torch.Generator().manual_seed(last)
    val = torch.randn(int(ro[-1]), generator=g).to(dt)
    val[~long.repeat_interleave(lens)] = float("nan")
    v = val.double()
    for off in (0, 1, 5):
        x = torch.empty(len(val) + off, dtype=dt, device=G.DEV)[off:]
        x.copy_(val)
        for kind in ("max", "sum"):
            out = torch.zeros(len(lens), dtype=dt, device=G.DEV)
            sw.csr_row_reduce(ro.int().to(G.DEV), None, x, out, kind)
            got = out.cpu().double()
            assert torch.isnan(got[~long]).all()
            for r in long.nonzero()[:, 0].tolist():
                row = v[ro[r]:ro[r + 1]]
                if kind == "max":
                    assert got[r] == row.max()
                    continue
                # (a sum of n terms in any order, then the type's rounding)
                bound = (len(row) + 1) * 2.0 ** -24 * row.abs().sum()
                half = torch.finfo(dt).eps / 2
                assert abs(got[r] - row.sum()) <= bound + half * (
                    abs(row.sum()) + bound)
