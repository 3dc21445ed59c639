"""That the marks of tests/_fp4_marks.py show what attention may leave out."""
import pytest
import torch

import sparsewavecomp_amd as sw
from _fp4_check import attend, dequantise
from _fp4_marks import (CASES, build, expect, lengths_of, outputs,
                        relative_bound, weights)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_a_tile_shows(dtype, d, case):
    """A result without one of the tiles, or with it twice, is off by more than
    the bound in the element that it marks, whichever tile and row."""
    *_, window, sinks, h, hk = CASES[case]
    w, seen = weights(max(lengths_of(case)), h, d, window, sinks)
    most = relative_bound(int((seen > 0).sum()), dtype)
    mark = torch.arange(w.shape[1]) % d
    total = w.sum(1, keepdim=True)
    own = torch.zeros(h, d, dtype=torch.float64).index_add_(1, mark, w)[:, mark]
    whole = seen == 32  # (the others are at the ends of what is seen)
    for sign in (-1, 1):
        off = ((own + sign * w) / own * total / (total + sign * w) - 1).abs()
        assert (off[:, whole] > most).all()


def test_closed_form():
    """The marks' closed form against attention over the codes' values."""
    for d, page in ((32, 16), (96, 0)):
        x = build(torch.float32, [70, 0, 300], page, 4, 2, d, 300, 3)
        out = torch.zeros(3, 4, d)
        for i, n in enumerate((70, 0, 300)):
            j = torch.arange(n)
            at, slot = torch.full_like(j, i), j
            if page:
                at, slot = x["table"][i].long()[j // page], j % page
            k, v = (dequantise(c[at, slot], s[at, slot]) for c, s in (
                x["key_cache"], x["value_cache"]))
            see = (j >= n - 200) | (j < 40)
            for head in range(2):
                rows = slice(2 * head, 2 * head + 2)
                o, _ = attend(x["query"][i, rows].double(), k[see, head],
                              v[see, head], 1.0, torch.float32)
                if n:
                    w, _ = weights(n, 4, d, 200, 40)
                    assert torch.allclose(outputs(w, i, 2, d)[rows], o,
                                          rtol=1e-12, atol=0)
                out[i, rows] = o.float()
        expect(x, out, 200, 40)
        out[2, 1] = 0
        with pytest.raises(AssertionError, match="sequence 2"):
            expect(x, out, 200, 40)


def test_cases_are_split():
    need = sw.load_library().sw_window_attention_decode_fp4_workspace_bytes
    joined = set()
    for n, _, _, room, page, window, sinks, h, hk in CASES:
        for d in (32, 64, 96, 128):
            size, width = (page, -(-room // page)) if page else (room, 1)
            assert need(n, size, width, h, hk, d, window, sinks) > 0
        joined.add(n * h > 512)
    assert joined == {False, True}
