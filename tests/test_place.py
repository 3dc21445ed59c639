"""The device and stream that the rotary and 4-bit cache calls go to, on a torch
with and without the names that give them quickest."""
import pytest
import torch

import sparsewavecomp_amd as sw


class Current:
    cuda_stream = 77


@pytest.mark.parametrize("missing", [
    (), ("_cuda_getDevice",), ("_cuda_getCurrentRawStream",),
    ("_cuda_getDevice", "_cuda_getCurrentRawStream")])
def test_place_of_the_current_stream(monkeypatch, missing):
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: Current)
    for name, f in (("_cuda_getDevice", lambda: 3),
                    ("_cuda_getCurrentRawStream", lambda at: 74 + at)):
        monkeypatch.setattr(torch._C, name, f, raising=False)
        if name in missing:
            monkeypatch.delattr(torch._C, name)
    sw._load_torch()
    assert sw._place(None) == (3, 77)


def test_place_before_torch_has_begun(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: False)
    sw._load_torch()
    assert sw._place(Current) == (-2, None)
    assert sw._place(None) == (-2, None)
