"""Sizes beyond what the linear cross entropy takes are refused by name.  (Tensors without memory stand for the large ones.)"""
import pytest
import torch

from warpconvnet_b200.nn.functional import linear_cross_entropy as lce


@pytest.mark.parametrize("n,c,v,what", [(4, 32769, 5, "channels"), (0x7FFFFF00, 8, 5, "rows"), (4, 8, 0x7FFFFF00, "classes")])
def test_sizes(monkeypatch, n, c, v, what):
    monkeypatch.setattr(lce, "require_cuda", lambda *a: None)
    x, w, labels = torch.empty(n, c, device="meta"), torch.empty(v, c, device="meta"), torch.empty(n, dtype=torch.int64, device="meta")
    with pytest.raises(ValueError, match=what):
        lce.linear_cross_entropy(x, w, labels)
