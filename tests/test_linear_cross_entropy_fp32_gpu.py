"""The linear cross entropy in fp32: what its roundings come to, and what it takes beside its results."""
import pytest
import torch

from warpconvnet_b200 import linear_cross_entropy

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_large_logits_keep_their_differences():
    """Logits around 200 that are exact (x against an identity, multiples of 1/8).  A loss is a difference of such numbers, which is
    exact, and the logarithm of a sum of 64 (at most 3e-6 of it, and a rounding of up to 12); a gradient has one rounding of the
    log-sum-exp, by at most 2^-17, 0.58 of that in the mean."""
    g = torch.Generator().manual_seed(0)
    n, v = 4000, 64
    z = (200 + 1.5 * torch.randn(n, v, generator=g)).mul(8).round() / 8
    labels = torch.randint(0, v, (n,), generator=g)
    zd = z.double()
    want = torch.logsumexp(zd, 1) - zd.gather(1, labels[:, None])[:, 0]
    x = z.to(DEV).requires_grad_(True)
    row = linear_cross_entropy(x, torch.eye(v, device=DEV), labels.to(DEV), reduction="none")
    assert float((row.detach().cpu().double() - want).abs().max()) <= 3e-6
    (dx,) = torch.autograd.grad(row, [x], torch.ones(n, device=DEV))
    p = torch.softmax(zd, 1)
    p[torch.arange(n), labels] = 0   # (the label's is made from the loss)
    got = dx.cpu().double()
    got[torch.arange(n), labels] = 0
    assert float((got - p).norm() / p.norm()) <= 0.58 * 2.0 ** -17 + 1e-6
