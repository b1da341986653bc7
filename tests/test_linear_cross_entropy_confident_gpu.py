"""Rows that are nearly certain of their class: small losses, whose gradients are as small, against the formula in 64 bits."""
import pytest
import torch

from warpconvnet_b200 import linear_cross_entropy

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# two roundings to 16 bits (the logits' gradient, the result), 0.6 of each in the mean
TOL = {torch.float16: 6e-4, torch.bfloat16: 5e-3}
# a loss is the logarithm of a sum that begins with one: half a spacing of 2^-23 for each of some additions to it is, of such losses,
# less than those roundings
LOSSES = {torch.float16: (1e-3, 1e-2), torch.bfloat16: (1e-4, 1e-3)}
SIZES = [(64, 40), (96, 200), (64, 700), (128, 4096), (512, 300), (256, 256)]


def problem(c, v, dtype, n=600):
    """Rows along the weights of their class, as far as their loss comes to lie between the limits; logits of up to 30."""
    g = torch.Generator().manual_seed(c + v)
    w = torch.randn(v, c, generator=g)
    w = (w / w.norm(dim=1, keepdim=True) * 5).to(dtype)
    labels = torch.randint(0, v, (n,), generator=g)
    noise = 0.3 * torch.randn(n, c, generator=g).double()
    low, high = LOSSES[dtype]
    want = torch.exp(torch.empty(n, dtype=torch.float64).uniform_(float(torch.tensor(low).log()), float(torch.tensor(high).log()), generator=g))
    lo, hi = torch.zeros(n, dtype=torch.float64), torch.full((n,), 4.0, dtype=torch.float64)
    wd = w.double()
    for _ in range(40):
        mid = (lo + hi) / 2
        z = (mid[:, None] * wd[labels] + noise) @ wd.t()
        loss = torch.logsumexp(z, 1) - z.gather(1, labels[:, None])[:, 0]
        lo, hi = torch.where(loss > want, mid, lo), torch.where(loss > want, hi, mid)
    return (lo[:, None] * wd[labels] + noise).to(dtype), w, labels


@pytest.mark.parametrize("dtype", list(TOL))
@pytest.mark.parametrize("c,v", SIZES)
def test_small_losses_and_their_gradients(c, v, dtype):
    x, w, labels = problem(c, v, dtype)
    xd, wd = x.double(), w.double()
    z = xd @ wd.t()
    want = torch.logsumexp(z, 1) - z.gather(1, labels[:, None])[:, 0]
    leaf = x.to(DEV).requires_grad_(True)
    row = linear_cross_entropy(leaf, w.to(DEV), labels.to(DEV), reduction="none")
    # eight spacings of the sum; the logits' own, sums of C products, to a loss their relative error
    assert float(((row.detach().cpu().double() - want).abs() - 1e-4 * want).max()) <= 8 * 2.0 ** -23
    weights = 1 / want   # (all rows count alike)
    (dx,) = torch.autograd.grad(row, [leaf], weights.float().to(DEV))
    p = torch.softmax(z, 1)
    p[torch.arange(len(p)), labels] = torch.expm1(-want)
    exact = (p * weights.float().double()[:, None]) @ wd
    assert float((dx.cpu().double() - exact).norm() / exact.norm()) <= TOL[dtype]
