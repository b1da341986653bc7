"""Group norm of rows that hardly differ, against the formula in 64 bits, with its gradients."""
import pytest
import torch

from warpconvnet_b200 import segmented_group_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = [torch.float16, torch.bfloat16]
# a result is rounded once: 0.6 of 2^-11 / 2^-8 in the mean
TOL = {torch.float16: 6e-4, torch.bfloat16: 5e-3}


def off(a, b, scale=None):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).norm() / max(float(b.norm()), float(scale.norm()) if scale is not None else 0.0, 1e-300))


def run(x, offsets, groups, w, b, dy, eps=1e-5):
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    y = segmented_group_norm(leaves[0], offsets, groups, leaves[1], leaves[2], eps)
    return [y.detach().cpu(), *(t.cpu() for t in torch.autograd.grad(y, leaves, dy.to(DEV)))]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("value", [10.0, 100.0, 1000.0, -30000.0])
@pytest.mark.parametrize("offsets,c,groups", [([0, 300, 1001], 16, 2), ([0, 300, 1001], 12, 12), (list(range(41)), 24, 24), ([0, 7, 8, 3000], 20, 4)])
def test_constant_groups(dtype, value, offsets, c, groups):
    """The distance from the mean is nothing whatever 1 / std is: y is beta, rounded, and the gradient of gamma nothing."""
    g = torch.Generator().manual_seed(0)
    n = offsets[-1]
    x = torch.full((n, c), value).to(dtype)
    w, b, dy = torch.rand(c, generator=g) + 0.5, torch.randn(c, generator=g), torch.randn(n, c, generator=g).to(dtype)
    y, dx, dw, db = run(x, offsets, groups, w, b, dy)
    assert torch.equal(y, b.expand(n, c).to(dtype))
    assert not dw.any()
    want = torch.empty(n, c, dtype=torch.float64)
    for lo, hi in zip(offsets, offsets[1:]):
        h = (dy[lo:hi].double() * w.double()).view(hi - lo, groups, -1)
        want[lo:hi] = ((h - h.mean((0, 2), keepdim=True)) / 1e-5 ** 0.5).view(hi - lo, c)
    assert off(dx, want, dy.double() * w / 1e-5 ** 0.5) <= TOL[dtype]
    assert off(db, dy.double().sum(0), dy.double().norm(dim=0)) <= 4e-6


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("channels_alike", [True, False])
def test_means_that_are_large_against_the_spread(dtype, channels_alike):
    """Two values one spacing apart: half the rows have either, so that the mean is a number of 32 bits and xhat +-1 (the tile's sums
    of distances are exact too).  Or channels of unlike size in groups of their own."""
    n, c = 4000, 16
    low = torch.full((c,), 512.0) if channels_alike else torch.exp2(torch.arange(c) % 14 + 1.0)
    x = low.expand(n, c).clone()
    x[n // 2:] += low * (2.0 ** -10 if dtype == torch.float16 else 2.0 ** -7)
    x = x[torch.randperm(n, generator=torch.Generator().manual_seed(0))].to(dtype)
    g = torch.Generator().manual_seed(1)
    w, b, dy = torch.rand(c, generator=g) + 0.5, torch.randn(c, generator=g), torch.randn(n, c, generator=g).to(dtype)
    xr, wr, br = (t.double().requires_grad_(True) for t in (x, w, b))
    mean = xr.mean(0)
    yr = (xr - mean) * torch.rsqrt((xr - mean).square().mean(0) + 1e-5) * wr + br
    want = torch.autograd.grad(yr, [xr, wr, br], dy.double())
    y, dx, dw, db = run(x, None, c, w, b, dy)
    rstd = 1 / (x.double().var(0, correction=0) + 1e-5).sqrt()
    assert off(y, yr) <= TOL[dtype] and off(dx, want[0], dy.double() * w * rstd) <= TOL[dtype]
    terms = dy.double().norm(dim=0)
    assert off(dw, want[1], terms) <= 4e-6 and off(db, want[2], terms) <= 4e-6
