"""The linear cross entropy in fp32: what its roundings come to, and what it takes beside its results."""
import pytest
import torch

from warpconvnet_b200 import linear_cross_entropy
from warpconvnet_b200._native import WCN_F32, query_bytes

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


def test_what_the_losses_take_does_not_grow_with_the_classes():
    """Beside lse and loss: a pair for each row and group of classes, of which there are at most 256."""
    few, many = (query_bytes("wcn_linear_ce_workspace_bytes", 100000, 16, v, WCN_F32, 0) for v in (16384, 200000))
    assert many <= few <= 100000 * 256 * 8 + (1 << 20)


@pytest.mark.parametrize("v", [16384, 16385, 40007])
def test_many_classes(v):
    g = torch.Generator().manual_seed(v)
    n, c = 130, 12
    x, w, b, labels = torch.randn(n, c, generator=g), torch.randn(v, c, generator=g), torch.randn(v, generator=g), torch.randint(0, v, (n,), generator=g)
    labels[3], labels[4] = v - 1, 0
    x[5] = 0
    b[v // 2:] -= 200.0   # (whole groups of classes far below the others)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    row = linear_cross_entropy(leaves[0], leaves[1], labels.to(DEV), leaves[2], reduction="none")
    xd, wd, bd = (t.double().to(DEV).requires_grad_(True) for t in (x, w, b))
    z = xd @ wd.t() + bd
    want = torch.logsumexp(z, 1) - z.gather(1, labels.to(DEV)[:, None])[:, 0]
    room = 1.2e-7 * (2 + c / 16) * (1 + float((x.abs().double() @ w.abs().double().t() + b.abs().double()).max()))
    assert float((row.detach().double() - want).abs().max()) <= room
    for a, r in zip(torch.autograd.grad(row.mean(), leaves), torch.autograd.grad(want.mean(), [xd, wd, bd])):
        assert float((a.double() - r).norm() / r.norm()) <= 3e-6 + room


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_more_classes_than_a_grid_has_rows(dtype):
    """4.3 million classes: 65 535 tiles of 64 of them are fewer."""
    g = torch.Generator(device=DEV).manual_seed(0)
    n, c, v = 3, 8, 4_300_037
    x, w = (torch.randn(k, c, generator=g, device=DEV).to(dtype) for k in (n, v))
    labels = torch.tensor([0, v - 1, 4_200_000], device=DEV)
    leaves = [t.requires_grad_(True) for t in (x, w)]
    loss = linear_cross_entropy(*leaves, labels)
    xd, wd = (t.detach().double().requires_grad_(True) for t in (x, w))
    z = xd @ wd.t()
    want = (torch.logsumexp(z, 1) - z.gather(1, labels[:, None])[:, 0]).mean()
    assert abs(float(loss) - float(want)) <= 1e-5
    tol = 5e-3 if dtype == torch.bfloat16 else 1e-5
    for a, r in zip(torch.autograd.grad(loss, leaves), torch.autograd.grad(want, [xd, wd])):
        assert float((a.double() - r).norm() / r.norm()) <= tol
