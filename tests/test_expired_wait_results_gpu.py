"""What group norm and the linear cross entropy leave where an earlier kernel gave up waiting: numbers that can't be mistaken for
results, and everything that is shared between launches as it was.  (The status word is set from the host: nothing waits.)"""
import pytest
import torch

from warpconvnet_b200 import linear_cross_entropy, segmented_group_norm
from warpconvnet_b200._native import check_device_status, device_status

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EXPIRED = -7


class expired:
    def __enter__(self):
        device_status(DEV).fill_(EXPIRED)

    def __exit__(self, *exc):
        assert int(device_status(DEV)) == EXPIRED   # (stays until it is read)
        device_status(DEV).zero_()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("offsets,c", [([0, 1, 5], 6), ([0, 300, 1000], 32), ([0, 90000, 200000], 64), (list(range(0, 4001, 10)), 16)])
def test_group_norm(dtype, offsets, c):
    g = torch.Generator().manual_seed(0)
    n = offsets[-1]
    x = torch.randn(n, c, generator=g).to(dtype).to(DEV).requires_grad_(True)
    w, b = (torch.rand(c, generator=g).to(DEV).requires_grad_(True) for _ in range(2))
    forward = lambda: segmented_group_norm(x, offsets, 2, w, b, activation="silu")   # noqa: E731
    y = forward()
    want = [y.detach(), *torch.autograd.grad(y, [x, w, b], torch.ones_like(y), retain_graph=True)]
    with expired():
        bad = [forward().detach(), *torch.autograd.grad(y, [x, w, b], torch.ones_like(y), retain_graph=True)]
        with torch.no_grad():
            bad.append(forward())
    assert all(torch.isnan(t).all() for t in bad)
    for _ in range(2):
        y = forward()
        got = [y.detach(), *torch.autograd.grad(y, [x, w, b], torch.ones_like(y))]
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    check_device_status(DEV)


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("dtype,n,c,v", [(torch.float32, 300, 40, 70), (torch.bfloat16, 300, 40, 20), (torch.float16, 30000, 96, 200), (torch.bfloat16, 700, 64, 1000),
                                         (torch.bfloat16, 300, 512, 500), (torch.float16, 400, 256, 256)])
def test_linear_cross_entropy(dtype, n, c, v, reduction):
    g = torch.Generator().manual_seed(0)
    x, w = (torch.randn(k, c, generator=g).to(dtype).to(DEV).requires_grad_(True) for k in (n, v))
    b, labels = torch.randn(v, generator=g).to(dtype).to(DEV).requires_grad_(True), torch.randint(0, v, (n,), generator=g).to(DEV)
    forward = lambda: linear_cross_entropy(x, w, labels, b, reduction=reduction)   # noqa: E731
    loss = forward()
    want = [loss.detach(), *torch.autograd.grad(loss, [x, w, b], torch.ones_like(loss), retain_graph=True)]
    with expired():
        bad = [forward().detach(), *torch.autograd.grad(loss, [x, w, b], torch.ones_like(loss), retain_graph=True)]
        for t in (x, w, b):
            bad += torch.autograd.grad(loss, [t], torch.ones_like(loss), retain_graph=True)
    assert all(torch.isnan(t).all() for t in bad)
    for _ in range(2):
        loss = forward()
        got = [loss.detach(), *torch.autograd.grad(loss, [x, w, b], torch.ones_like(loss))]
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    check_device_status(DEV)
