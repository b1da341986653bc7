"""Row losses of the linear cross entropy and their gradients, where rows have weights of unlike size."""
import pytest
import torch

from warpconvnet_b200 import linear_cross_entropy

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
# as for the mean: two roundings to 16 bits (the logits' gradient, the result), 0.6 of each in the mean; fp32: sums of 128 products
TOL = {torch.float32: 3e-6, torch.float16: 6e-4, torch.bfloat16: 5e-3}
SIZES = [(300, 64, 40), (500, 96, 700), (300, 512, 300), (200, 40, 256)]   # a kernel for each: few classes, many, wide rows


def off(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).norm() / max(float(b.norm()), 1e-300))


def problem(n, c, v, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(v, c, generator=g) / c ** 0.5
    labels = torch.randint(0, v, (n,), generator=g)
    x = torch.randn(n, c, generator=g) + 2 * torch.rand(n, 1, generator=g) * w[labels]
    return x.to(dtype), w.to(dtype), labels, torch.randn(v, generator=g).to(dtype)


def exact(x, w, labels, b, grad, ignore=-100):
    """Gradients of x, w and the bias in 64 bits."""
    x, w, b = (t.double() for t in (x, w, b))
    p = torch.softmax(x @ w.t() + b, 1)
    counts = labels != ignore
    p[torch.arange(len(x))[counts], labels[counts]] -= 1
    p = torch.where(counts[:, None], p * grad.double()[:, None], 0.0)
    return p @ w, p.t() @ x, p.sum(0)


def gradients(x, w, labels, b, grad, wanted=(0, 1, 2)):
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    row = linear_cross_entropy(leaves[0], leaves[1], labels.to(DEV), leaves[2], reduction="none")
    return torch.autograd.grad(row, [leaves[i] for i in wanted], grad.to(DEV))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,c,v", SIZES)
def test_a_row_of_great_weight_leaves_the_others_their_gradients(dtype, n, c, v):
    x, w, labels, b = problem(n, c, v, dtype)
    grad = torch.ones(n)
    grad[7] = 2.0 ** 40   # (in fp16 its own gradient is beyond the type)
    want = exact(x, w, labels, b, grad)
    others = torch.arange(n) != 7
    for wanted in ((0,), (0, 1, 2)):
        dx = gradients(x, w, labels, b, grad, wanted)[0].cpu()
        assert off(dx[others], want[0][others]) <= TOL[dtype]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,c,v", SIZES)
def test_weights_of_unlike_size(dtype, n, c, v):
    """Weights over 20 octaves.  Each row's gradient over its weight is as exact as any other's."""
    x, w, labels, b = problem(n, c, v, dtype, seed=1)
    grad = torch.exp2(10.0 - torch.arange(n) % 21) * torch.where(torch.arange(n) % 2 == 0, 1.0, -1.0)
    want = exact(x, w, labels, b, grad)
    got = gradients(x, w, labels, b, grad)
    dx = got[0].double().cpu() / grad[:, None]
    least = 2.0 ** -24 / grad.abs().double()[:, None] if dtype == torch.float16 else torch.zeros(n, 1, dtype=torch.float64)   # fp16's spacing below 2^-14
    off_by = (dx - want[0] / grad[:, None]).abs()
    assert float((off_by - least).clamp(min=0).norm() / (want[0] / grad[:, None]).norm()) <= TOL[dtype]
    assert off(got[1], want[1]) <= TOL[dtype] and off(got[2], want[2]) <= TOL[dtype]
    alone = gradients(x, w, labels, b, grad, (1, 2))
    assert torch.equal(alone[0], got[1]) and torch.equal(alone[1], got[2])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,c,v", SIZES)
def test_weights_of_rows_that_do_not_count(dtype, n, c, v):
    """Whatever they are, also far above the others."""
    x, w, labels, b = problem(n, c, v, dtype, seed=2)
    labels[5], labels[60] = -100, -100
    grad = torch.randn(n, generator=torch.Generator().manual_seed(3))
    clean = gradients(x, w, labels, b, grad)
    want = exact(x, w, labels, b, grad)
    grad[5], grad[60] = 2.0 ** 60, -1e30
    got = gradients(x, w, labels, b, grad)
    assert all(off(p, q) <= TOL[dtype] for p, q in zip(got, want))
    assert all(torch.equal(p, q) for p, q in zip(got, clean))


def test_row_losses_hold_no_more_than_themselves():
    x, w, labels, b = (t.to(DEV) for t in problem(1000, 64, 40, torch.bfloat16))
    for rows in (linear_cross_entropy(x, w, labels, b, reduction="none"), linear_cross_entropy(x.requires_grad_(True), w, labels, b, reduction="none").detach()):
        assert rows.untyped_storage().nbytes() == 4 * 1000
