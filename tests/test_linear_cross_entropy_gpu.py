"""Cross entropy of a linear layer without its logits, against the formula in 64 bits."""
import os
import subprocess
import sys

import pytest
import torch

from warpconvnet_b200 import LinearCrossEntropy, Voxels, linear_cross_entropy
from warpconvnet_b200._native import check_device_status, device_status

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
# a gradient in 16 bits is rounded twice (the logits' gradient and the result), each by at most 2^-11 / 2^-8 of a value and 0.6 of
# that in the mean; in fp32 sums of up to 128 products and of their sums
TOL = {torch.float32: 3e-6, torch.float16: 6e-4, torch.bfloat16: 5e-3}


def inputs(n, c, v, dtype, bias, seed=0, ignored=0.1):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(v, c, generator=g) / c ** 0.5
    labels = torch.randint(0, v, (n,), generator=g)
    x = torch.randn(n, c, generator=g) + 4 * torch.rand(n, 1, generator=g) * w[labels]
    labels[torch.rand(n, generator=g) < ignored] = -100
    b = torch.randn(v, generator=g) if bias else None
    return x.to(dtype), w.to(dtype), labels, None if b is None else b.to(dtype)


def losses(x, w, labels, b, ignore=-100):
    """Row losses in 64 bits, and which rows count."""
    z = x.double() @ w.double().t()
    z = z if b is None else z + b.double()
    counts = (labels != ignore) & (labels >= 0) & (labels < len(w))
    at = torch.where(counts, labels, 0)
    row = torch.logsumexp(z, 1) - z.gather(1, at[:, None])[:, 0]
    return torch.where(counts, row, 0.0), counts


def off(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).norm() / max(float(b.norm()), 1e-300))


SIZES = [(1, 8, 1), (1, 1, 2), (7, 3, 5), (127, 40, 20), (128, 64, 16), (129, 96, 200), (300, 100, 255), (1000, 33, 257), (513, 256, 256), (260, 264, 1000),
         (2000, 96, 20), (5000, 48, 513), (100, 512, 700), (640, 72, 3001), (20011, 32, 13), (1, 128, 5000), (50, 1000, 300)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("n,c,v", SIZES)
def test_against_the_formula(dtype, bias, n, c, v):
    x, w, labels, b = inputs(n, c, v, dtype, bias, seed=n + c + v, ignored=0.1 if n > 1 else 0.0)
    ref = [t.double().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    mine = [t.to(DEV).requires_grad_(True) if t is not None else None for t in (x, w, b)]
    row, counts = losses(ref[0], ref[1], labels, ref[2])
    grad_row = torch.randn(n, generator=torch.Generator().manual_seed(1))
    # a logit is a sum whose partial sums lose up to 2^-23 of themselves, C / 16 times
    room = 1.2e-7 * (2 + c / 16) * (1 + float((x.double().abs() @ w.double().abs().t()).max()))
    for reduction, want, grad in (("mean", row.sum() / counts.sum(), torch.tensor(3.0)), ("sum", row.sum(), torch.tensor(0.25)), ("none", row, grad_row)):
        got = linear_cross_entropy(mine[0], mine[1], labels.to(DEV), mine[2], reduction=reduction)
        assert got.dtype == torch.float32 and got.shape == want.shape
        assert float((got.detach().cpu().double() - want.detach()).abs().max()) <= room * (max(1, int(counts.sum())) if reduction == "sum" else 1)
        with torch.no_grad():
            assert torch.equal(linear_cross_entropy(mine[0], mine[1], labels.to(DEV), mine[2], reduction=reduction), got)
        some = [t for t in mine if t is not None]
        grads = torch.autograd.grad(got, some, grad.to(DEV), retain_graph=True)
        again = torch.autograd.grad(got, some, grad.to(DEV))
        wants = torch.autograd.grad(want, [t for t in ref if t is not None], grad.double(), retain_graph=True)
        for a, z, y, t in zip(grads, again, wants, some):
            assert a.dtype == t.dtype and a.shape == t.shape and torch.equal(a, z)
            if v > 1 and off(y.to(dtype), y) > TOL[dtype]:
                # fp16 below 2^-14: the formula's own value, rounded, is further off; a spacing of 2^-24 for each number
                assert float((a.cpu().double() - y).abs().max()) <= 2.0 ** -24 + TOL[dtype] * float(y.abs().max())
            elif v > 1:
                assert off(a, y) <= TOL[dtype]
            else:
                assert not a.any()   # one class: certain
    check_device_status(DEV)


@pytest.mark.parametrize("n,c,v", [(40000, 64, 8000), (60000, 96, 200), (60000, 72, 20), (50001, 128, 130), (30000, 160, 40), (100000, 32, 600)])
def test_many_pieces(n, c, v):
    """Rows and classes beyond one piece of the logits' gradient, and many tiles for each block."""
    x, w, labels, b = inputs(n, c, v, torch.bfloat16, True)
    mine = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    loss = linear_cross_entropy(mine[0], mine[1], labels.to(DEV), mine[2])
    grads = torch.autograd.grad(loss, mine)
    xd, wd, bd, ld = (t.to(DEV) for t in (x.double(), w.double(), b.double(), labels))
    p = torch.softmax(torch.addmm(bd, xd, wd.t()), 1)
    used = ld >= 0
    p[torch.arange(n, device=DEV)[used], ld[used]] -= 1
    p *= used[:, None] / used.sum()
    for a, y in zip(grads, (p @ wd, p.t() @ xd, p.sum(0))):
        assert off(a, y) <= TOL[torch.bfloat16]
    assert abs(float(loss.detach()) - float(losses(xd, wd, ld, bd)[0].sum() / used.sum())) < 1e-4


def test_gradient_against_differences():
    n, c, v = 40, 12, 17
    x, w, labels, b = inputs(n, c, v, torch.float32, True)
    g = torch.Generator().manual_seed(5)
    u = [torch.randn(t.shape, generator=g) for t in (x, w, b)]
    mine = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(linear_cross_entropy(mine[0], mine[1], labels.to(DEV), mine[2]), mine)
    slope = sum(float((a.cpu().double() * d.double()).sum()) for a, d in zip(grads, u))

    def loss(h):
        row, counts = losses(*(t.double() + h * d.double() for t, d in zip((x, w), u)), labels, b.double() + h * u[2].double())
        return float(row.sum() / counts.sum())
    h = 1e-5
    assert abs((loss(h) - loss(-h)) / (2 * h) - slope) <= 1e-5 * max(1.0, abs(slope))


@pytest.mark.parametrize("dtype", DTYPES)
def test_labels_that_do_not_count(dtype):
    x, w, labels, b = (t.to(DEV) for t in inputs(200, 32, 40, dtype, True))
    x, w, b = (t.requires_grad_(True) for t in (x, w, b))
    # none counts: the mean of nothing, gradients of zero
    loss = linear_cross_entropy(x, w, torch.full_like(labels, -100), b)
    assert torch.isnan(loss) and all(not t.any() for t in torch.autograd.grad(loss, [x, w, b]))
    assert float(linear_cross_entropy(x, w, torch.full_like(labels, -100), b, reduction="sum")) == 0.0
    # another number for them, which may be a class
    row = linear_cross_entropy(x, w, labels.clamp(min=3), b, ignore_index=3, reduction="none")
    want, counts = losses(x.detach().cpu(), w.detach().cpu(), labels.cpu().clamp(min=3), b.detach().cpu(), ignore=3)
    assert not row[~counts.to(DEV)].any() and off(row, want) <= 1e-5
    check_device_status(DEV)
    # no class of that number: reported, and as if it did not count
    wrong = labels.clone()
    wrong[0], wrong[1], wrong[2] = 40, -1, 1 << 40
    none = wrong.clone()
    none[:3] = -100
    for reduction in ("mean", "none"):
        got = linear_cross_entropy(x, w, wrong, b, reduction=reduction)
        with pytest.raises(RuntimeError):
            check_device_status(DEV)
        ref = linear_cross_entropy(x, w, none, b, reduction=reduction)
        assert torch.equal(got, ref)
        grads = [torch.autograd.grad(t.sum(), [x, w, b]) for t in (got, ref)]
        assert all(torch.equal(p, q) for p, q in zip(*grads))
    device_status(DEV).zero_()


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_what_is_no_number(dtype):
    n, c, v = 150, 32, 300
    x, w, labels, _ = inputs(n, c, v, dtype, False, ignored=0.0)
    labels[:] = 5
    labels[7], labels[9] = 290, 100
    b = torch.zeros(v)
    b[100:290] = float("-inf")   # classes that cannot be
    got = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    row = linear_cross_entropy(got[0], got[1], labels.to(DEV), got[2], reduction="none")
    want, _ = losses(x, w, labels, b)
    keep = torch.arange(n) != 9
    assert torch.isposinf(row[9]) and off(row.detach().cpu()[keep], want[keep]) <= 1e-5
    grad = torch.ones(n)
    grad[9] = 0.0
    dx, dw, db = torch.autograd.grad(row, got, grad.to(DEV))
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all() and not dw[100:290].any() and not db[100:290].any()
    # nothing can be: no probabilities
    row = linear_cross_entropy(got[0], got[1], labels.to(DEV), torch.full((v,), float("-inf"), device=DEV), reduction="none")
    assert torch.isnan(row).all()
    # a row that is no number is alone with it, and a row that does not count has no gradient whatever is in it
    bad = x.clone()
    bad[3, 4], bad[20, 1] = float("nan"), float("inf")
    used = labels.clone()
    used[50] = -100
    bad[50] = float("nan")
    xs = bad.to(DEV).requires_grad_(True)
    row = linear_cross_entropy(xs, w.to(DEV), used.to(DEV), reduction="none")
    (dx,) = torch.autograd.grad(row, [xs], torch.ones(n, device=DEV))
    fine = torch.ones(n, dtype=torch.bool)
    fine[[3, 20, 50]] = False
    clean = linear_cross_entropy(x.to(DEV), w.to(DEV), used.to(DEV), reduction="none")
    assert torch.isnan(row[[3, 20]]).all() and float(row[50]) == 0.0 and torch.equal(row.detach().cpu()[fine], clean.cpu()[fine])
    assert torch.isnan(dx[3]).all() and torch.isfinite(dx.cpu()[fine]).all() and not dx[50].any()
    check_device_status(DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [40, 300])
def test_gradients_that_are_no_numbers_stay_with_their_rows(dtype, v):
    x, w, labels, _ = (None if t is None else t.to(DEV) for t in inputs(200, 32, v, dtype, False, ignored=0.0))
    x = x.requires_grad_(True)
    grad = torch.randn(200, device=DEV)
    row = linear_cross_entropy(x, w, labels, reduction="none")
    (want,) = torch.autograd.grad(row, [x], grad, retain_graph=True)
    bad = grad.clone()
    bad[3], bad[70] = float("inf"), float("nan")
    (got,) = torch.autograd.grad(row, [x], bad, retain_graph=True)
    fine = torch.ones(200, dtype=torch.bool, device=DEV)
    fine[[3, 70]] = False
    # (the others are divided by the largest of them and multiplied again: two roundings of fp32, or of one in 16 bits otherwise)
    assert off(got[fine], want[fine]) <= TOL[dtype] and not torch.isfinite(got[3]).all() and torch.isnan(got[70]).all()
    (none,) = torch.autograd.grad(row, [x], torch.zeros_like(grad))
    assert not none.any()


def test_certain_rows_and_large_logits():
    """Losses that round to zero are not negative; logits of hundreds do not overflow."""
    for dtype in DTYPES:
        w = (torch.eye(64) * 20).to(dtype).to(DEV)
        x = (torch.eye(64).repeat(3, 1) * 20).to(dtype).to(DEV).requires_grad_(True)
        labels = torch.arange(64, device=DEV).repeat(3)
        row = linear_cross_entropy(x, w, labels, reduction="none")
        assert not row.any() and not torch.autograd.grad(row.sum(), [x])[0].any()
        row = linear_cross_entropy(x, w, (labels + 1) % 64, reduction="none")
        assert float((row - 400).abs().max()) <= 1e-3


@pytest.mark.parametrize("dtype", DTYPES)
def test_any_strides_and_addresses(dtype):
    n, c, v = 300, 40, 130
    x, w, labels, b = (t.to(DEV) for t in inputs(n, c, v, dtype, True))
    want = None
    wide_x, wide_w = torch.zeros(n, 3 * c, dtype=dtype, device=DEV), torch.zeros(v, 2 * c + 3, dtype=dtype, device=DEV)
    wide_x[:, c:2 * c], wide_w[:, 3:3 + c] = x, w
    odd = torch.cat([x.new_zeros(1), x.flatten()])[1:].view(n, c)
    labels2 = torch.stack([labels, labels], 1)[:, 0]
    bias2 = torch.stack([b, b], 1)[:, 0]
    for xs, ws, ls, bs in ((x, w, labels, b), (wide_x[:, c:2 * c], w, labels2, bias2), (odd, wide_w[:, 3:3 + c], labels.int(), b),
                           (x.t().contiguous().t(), w.t().contiguous().t(), labels, b)):
        xs, ws, bs = (t.detach().requires_grad_(True) for t in (xs, ws, bs))
        loss = linear_cross_entropy(xs, ws, ls, bs)
        got = [loss, *torch.autograd.grad(loss, [xs, ws, bs])]
        want = want or got
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("which", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (0, 1, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_only_what_is_wanted(which, dtype):
    x, w, labels, b = (t.to(DEV) for t in inputs(500, 64, 90, dtype, True))
    full = [t.detach().requires_grad_(True) for t in (x, w, b)]
    some = [t.detach().requires_grad_(bool(k)) for t, k in zip((x, w, b), which)]
    want = torch.autograd.grad(linear_cross_entropy(full[0], full[1], labels, full[2]), full)
    got = torch.autograd.grad(linear_cross_entropy(some[0], some[1], labels, some[2]), [t for t in some if t.requires_grad])
    assert all(torch.equal(p, q) for p, q in zip(got, [t for t, k in zip(want, which) if k]))


def test_inputs_that_are_broadcast():
    x, w, labels, b = (t.to(DEV) for t in inputs(64, 32, 20, torch.float32, True))
    row = x[:1].clone().requires_grad_(True)
    (got,) = torch.autograd.grad(linear_cross_entropy(row.expand(64, 32), w, labels, b), [row])
    full = row.detach().repeat(64, 1).requires_grad_(True)
    (want,) = torch.autograd.grad(linear_cross_entropy(full, w, labels, b), [full])
    assert got.shape == (1, 32) and off(got, want.sum(0, keepdim=True)) <= 1e-6


def test_no_rows():
    w = torch.randn(5, 8, device=DEV, requires_grad=True)
    x, labels = torch.zeros(0, 8, device=DEV, requires_grad=True), torch.zeros(0, dtype=torch.int64, device=DEV)
    assert torch.isnan(linear_cross_entropy(x, w, labels)) and float(linear_cross_entropy(x, w, labels, reduction="sum")) == 0
    assert linear_cross_entropy(x, w, labels, reduction="none").shape == (0,)
    dx, dw = torch.autograd.grad(linear_cross_entropy(x, w, labels, reduction="sum"), [x, w])
    assert dx.shape == (0, 8) and not dw.any()


def test_second_derivatives():
    x, w, labels, _ = inputs(30, 8, 11, torch.float32, False)
    a, r = (t.clone().requires_grad_(True) for t in (x.to(DEV), x.double()))
    (ga,) = torch.autograd.grad(linear_cross_entropy(a, w.to(DEV), labels.to(DEV)), [a], create_graph=True)
    row, counts = losses(r, w, labels, None)
    (gr,) = torch.autograd.grad(row.sum() / counts.sum(), [r], create_graph=True)
    (gga,), (ggr,) = torch.autograd.grad(ga.square().sum(), [a]), torch.autograd.grad(gr.square().sum(), [r])
    assert off(ga, gr) <= 1e-5 and off(gga, ggr) <= 1e-5


def test_labels_of_no_class_in_a_graph_of_the_gradient():
    x, w, labels, _ = (None if t is None else t.to(DEV) for t in inputs(30, 8, 11, torch.float32, False))
    wrong = labels.clone()
    wrong[0] = 11
    labels[0] = -100
    x = x.requires_grad_(True)
    grads = [torch.autograd.grad(linear_cross_entropy(x, w, t), [x], create_graph=True)[0] for t in (wrong, labels)]
    assert torch.equal(*grads)
    device_status(DEV).zero_()


def test_captured_and_on_a_stream_of_its_own():
    x, w, labels, b = (t.to(DEV) for t in inputs(3000, 64, 500, torch.bfloat16, True))
    x, w = x.requires_grad_(True), w.requires_grad_(True)

    def step():
        loss = linear_cross_entropy(x, w, labels, b)
        return [loss.detach(), *torch.autograd.grad(loss, [x, w])]
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        for t in got:
            t.zero_()
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_the_first_thing_that_a_backward_thread_does():
    """In a process of its own: the gradient's launch is the first CUDA call of autograd's thread."""
    code = ("import torch\nfrom warpconvnet_b200 import linear_cross_entropy\n"
            "x = torch.randn(2000, 96, device='cuda').bfloat16().requires_grad_(True)\nw = torch.randn(20, 96, device='cuda').bfloat16()\n"
            "loss = linear_cross_entropy(x, w, torch.zeros(2000, dtype=torch.int64, device='cuda'))\n"
            "assert torch.isfinite(torch.autograd.grad(loss, [x], torch.ones((), device='cuda'))[0]).all()\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_module_on_a_geometry_and_under_autocast():
    torch.manual_seed(0)
    n = 300
    vox = Voxels(torch.arange(3 * n, dtype=torch.int32, device=DEV).view(n, 3), torch.randn(n, 32, device=DEV), offsets=torch.tensor([0, n]))
    head, labels = LinearCrossEntropy(32, 21).to(DEV), torch.randint(0, 21, (n,), device=DEV)
    loss = head(vox, labels)
    want = torch.nn.functional.cross_entropy(head.logits(vox), labels)
    assert abs(float(loss) - float(want)) <= 1e-5
    with torch.autocast("cuda", dtype=torch.bfloat16):
        low = head(vox, labels)
    low.backward()
    assert abs(float(low) - float(want)) <= 2e-2 and head.weight.grad.dtype == torch.float32 and head.bias.grad.dtype == torch.float32


def test_refusals():
    x, w, labels, b = (t.to(DEV) for t in inputs(10, 8, 5, torch.float32, True))
    for args, kw in (((x, w[:, :4], labels), {}), ((x[0], w, labels), {}), ((x, w, labels[:4]), {}), ((x, w, labels.float()), {}), ((x, w, labels, b[:2]), {}),
                     ((x.cpu(), w, labels), {}), ((x, w.cpu(), labels), {}), ((x, w, labels.cpu()), {}), ((x, w, labels, b.cpu()), {}),
                     ((x, w[:0], labels), {}), ((x, w, labels), {"reduction": "max"})):
        with pytest.raises(ValueError):
            linear_cross_entropy(*args, **kw)
    for args in ((x.half(), w, labels), (x.double(), w.double(), labels), (x, w, labels, b.double())):
        with pytest.raises(TypeError):
            linear_cross_entropy(*args)
    with pytest.raises(ValueError):
        LinearCrossEntropy(4, 5, reduction="max")
