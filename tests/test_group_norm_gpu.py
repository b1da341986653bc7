"""Group norm per scene with its activation against the formula in 64 bits."""
import pytest
import torch

from warpconvnet_b200 import SegmentedGroupNorm, Sequential, SparseConv3d, Voxels, segmented_group_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# fp32: a handful of roundings (and an exponential) of 2^-24 each; 16 bits: one rounding, at most 2^-11 / 2^-8 of a value,
# about 0.6 of that in the mean
TOL = {torch.float32: 2e-6, torch.float16: 4e-4, torch.bfloat16: 3e-3}
ACTS = [None, "relu", "silu", "gelu"]


def act64(z, act):
    if act == "relu":
        return torch.where((z > 0) | torch.isnan(z), z, 0.0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z / 2 ** 0.5))
    return z


def formula(x, offsets, groups, w, b, eps, act):
    """(y, rows' 1 / std) in 64 bits."""
    out, r = torch.zeros_like(x), torch.zeros_like(x)
    for lo, hi in zip(offsets, offsets[1:]):
        if hi > lo:
            xs = x[lo:hi].view(hi - lo, groups, -1)
            mean = xs.mean((0, 2), keepdim=True)
            rstd = 1 / torch.sqrt((xs - mean).square().mean((0, 2), keepdim=True) + eps)
            out[lo:hi] = ((xs - mean) * rstd).reshape(hi - lo, -1)
            r[lo:hi] = rstd.expand_as(xs).reshape(hi - lo, -1)
    return act64(out * w + b, act), r


def off(a, b, scale=None):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).norm() / max(float(b.norm()), float(scale.detach().norm()) if scale is not None else 0.0, 1e-300))


CASES = [([0, 1], 8, 1), ([0, 2, 2, 3], 6, 3), ([0, 0, 500, 500], 32, 4), ([0, 33, 1000, 1257], 24, 24), ([0, 700], 5, 1), ([0, 10, 300], 257, 257),
         ([0, 4097, 5000], 96, 8), ([0, 300, 40001], 64, 16), ([0, 129], 1024, 32), ([0, 50], 4096, 2), (list(range(0, 3003, 3)), 16, 4), ([0, 37], 2056, 8)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("offsets,c,groups", CASES, ids=[f"{len(o) - 1}x{o[-1]}_c{c}_g{g}" for o, c, g in CASES])
def test_against_the_formula(dtype, act, offsets, c, groups):
    g = torch.Generator().manual_seed(c + groups)
    n = offsets[-1]
    x0 = (torch.randn(n, c, generator=g) + 3 * torch.randn(c, generator=g)).to(dtype)
    dy = torch.randn(n, c, generator=g).to(dtype)
    w0, b0 = torch.rand(c, generator=g) + 0.5, torch.randn(c, generator=g) * 0.5
    x, w, b = (t.to(DEV).requires_grad_(True) for t in (x0.clone(), w0, b0))
    y = segmented_group_norm(x, torch.tensor(offsets), groups, w, b, 1e-3, act)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy.to(DEV))
    xr, wr, br = (t.double().requires_grad_(True) for t in (x0, w0, b0))
    yr, rstd = formula(xr, offsets, groups, wr, br, 1e-3, act)
    dxr, dwr, dbr = torch.autograd.grad(yr, [xr, wr, br], dy.double())
    assert y.dtype == dtype and dx.dtype == dtype
    assert off(y, yr) <= TOL[dtype]
    # the gradient of x is a difference: measured against its first term; sums of fp32 numbers against their terms
    assert off(dx, dxr, dy.double() * wr * rstd) <= TOL[dtype]
    terms = dy.double().norm(dim=0)
    assert off(dw, dwr, terms) <= 4e-6 and off(db, dbr, terms) <= 4e-6
    with torch.no_grad():
        assert torch.equal(segmented_group_norm(x, offsets, groups, w, b, 1e-3, act), y)   # the same bits on every run


@pytest.mark.parametrize("act", ACTS)
def test_gradient_against_differences(act):
    g = torch.Generator().manual_seed(3)
    offsets, n, c = [0, 20, 57], 57, 12
    x, u = torch.randn(n, c, generator=g), torch.randn(n, c, generator=g)
    w, b, dy = torch.rand(c, generator=g) + 0.5, torch.randn(c, generator=g), torch.randn(n, c, generator=g)
    dw, db = torch.randn(c, generator=g), torch.randn(c, generator=g)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    y = segmented_group_norm(leaves[0], offsets, 4, leaves[1], leaves[2], 1e-5, act)
    grads = torch.autograd.grad(y, leaves, dy.to(DEV))
    slope = sum(float((a.double().cpu() * d.double()).sum()) for a, d in zip(grads, (u, dw, db)))

    def loss(h):
        y, _ = formula(x.double() + h * u.double(), offsets, 4, w.double() + h * dw.double(), b.double() + h * db.double(), 1e-5, act)
        return float((y * dy.double()).sum())
    h = 1e-6
    # the second difference over h, an fp32 gradient, and a ReLU's kinks that lie within h (none here)
    assert abs((loss(h) - loss(-h)) / (2 * h) - slope) <= 1e-4 * max(1.0, abs(slope))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_rows_of_a_wider_buffer_and_of_any_address(dtype):
    """Column blocks on and off 16-byte boundaries, a transposed matrix, and a broadcast gradient."""
    n, c, offsets = 300, 32, [0, 100, 300]
    g = torch.Generator().manual_seed(0)
    wide = torch.randn(n, 100, generator=g).to(dtype).to(DEV)
    w, b = torch.rand(c, generator=g).to(DEV), torch.randn(c, generator=g).to(DEV)
    for x in (wide[:, 8:8 + c], wide[:, 3:3 + c], wide[:, :c].t().contiguous().t(), wide[::2, :c].repeat(2, 1)[:n]):
        results = []
        for rows in (x, x.contiguous().clone()):
            rows = rows.detach().requires_grad_(True)
            y = segmented_group_norm(rows, offsets, 4, w, b, activation="silu")
            results.append([y, *torch.autograd.grad(y.sum(), [rows])])   # (the gradient of a sum is one number, expanded)
        assert all(off(p, q) <= TOL[dtype] for p, q in zip(*results))


def test_precision_beside_a_large_mean_and_a_row_far_away():
    g = torch.Generator().manual_seed(0)
    for n in (1000, 60001):
        x = torch.randn(n, 16, generator=g) + 1000.0
        want, _ = formula(x.double(), [0, n], 4, 1.0, 0.0, 1e-5, None)
        # the mean's own rounding is 2^-25 * 1000 = 3e-5 of the spread
        assert off(segmented_group_norm(x.to(DEV), None, 4), want) <= 6e-5
        for row in (0, n // 2, n - 1):
            x = torch.randn(n, 16, generator=g)
            x[row] = 1000.0
            want, _ = formula(x.double(), [0, n], 4, 1.0, 0.0, 1e-5, None)
            got = segmented_group_norm(x.to(DEV), None, 4).cpu()
            keep = torch.arange(n) != row
            assert off(got, want) <= 2e-6 and off(got[keep], want[keep]) <= 1e-5


def test_constant_groups_and_what_is_no_number():
    x = torch.full((100, 8), 2.5, device=DEV)
    assert torch.equal(segmented_group_norm(x, [0, 1, 100], 2), torch.zeros_like(x))
    x = torch.randn(100, 8, device=DEV)
    clean = segmented_group_norm(x, [0, 40, 100], 2, activation="relu")
    for bad in (float("nan"), float("inf"), float("-inf")):
        y = x.clone()
        y[50, 6] = bad
        got = segmented_group_norm(y, [0, 40, 100], 2, activation="relu")
        assert torch.isnan(got[40:, 4:]).all()
        assert torch.equal(got[:40], clean[:40]) and torch.equal(got[40:, :4], clean[40:, :4])


def test_no_rows():
    x = torch.zeros(0, 8, device=DEV, requires_grad=True)
    w = torch.ones(8, device=DEV, requires_grad=True)
    for offsets in ([0], [0, 0], None):
        y = segmented_group_norm(x, offsets, 2, w)
        dx, dw = torch.autograd.grad(y.sum(), [x, w])
        assert y.shape == (0, 8) and dx.shape == (0, 8) and torch.equal(dw, torch.zeros(8, device=DEV))


@pytest.mark.parametrize("params", [torch.float32, torch.float16])
@pytest.mark.parametrize("which", [(True, False, False), (False, True, False), (False, False, True), (True, False, True)])
def test_only_what_is_wanted(params, which):
    g = torch.Generator().manual_seed(0)
    x, w, b = torch.randn(500, 16, generator=g).half(), torch.rand(16, generator=g).to(params), torch.randn(16, generator=g).to(params)
    leaves = [t.to(DEV).requires_grad_(need) for t, need in zip((x, w, b), (True, True, True))]
    some = [t.detach().requires_grad_(need) for t, need in zip(leaves, which)]
    full = torch.autograd.grad(segmented_group_norm(leaves[0], None, 4, leaves[1], leaves[2], activation="gelu").float().square().sum(), leaves)
    part = torch.autograd.grad(segmented_group_norm(some[0], None, 4, some[1], some[2], activation="gelu").float().square().sum(),
                               [t for t in some if t.requires_grad])
    want = [t for t, need in zip(full, which) if need]
    assert all(a.dtype == b.dtype and torch.equal(a, b) for a, b in zip(part, want))


def test_second_derivatives_and_function_transforms():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(50, 8, generator=g, dtype=torch.float64)
    xs = x.float().to(DEV).requires_grad_(True)
    xd = x.clone().requires_grad_(True)
    y, yd = segmented_group_norm(xs, [0, 20, 50], 2, activation="silu"), formula(xd, [0, 20, 50], 2, 1.0, 0.0, 1e-5, "silu")[0]
    (gx,), (gd,) = torch.autograd.grad(y.pow(3).sum(), [xs], create_graph=True), torch.autograd.grad(yd.pow(3).sum(), [xd], create_graph=True)
    (ggx,), (ggd,) = torch.autograd.grad(gx.square().sum(), [xs]), torch.autograd.grad(gd.square().sum(), [xd])
    assert off(gx, gd) <= 1e-5 and off(ggx, ggd) <= 1e-4
    fn = lambda t: segmented_group_norm(t, [0, 20, 50], 2, activation="silu")   # noqa: E731
    tangent = torch.ones_like(xs)
    _, jvp = torch.func.jvp(fn, (xs.detach(),), (tangent,))
    back = torch.autograd.grad(fn(xs).sum(), [xs])[0]
    assert abs(float(jvp.sum()) - float(back.sum())) <= 1e-3


def test_captured():
    x = torch.randn(5000, 32, device=DEV)
    want = segmented_group_norm(x, [0, 100, 5000], 4, activation="relu")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = segmented_group_norm(x, torch.tensor([0, 100, 5000]), 4, activation="relu")
    y.zero_()
    graph.replay()
    assert torch.equal(y, want)


def test_on_a_stream_of_its_own():
    x = torch.randn(200000, 64, device=DEV)
    want = segmented_group_norm(x, None, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = segmented_group_norm(x, None, 4)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want)


def test_module_in_a_sequence():
    g = torch.Generator().manual_seed(0)
    xyz = torch.unique(torch.randint(0, 16, (2000, 3), generator=g, dtype=torch.int32), dim=0)
    n = len(xyz)
    vox = Voxels(xyz.to(DEV), torch.randn(n, 16, generator=g).to(DEV), offsets=torch.tensor([0, n // 3, n]))
    seq = Sequential(SparseConv3d(16, 32, 3, bias=False), SegmentedGroupNorm(8, 32, activation="relu")).to(DEV)
    y = seq(vox).feature_tensor
    want = segmented_group_norm(seq[0](vox).feature_tensor, vox.offsets, 8, seq[1].weight, seq[1].bias, activation="relu")
    assert off(y, want) <= 1e-6
    y.square().sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in seq.parameters())
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert seq(vox).feature_tensor.dtype == torch.bfloat16


def test_refusals():
    x = torch.zeros(10, 8, device=DEV)
    for args, kw in (((x, [0, 9], 2), {}), ((x, [1, 10], 2), {}), ((x, [0, 7, 3, 10], 2), {}), ((x, [0, 10], 3), {}), ((x, [0, 10], 0), {}),
                     ((x, [], 2), {}), ((x, torch.tensor([0.0, 10.0]), 2), {}), ((x.view(2, 5, 8), [0, 10], 2), {}), ((x.cpu(), [0, 10], 2), {}),
                     ((x, [0, 10], 2), {"activation": "tanh"}), ((x, [0, 10], 2, x[0, :4]), {}), ((x, [0, 10], 2, x[0].cpu()), {}),
                     ((x, [0, 10], 2, x[0].int()), {}), ((torch.zeros(3, 5000, device=DEV), [0, 3], 1), {})):
        with pytest.raises(ValueError):
            segmented_group_norm(*args, **kw)
    with pytest.raises(TypeError):
        segmented_group_norm(x.double(), [0, 10], 2)
    with pytest.raises(ValueError):
        SegmentedGroupNorm(3, 8)
    with pytest.raises(ValueError):
        SegmentedGroupNorm(2, 8, activation="tanh")
