"""RMS norm with the residual's addition, its gradients and its result in 8 bits, against the formula in 64 bits."""
import pytest
import torch

from warpconvnet_b200.nn.functional.rms_norm import quantize_rows, rms_norm, rms_norm_8bit

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24
# (rows, channels): one warp's rows and a block's, pieces of 16, 8 and 2 bytes, threads without a piece, rows behind the last block
SIZES = [(1, 1), (1, 256), (3, 8), (5, 13), (130, 32), (257, 100), (64, 96), (1000, 48), (33, 384), (9, 511), (7, 1024), (5, 1028), (6, 1031), (3, 2048), (2, 4100), (4, 8192),
         (2, 8191), (40001, 16)]


def half(dtype):
    return torch.finfo(dtype).eps / 2


def make(n, c, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + n + c)
    size = torch.exp(torch.randn(n, 1, generator=g))
    return [(torch.randn(n, c, generator=g) * size).to(dtype).to(DEV) for _ in range(4)] + [(torch.rand(c, generator=g) + 0.5).to(DEV)]


def norm64(h, w, eps):
    h = h.double()
    s = 1 / torch.sqrt(h.square().mean(1, keepdim=True) + eps)
    return h * s * (1.0 if w is None else w.double()), s


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("n,c", SIZES)
def test_against_the_formula(dtype, residual, n, c):
    x, r, dy, dh, w = make(n, c, dtype)
    if not residual:
        r = None
    leaves = [t.clone().requires_grad_(True) for t in (x, r, w) if t is not None]
    lx, lr, lw = (leaves[0], leaves[1], leaves[2]) if residual else (leaves[0], None, leaves[1])
    got = rms_norm(lx, lw, 1e-5, lr)
    y, h = got if residual else (got, lx)
    h0 = (x.float() + r.float()).to(dtype) if residual else x
    assert torch.equal(h.detach(), h0)
    ref, s = norm64(h0, w, 1e-5)
    # squares, their sum (some twenty roundings, halved by the root), root, quotient, two products; then the result's own rounding
    assert ((y.detach().double() - ref).abs() <= (half(dtype) + 16 * U) * ref.abs() + (2e-7 if dtype == torch.float16 else 0)).all()
    grads = torch.autograd.grad([y, h] if residual else [y], leaves, [dy, dh] if residual else [dy])
    xh, u = h0.double() * s, dy.double() * w.double()
    mean = (u * xh).mean(1, keepdim=True)
    dx = s * (u - xh * mean) + (dh.double() if residual else 0)
    terms = s * (u.abs() + xh.abs() * (u * xh).abs().mean(1, keepdim=True)) + (dh.double().abs() if residual else 0)
    assert grads[0].dtype == dtype and ((grads[0].double() - dx).abs() <= half(dtype) * dx.abs() + 48 * U * terms + (2e-7 if dtype == torch.float16 else 0)).all()
    if residual:
        assert torch.equal(grads[0], grads[1])
    dw, all_terms = (dy.double() * xh).sum(0), (dy.double() * xh).abs().sum(0)
    assert ((grads[-1].double() - dw).abs() <= 64 * U * all_terms).all()
    with torch.no_grad():
        again = rms_norm(x, w, 1e-5, r)
        assert torch.equal(again[0] if residual else again, y)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(*_again(lx, lw, lr, leaves, dy, dh)), grads))   # the same bits on every run


def _again(lx, lw, lr, leaves, dy, dh):
    got = rms_norm(lx, lw, 1e-5, lr)
    return (list(got), leaves, [dy, dh]) if lr is not None else ([got], leaves, [dy])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("n,c", SIZES)
def test_eight_bits(dtype, residual, n, c):
    x, r, _, _, w = make(n, c, dtype, 1)
    got = rms_norm_8bit(x, w, 1e-5, r if residual else None)
    h0 = (x.float() + r.float()).to(dtype) if residual else x
    if residual:
        assert torch.equal(got[2], h0)
    check_codes(got[0], got[1], norm64(h0, w, 1e-5)[0])
    check_codes(*quantize_rows(x), x.double())


def check_codes(q, scale, y):
    assert q.dtype == torch.float8_e4m3fn and scale.dtype == torch.float32
    t = (y.abs().amax(1) / 448).clamp(min=2.0 ** -126)
    assert ((scale.double() - t).abs() <= 24 * U * t).all()
    want = y / t[:, None]
    # half a step of e4m3: 2^-4 of the number, 2^-10 below 2^-6; the numbers themselves some roundings of fp32 off
    assert ((q.double() - want).abs() <= (2.0 ** -4 * want.abs()).clamp(min=2.0 ** -10) + 32 * U * want.abs()).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_boundaries(dtype):
    """Column blocks of wider buffers, starts on odd elements, rows in reverse, one row of many, transposed."""
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(50, 210, generator=g).to(dtype).to(DEV)
    w = torch.rand(64, generator=g).to(DEV)
    for view in (wide[:, 8:72], wide[:, 3:67], wide[::2, 64:128], wide[:1, 5:69], wide.t()[:64, :64].t()[:50], wide[:0, :64], wide[:1, :64].expand(30, 64)):
        want = norm64(view, w, 1e-6)[0]
        got = rms_norm(view, w)
        assert ((got.double() - want).abs() <= (half(dtype) + 16 * U) * want.abs() + (2e-7 if dtype == torch.float16 else 0)).all() and got.is_contiguous()
        got, h = rms_norm(view.contiguous(), w, residual=view)
        assert torch.equal(h, (view.float() + view.float()).to(dtype))
        q, scale = rms_norm_8bit(view, w)
        check_codes(q, scale, want)
    odd = torch.rand(65, generator=g).to(DEV)[1:]   # a weight that starts between boundaries
    assert torch.equal(rms_norm(wide[:, :64], odd), rms_norm(wide[:, :64], odd.clone()))
    assert torch.equal(rms_norm(wide[:, :64], w.to(torch.bfloat16)), rms_norm(wide[:, :64], w.to(torch.bfloat16).float()))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_are_not_numbers(dtype):
    """They stay with themselves; zeros are zeros; numbers whose squares pass the end of fp32 are normed like others."""
    x = torch.randn(40, 64, device=DEV).to(dtype)
    clean = rms_norm(x)
    bad = x.clone()
    bad[3, 5], bad[7, 0], bad[11] = float("nan"), float("inf"), 0.0
    y = rms_norm(bad)
    assert torch.isnan(y[3]).all() and torch.isnan(y[7, 0]) and not y[7, 1:].any() and not y[11].any()
    keep = [i for i in range(40) if i not in (3, 7, 11)]
    assert torch.equal(y[keep], clean[keep])
    q, scale = rms_norm_8bit(bad)
    assert torch.isnan(scale[[3, 7]]).all() and torch.isnan(q[[3, 7]].float()).all()
    assert float(scale[11]) == 2.0 ** -126 and not q[11].float().any()
    if dtype != torch.float16:
        huge = x * 1e30
        got, want = rms_norm(huge, residual=None), norm64(huge, None, 1e-6)[0]
        assert ((got.double() - want).abs() <= (half(dtype) + 20 * U) * want.abs()).all()
        leaf = huge.clone().requires_grad_(True)
        dx, = torch.autograd.grad(rms_norm(leaf), [leaf], torch.ones_like(leaf) * 1e25)
        assert torch.isfinite(dx).all() and dx.any()
    tiny = (torch.randn(5, 64, device=DEV) * 1e-44)
    q, scale = quantize_rows(tiny)
    assert (scale == 2.0 ** -126).all() and ((q.float() * scale[:, None] - tiny).abs() <= 2.0 ** -136).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("c", [13, 17, 96, 1031, 8192])
def test_rows_at_the_end_of_the_range(dtype, c):
    """Numbers as large as the type has, a mask's lowest value among them: their norm, its codes and its gradient are those of other rows."""
    g = torch.Generator().manual_seed(c)
    most = torch.finfo(dtype).max
    rows = torch.stack([torch.full((c,), most), torch.full((c,), -most), most * (torch.rand(c, generator=g) - 0.5) * 2, torch.randn(c, generator=g) * 1e36])
    x, dy = rows.to(dtype).to(DEV), (torch.randn(4, c, generator=g) * 1e30).to(dtype).to(DEV)
    w = (torch.rand(c, generator=g) + 0.5).to(DEV)
    ref, s = norm64(x, w, 1e-6)
    own = 16 * U + 2.0 ** -149 / s   # (and 1 / root mean square may be a number without all its places)
    leaf, lw = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = rms_norm(leaf, lw)
    assert ((y.detach().double() - ref).abs() <= (half(dtype) + own) * ref.abs()).all()
    if dtype == torch.bfloat16:   # (their errors, 2^-19 at most, lie far below half a step beside 1)
        assert (rms_norm(x[:1]) == 1).all() and (rms_norm(x[1:2]) == -1).all()
    assert torch.equal(rms_norm(x, residual=torch.zeros_like(x))[0], rms_norm(x))
    q, scale = rms_norm_8bit(x, w)
    t = ref.abs().amax(1, keepdim=True) / 448
    assert ((scale[:, None].double() - t).abs() <= (own + 4 * U) * t).all()
    # a code is off by half a step, 2^-4 of the number or 2^-10 of the scale at least
    assert ((q.double() * scale[:, None].double() - ref).abs() <= (2.0 ** -4 + 2 * own + 4 * U) * ref.abs() + 2.0 ** -10 * t).all()
    dx, dw = torch.autograd.grad(y, [leaf, lw], dy)
    xh, u = x.double() * s, dy.double() * w.double()
    want = s * (u - xh * (u * xh).mean(1, keepdim=True))
    terms = s * (u.abs() + xh.abs() * (u * xh).abs().mean(1, keepdim=True))
    assert ((dx.double() - want).abs() <= half(dtype) * want.abs() + (32 * U + 4 * own) * terms).all()
    each = dy.double() * xh
    assert ((dw.double() - each.sum(0)).abs() <= ((own + 16 * U) * each.abs()).sum(0)).all()


def test_an_eps_that_counts_beside_large_rows():
    x = torch.randn(9, 96, device=DEV) * 1e20
    ref = norm64(x, None, 1e38)[0]   # the mean of squares is some 1e40
    assert ((rms_norm(x, eps=1e38).double() - ref).abs() <= 16 * U * ref.abs()).all()
    x = torch.full((9, 1), 1.5e19, device=DEV)   # 2.25e38: with eps beyond the end of fp32
    ref = norm64(x, None, 3e38)[0]
    assert ((rms_norm(x, eps=3e38).double() - ref).abs() <= (16 * U) * ref.abs()).all()


def test_an_eps_beyond_fp32_is_refused():
    x = torch.ones(4, 8, device=DEV)
    for f in (rms_norm, rms_norm_8bit):
        for eps in (3.5e38, float("inf")):
            with pytest.raises(ValueError, match="eps"):
                f(x, eps=eps)
    assert torch.isfinite(rms_norm(x, eps=3.4e38)).all()


def test_gradient_against_differences():
    g = torch.Generator().manual_seed(3)
    x, r, w, dy, dh, u, v = (torch.randn(s, generator=g) for s in ((31, 24), (31, 24), (24,), (31, 24), (31, 24), (31, 24), (24,)))
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, r, w)]
    got = torch.autograd.grad(list(rms_norm(leaves[0], leaves[2], 1e-3, leaves[1])), leaves, [dy.to(DEV), dh.to(DEV)])

    def value(t):
        h = x.double() + r.double() + t * u.double()
        return float((norm64(h, w.double() + t * v.double(), 1e-3)[0] * dy.double()).sum() + (h * dh.double()).sum())
    t = 1e-4
    want = (8 * (value(t) - value(-t)) - (value(2 * t) - value(-2 * t))) / (12 * t)
    along = float((got[0].double().cpu() * u).sum() + (got[2].double().cpu() * v).sum())
    assert abs(along - want) <= 1e-5 * max(1.0, abs(want))   # (h in the kernel is rounded to fp32)


def test_gradients_of_some_inputs_and_results():
    x, r, dy, dh, w = make(70, 40, torch.bfloat16)
    lx, lr, lw = (t.clone().requires_grad_(True) for t in (x, r, w))
    every = torch.autograd.grad(list(rms_norm(lx, lw, 1e-6, lr)), [lx, lr, lw], [dy, dh])
    y, h = rms_norm(lx, w, 1e-6, r)
    assert torch.equal(torch.autograd.grad([y, h], [lx], [dy, dh])[0], every[0])
    y, h = rms_norm(x, lw, 1e-6, r)
    assert torch.equal(torch.autograd.grad([y], [lw], [dy])[0], every[2])
    y, h = rms_norm(lx, lw, 1e-6, lr)
    assert torch.equal(torch.autograd.grad([h], [lx, lr, lw], [dh], allow_unused=True)[0], dh)
    y, h = rms_norm(lx, None, 1e-6, lr)
    only = torch.autograd.grad([y], [lx], [dy])[0]
    summed = h.detach().requires_grad_(True)
    assert torch.equal(only, torch.autograd.grad(rms_norm(summed), [summed], [dy])[0])
    half_weight = w.to(torch.float16).requires_grad_(True)
    assert torch.autograd.grad(rms_norm(x, half_weight).sum(), [half_weight])[0].dtype == torch.float16
    empty = torch.zeros(0, 40, device=DEV, requires_grad=True)
    gx, gw = torch.autograd.grad(rms_norm(empty, lw).sum(), [empty, lw])
    assert gx.shape == (0, 40) and not gw.any()


def test_graphs_of_the_gradient_and_transforms():
    x, r, dy, dh, w = make(20, 16, torch.float32)
    lx, lr, lw = (t.clone().requires_grad_(True) for t in (x, r, w))
    first = torch.autograd.grad(list(rms_norm(lx, lw, 1e-3, lr)), [lx, lr, lw], [dy, dh], create_graph=True)
    plain = torch.autograd.grad(list(rms_norm(lx, lw, 1e-3, lr)), [lx, lr, lw], [dy, dh])
    assert all(torch.allclose(p, q, rtol=1e-4, atol=1e-5) for p, q in zip(first, plain))
    second = torch.autograd.grad((first[0] * dh).sum(), [lx, lw])
    h64, w64 = (x.double() + r.double()).requires_grad_(True), w.double().requires_grad_(True)
    g64, = torch.autograd.grad(norm64(h64, w64, 1e-3)[0], [h64], dy.double(), create_graph=True)
    want = torch.autograd.grad((g64 * dh.double()).sum(), [h64, w64])
    assert all(torch.allclose(p.double(), q, rtol=1e-4, atol=1e-5) for p, q in zip(second, want))
    value, tangent = torch.func.jvp(lambda t: rms_norm(t, w), (x,), (dy,))
    t64 = torch.func.jvp(lambda t: norm64(t, w, 1e-6)[0], (x.double(),), (dy.double(),))[1]
    assert torch.allclose(tangent.double(), t64, rtol=1e-4, atol=1e-5)


def test_captured_and_on_another_stream():
    x, r, dy, dh, w = make(5000, 96, torch.bfloat16)
    lx, lr, lw = (t.clone().requires_grad_(True) for t in (x, r, w))

    def step():
        y, h = rms_norm(lx, lw, 1e-6, lr)
        return [y.detach(), h.detach(), *torch.autograd.grad([y, h], [lx, lr, lw], [dy, dh]), *rms_norm_8bit(x, w)]
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = step()
    torch.cuda.current_stream().wait_stream(side)
    same = lambda a, b: all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(a, b))   # noqa: E731
    assert same(there, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        for t in got:
            t.zero_()
        graph.replay()
        assert same(got, want)


def test_refusals():
    x, w = torch.zeros(4, 8, device=DEV), torch.ones(8, device=DEV)
    for bad, error in ((lambda: rms_norm(x[0]), "N, C"), (lambda: rms_norm(x, w[:7]), "weight"), (lambda: rms_norm(x, w.int()), "weight"), (lambda: rms_norm(x, w.cpu()), "weight"),
                       (lambda: rms_norm(x, w, 0.0), "eps"), (lambda: rms_norm(x, w, float("nan")), "eps"), (lambda: rms_norm(x, residual=x[:3]), "residual"),
                       (lambda: rms_norm(x, residual=x.half()), "residual"), (lambda: rms_norm(x, residual=x.cpu()), "residual"),
                       (lambda: rms_norm(torch.zeros(1, 8193, device=DEV)), "8192"), (lambda: rms_norm(torch.zeros(3, 0, device=DEV)), "channels"),
                       (lambda: rms_norm_8bit(x, w.clone().requires_grad_(True)), "no_grad"), (lambda: quantize_rows(x.clone().requires_grad_(True)), "no_grad")):
        with pytest.raises(ValueError, match=error):
            bad()
    with pytest.raises(TypeError):
        rms_norm(x.double())
