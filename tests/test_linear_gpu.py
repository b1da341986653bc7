"""Linear layers with bias, activation, dropout and residual, and their gradients, against the formula in 64 bits."""
import pytest
import torch

from warpconvnet_b200._native import check_device_status, device_status
from warpconvnet_b200._native import dtype_code, query_bytes
from warpconvnet_b200.nn.functional.dropout import dropout
from warpconvnet_b200.nn.functional.linear import linear, linear_8bit
from warpconvnet_b200.nn.functional.rms_norm import quantize_rows

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
ACTS = [None, "relu", "silu", "gelu"]
U = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def normal64(z):
    """(torch.special.ndtr gives 0 on a GPU from -8.34 on, where it is 3.6e-17.)"""
    return 0.5 * torch.special.erfc(z * -0.5 ** 0.5)


def act64(z, act):
    """act(z) and its derivative."""
    one = torch.ones_like(z)
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s)
    if act == "gelu":
        p = normal64(z)
        return z * p, p + z * torch.exp(-z * z / 2) * 0.3989422804014327
    return z, one


def make(n, k, m, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + n + 3 * k + 7 * m)
    x = torch.randn(n, k, generator=g) * torch.exp(0.5 * torch.randn(n, 1, generator=g))
    w, b = torch.randn(m, k, generator=g) / k ** 0.5, torch.randn(m, generator=g)
    r, dy = torch.randn(n, m, generator=g), torch.randn(n, m, generator=g)
    return [t.to(dtype).to(DEV) for t in (x, w, b, r, dy)]


def off(a, b):
    return float((a.double() - b).norm() / b.norm().clamp(min=1e-300))


def sums(k, terms, dtype):
    """What a sum of k products may be off: fp32 in chains of 128; on the tensor cores 16 products at a time with sums cut, not rounded."""
    return (128 + k / 128 + 4) * U * terms if dtype == torch.float32 else (k / 16 + 8) * 2 * U * terms


def within(got, want, bound):
    d = (got.double() - want).abs()
    assert (d <= bound).all(), (float(d.max()), float((d / bound.clamp(min=1e-300)).max()))


# tiles cut in all directions, one row, one column, one input; columns that stay in shared memory and that do not; several groups of
# columns; pitches that TMA does not take (outputs that are no multiple of 8); inputs that have to be copied
SIZES = [(1, 1, 1), (1, 256, 1024), (3, 8, 20), (130, 96, 384), (257, 100, 13), (64, 40, 33), (128, 64, 32), (300, 384, 96), (700, 256, 1000), (200, 1024, 520), (5, 2000, 7),
         (2049, 64, 256), (1000, 33, 129), (9, 520, 72), (513, 160, 1)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act,residual,p,bias", [(None, False, 0.0, True), (None, True, 0.0, False), ("relu", True, 0.3, True), ("silu", False, 0.0, True), ("gelu", False, 0.1, True),
                                                 ("gelu", True, 0.0, False), (None, True, 0.5, True)])
@pytest.mark.parametrize("n,k,m", SIZES)
def test_against_the_formula(dtype, act, residual, p, bias, n, k, m):
    x, w, b, r, dy = make(n, k, m, dtype)
    b, r = b if bias else None, r if residual else None
    lx, lw, lb, lr = (t if t is None else t.clone().requires_grad_(True) for t in (x, w, b, r))
    y = linear(lx, lw, lb, act, lr, p, seed=5)
    leaves = [t for t in (lx, lw, lb, lr) if t is not None]
    got = dict(zip([s for s, t in zip("xwbr", (lx, lw, lb, lr)) if t is not None], torch.autograd.grad(y, leaves, dy)))
    X, W = x.double(), w.double()
    z = X @ W.t() + (b.double() if bias else 0)
    keep = dropout(torch.ones(n, m, device=DEV), p, 5).double() if p else torch.ones(n, m, device=DEV, dtype=torch.float64)   # (factor and all, rounded to fp32)
    a, slope = act64(z, act)
    want = a * keep + (r.double() if residual else 0)
    # the sum; bias, activation (within 2e-5 of its value in 16 bits, and of its slope's largest value), factor and residual; the rounding
    z_off = sums(k, X.abs() @ W.abs().t(), dtype) + 2 * U * z.abs()
    fine = 16 * U if dtype == torch.float32 else 2e-5
    tiny = 6e-8 if dtype == torch.float16 else 0
    within(y.detach(), want, half(dtype) * want.abs() + keep * (1.13 * z_off + fine * a.abs() + 1e-11) + 4 * U * want.abs() + tiny)
    assert off(y.detach(), want) <= (half(dtype) if dtype != torch.float32 else 2e-6)
    dz = dy.double() * keep * slope
    direct = act is None and not p
    # of dz: what z is off times the second derivative (a step of relu's where z may have either sign), its rounding
    dz_off = dy.double().abs() * keep * ((1.13 * z_off + 2 * fine) if act in ("silu", "gelu") else (z.abs() <= z_off).double() if act == "relu" else 0 * z)
    dz_off = dz_off + (0 if direct else half(dtype) * dz.abs() + 4 * U * dz.abs() + tiny)
    within(got["x"], dz @ W, half(dtype) * (dz @ W).abs() + sums(m, dz.abs() @ W.abs(), dtype) + dz_off @ W.abs() + tiny)
    within(got["w"], dz.t() @ X, half(dtype) * (dz.t() @ X).abs() + sums(n, dz.abs().t() @ X.abs(), dtype) + dz_off.t() @ X.abs() + tiny)
    if bias:
        within(got["b"], dz.sum(0), half(dtype) * dz.sum(0).abs() + sums(n, dz.abs().sum(0), dtype) + dz_off.sum(0) + tiny)
    if residual:
        assert torch.equal(got["r"], dy)
    with torch.no_grad():
        assert torch.equal(linear(x, w, b, act, r, p, torch.tensor([5], device=DEV)), y)
    again = torch.autograd.grad(linear(lx, lw, lb, act, lr, p, seed=5), leaves, dy)
    assert all(torch.equal(s, t) for s, t in zip(again, got.values()))   # the same bits on every run
    check_device_status(DEV)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", ACTS)
def test_mean_errors_are_those_of_the_roundings(dtype, act):
    """A rounding's error is 0.58 of half a step in the mean at most, two of them 0.82."""
    n, k, m = 3000, 192, 264
    x, w, b, r, dy = make(n, k, m, dtype)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = linear(*leaves, act)
    got = torch.autograd.grad(y, leaves, dy)
    z = x.double() @ w.double().t() + b.double()
    a, slope = act64(z, act)
    dz = dy.double() * slope
    assert off(y.detach(), a) <= 0.6 * half(dtype)
    assert all(off(g, t) <= 0.85 * half(dtype) for g, t in zip(got, (dz @ w.double(), dz.t() @ x.double(), dz.sum(0))))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_activations_over_their_whole_range(dtype, act):
    """z from the bias alone: values and slopes at every place, infinities and what is no number."""
    z = torch.cat([torch.linspace(-12, 12, 4001), torch.logspace(-6, 4, 300), -torch.logspace(-6, 4, 300)]).to(dtype).to(DEV)
    x, w = torch.zeros(1, 8, dtype=dtype, device=DEV), torch.zeros(len(z), 8, dtype=dtype, device=DEV)
    b = z.clone().requires_grad_(True)
    y = linear(x, w, b, act)
    slope_got, = torch.autograd.grad(y, [b], torch.ones_like(y))
    value, slope = act64(z.double(), act)
    # (a slope's cancelling terms are 1.13 at most)
    within(y[0].detach(), value, (half(dtype) + 2e-5) * value.abs() + 1e-10 + (6e-8 if dtype == torch.float16 else 0))
    within(slope_got, slope, (2 * half(dtype) + 2e-5) * slope.abs() + 2e-5)
    odd = torch.tensor([float("inf"), float("nan")], dtype=dtype, device=DEV)
    y = linear(x, w[:2], odd, act)
    assert float(y[0, 0]) == float("inf") and torch.isnan(y[0, 1])


@pytest.mark.parametrize("act,p", [(None, 0.0), ("gelu", 0.0), ("relu", 0.2)])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("n,k,m", [(60001, 64, 32), (45000, 40, 20), (60000, 96, 96), (45003, 128, 160), (30000, 264, 136), (40000, 72, 400), (9000, 512, 1100),
                                   (20001, 800, 512), (9473, 1024, 256), (38000, 1000, 96)])   # (the last ones: pairs of blocks)
def test_several_tiles_a_multiprocessor(n, k, m, residual, act, p):
    """More tiles than multiprocessors, of one to eight pieces of columns, a group of columns a block and not: gradients too."""
    x, w, b, r, dy = make(n, k, m, torch.bfloat16)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = linear(*leaves, act, r if residual else None, p, 6)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    keep = dropout(torch.ones(n, m, device=DEV), p, 6).double()
    z = x.double() @ w.double().t() + b.double()
    a, slope = act64(z, act)
    want = a * keep + (r.double() if residual else 0)
    h = half(torch.bfloat16)
    within(y.detach(), want, h * want.abs() + keep * (1.13 * (sums(k, x.double().abs() @ w.double().abs().t(), torch.bfloat16) + 2 * U * z.abs()) + 2e-5 * a.abs() + 1e-11) + 4 * U * want.abs())
    dz = dy.double() * keep * slope
    assert off(dx, dz @ w.double()) <= h and off(dw, dz.t() @ x.double()) <= h and off(db, dz.sum(0)) <= h
    rows = torch.linspace(0, n - 1, 500, device=DEV).long()   # every row is its own
    assert off(dx[rows], (dz @ w.double())[rows]) <= 1.3 * h
    check_device_status(DEV)


def test_gradient_against_differences():
    g = torch.Generator().manual_seed(3)
    n, k, m = 37, 20, 24
    x, w, b, r, dy = (torch.randn(s, generator=g) for s in ((n, k), (m, k), (m,), (n, m), (n, m)))
    u = [torch.randn(s, generator=g) for s in ((n, k), (m, k), (m,), (n, m))]
    for act in ("silu", "gelu"):
        leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b, r)]
        got = torch.autograd.grad(linear(*leaves[:3], act, leaves[3], 0.25, seed=2), leaves, dy.to(DEV))
        keep = dropout(torch.ones(n, m, device=DEV), 0.25, 2).double().cpu()

        def value(t):
            X, W, B, R = (p.double() + t * q.double() for p, q in zip((x, w, b, r), u))
            return float(((act64(X @ W.t() + B, act)[0] * keep + R) * dy.double()).sum())
        t = 1e-4
        want = (8 * (value(t) - value(-t)) - (value(2 * t) - value(-2 * t))) / (12 * t)
        along = sum(float((p.double().cpu() * q).sum()) for p, q in zip(got, u))
        assert abs(along - want) <= 2e-5 * max(1.0, abs(want))


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_in_pieces(dtype):
    """More rows than a piece of the inner gradient has: the same as those of parts, the rows' own bit for bit."""
    n, k, m = (34000, 32, 520) if dtype == torch.float32 else (70000, 32, 520)   # 70 MB
    x, w, b, _, dy = make(n, k, m, dtype)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(linear(*leaves, "relu", dropout_p=0.2, seed=9), leaves, dy)
    keep = dropout(torch.ones(n, m, device=DEV), 0.2, 9).double()
    z = x.double() @ w.double().t() + b.double()
    dz = dy.double() * keep * (z > 0)
    assert off(dx, dz @ w.double()) <= max(1.0 * half(dtype), 2e-6)
    assert off(dw, dz.t() @ x.double()) <= max(1.0 * half(dtype), 2e-6) and off(db, dz.sum(0)) <= max(1.0 * half(dtype), 2e-6)
    one = x[-300:].clone().requires_grad_(True)   # (rows without dropout do not depend on their place)
    part = torch.autograd.grad(linear(one, w, b, "relu"), [one], dy[-300:])[0]
    whole = torch.autograd.grad(linear(leaves[0], w, b, "relu"), [leaves[0]], dy)[0]
    assert torch.equal(part, whole[-300:])


@pytest.mark.parametrize("n,k,m,act", [(5_000_000, 32, 32, None), (2_500_000, 16, 40, "relu"), (250_000, 256, 1024, None), (250_000, 256, 1024, "relu")])
def test_long_sums_of_one_sign(n, k, m, act):
    """Numbers of one sign, which a tensor core's accumulator cuts all one way: beside the result's rounding (half a step, 2^-11, of either sign)
    the weights' gradients may be a quarter of that off in the mean, however many rows there are."""
    g = torch.Generator(device=DEV).manual_seed(n)
    x = ((1 + torch.rand(n, k, device=DEV, generator=g)) * torch.linspace(1, 2, k, device=DEV)).half()   # (results all over a binade)
    dy = ((1 + torch.rand(n, m, device=DEV, generator=g)) * torch.linspace(1, 2, m, device=DEV) * 1000 / n).half()
    w, b = torch.rand(m, k, device=DEV, generator=g).half().requires_grad_(), torch.ones(m, device=DEV, dtype=torch.float16, requires_grad=True)
    dw, db = torch.autograd.grad(linear(x, w, b, act), [w, b], dy)
    want_w, want_b = torch.zeros(m, k, dtype=torch.float64, device=DEV), torch.zeros(m, dtype=torch.float64, device=DEV)
    for at in range(0, n, 1 << 18):
        part = dy[at:at + (1 << 18)].double()
        want_w += part.t() @ x[at:at + (1 << 18)].double()
        want_b += part.sum(0)
    for got, want in ((dw, want_w), (db, want_b)):
        short = (got.double() - want) / want
        assert abs(float(short.mean())) <= 2.0 ** -13 and float(short.abs().max()) <= half(torch.float16) + 2.0 ** -13


@pytest.mark.parametrize("m,act,p", [(1 << 18, None, 0.0), (1 << 20, "relu", 0.0), (1 << 18, None, 0.5)])
def test_long_sums_over_outputs(m, act, p):
    """The gradient of x is a sum over the outputs: half of half a step in the mean, as sums over the most inputs that there may be."""
    n, k = 300, 64
    g = torch.Generator(device=DEV).manual_seed(m)
    x = torch.rand(n, k, device=DEV, generator=g).half().requires_grad_()
    w = ((1 + torch.rand(m, k, device=DEV, generator=g)) * torch.linspace(1, 2, k, device=DEV)).half()
    dy = ((1 + torch.rand(n, m, device=DEV, generator=g)) * torch.linspace(1, 2, n, device=DEV)[:, None] * 1000 / m).half()
    dx, = torch.autograd.grad(linear(x, w, None, act, dropout_p=p, seed=5), [x], dy)
    dz = dy.double() if not p else dy.double() * dropout(torch.ones(n, m, device=DEV, dtype=torch.float16), p, 5).double()
    want = dz @ w.double()
    short = (dx.double() - want) / want
    assert abs(float(short.mean())) <= 2.0 ** -12 and float(short.abs().max()) <= half(torch.float16) + 2.0 ** -11


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,k,m", [(1, 8, 32769), (130, 33, 40001), (700, 96, 65544)])
def test_gradients_of_more_outputs_than_inputs_may_be(dtype, n, k, m):
    x, w, b, _, dy = make(n, k, m, dtype)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    for act, p in ((None, 0.0), ("gelu", 0.25)):
        got = torch.autograd.grad(linear(*leaves, act, dropout_p=p, seed=4), leaves, dy)
        x64, w64, b64 = (t.detach().double() for t in leaves)
        keep = dropout(torch.ones(n, m, device=DEV), p, 4).double() if p else 1.0
        dz = dy.double() * keep * act64(x64 @ w64.t() + b64, act)[1]
        for a, e in zip(got, (dz @ w64, dz.t() @ x64, dz.sum(0))):   # dz's rounding and the result's; sums beside them
            assert off(a, e) <= 2 * half(dtype)


# Wide in 16 bits (pieces of dz, the last one with other splits; dx of it in parts), narrow (rows of one launch; a gradient that is copied), fp32.
PIECES = [(300_001, 64, 1024, torch.bfloat16), (8_000, 64, 40_000, torch.float16), (1_300_001, 16, 40, torch.float16), (1_250_003, 24, 13, torch.bfloat16), (1_300_001, 64, 8, torch.float32)]


@pytest.mark.parametrize("act,p", [(None, 0.3), ("gelu", 0.3), ("gelu", 0.0)])
@pytest.mark.parametrize("n,k,m,dtype", PIECES)
def test_gradients_of_more_rows_than_a_piece(n, k, m, dtype, act, p):
    g = torch.Generator(device=DEV).manual_seed(n)
    x, dy = (torch.randn(n, c, device=DEV, generator=g).to(dtype) for c in (k, m))
    w, b = (torch.randn(m, k, device=DEV, generator=g) / k ** 0.5).to(dtype), torch.randn(m, device=DEV, generator=g).to(dtype)
    what, aligned = 7, int(dtype == torch.float32 or m % 8 == 0)
    one = query_bytes("wcn_linear_workspace_bytes", n // 3, k, m, dtype_code(dtype), what, 3 if act else 0, round(65536 * p), aligned)
    whole = query_bytes("wcn_linear_workspace_bytes", n, k, m, dtype_code(dtype), what, 3 if act else 0, round(65536 * p), aligned)
    assert 1.4 * one < whole < 2.1 * one   # two pieces (of one: three times as much, or for sums alone as much)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    got = torch.autograd.grad(linear(*leaves, act, dropout_p=p, seed=77), leaves, dy)
    keep = dropout(torch.ones(n, m, device=DEV, dtype=torch.bfloat16), p, 77) if p else None
    w64, b64 = w.detach().double(), b.detach().double()
    want = [torch.empty(n, k, dtype=torch.float64, device=DEV), torch.zeros(m, k, dtype=torch.float64, device=DEV), torch.zeros(m, dtype=torch.float64, device=DEV)]
    step = 1 << 13 if m > 10_000 else 1 << 17
    for at in range(0, n, step):
        rows = slice(at, at + step)
        x64 = x[rows].detach().double()
        dz = dy[rows].double() * act64(x64 @ w64.t() + b64, act)[1]
        if p:
            dz *= (keep[rows] != 0) / (1 - round(65536 * p) / 65536)
        want[0][rows] = dz @ w64
        want[1] += dz.t() @ x64
        want[2] += dz.sum(0)
    # in 16 bits dz is rounded and the result is; in fp32 as at fewer rows
    bound = 2 * half(dtype) if dtype != torch.float32 else 4e-6
    for a, e in zip(got, want):
        assert off(a, e) <= bound
    for rows in (slice(0, 500), slice(n // 2, n // 2 + 500), slice(n - 500, n)):
        assert off(got[0][rows], want[0][rows]) <= bound


def test_more_rows_than_a_piece_forward_in_fp32():
    n, k, m = 1_500_001, 64, 8
    g = torch.Generator(device=DEV).manual_seed(0)
    x, r = torch.randn(n, k, device=DEV, generator=g), torch.randn(n, m, device=DEV, generator=g)
    w, b = torch.randn(m, k, device=DEV, generator=g) / 8, torch.randn(m, device=DEV, generator=g)
    one = query_bytes("wcn_linear_workspace_bytes", n // 3, k, m, dtype_code(x.dtype), 0, 3, 20000, 0)
    assert query_bytes("wcn_linear_workspace_bytes", n, k, m, dtype_code(x.dtype), 0, 3, 20000, 0) < 2.1 * one   # two pieces
    y = linear(x, w, b, "gelu", r, 20000 / 65536, 3)
    keep = dropout(torch.ones(n, m, device=DEV), 20000 / 65536, 3) != 0
    z, _ = act64(x.double() @ w.double().t() + b.double(), "gelu")
    want = r.double() + torch.where(keep, z * (65536 / 45536), 0.0)
    # 64 products' sum and its rounding (|x| |w| has the norm of some 8 x 64^0.5 / 8), the activation's 3e-7, the addition's
    assert ((y.double() - want).abs() <= 64 * U * (1 + want.abs() + x.double().abs() @ w.double().abs().t())).all()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("n,k,m", [(300, 32, 64), (300, 512, 640)])   # in one kernel, and by way of dz
def test_large_gradients_in_fp16_under_dropout(n, k, m, act):
    """What is kept is multiplied by 8: the gradients are in range, though the one behind the activation times 8 is not."""
    x, w, b, _, dy = make(n, k, m, torch.float16)
    leaves = [t.requires_grad_() for t in (x * 0.002, w * 2.0 ** -11, b)]
    dy = (dy.sign() * 30000).half()
    dx, dw, _ = torch.autograd.grad(linear(*leaves, act, dropout_p=0.875, seed=2), leaves, dy)
    x64, w64, b64 = (t.detach().double() for t in leaves)
    keep = (dropout(torch.ones(n, m, device=DEV), 0.875, 2) != 0).double() * 8
    dz = dy.double() * keep * act64(x64 @ w64.t() + b64, act)[1]
    want = dz @ w64, dz.t() @ x64
    assert float(dz.abs().max()) > 2 * 65504 and max(float(e.abs().max()) for e in want) < 65000
    for a, e in zip((dx, dw), want):   # dz's rounding and the result's
        assert off(a, e) <= 2 * half(torch.float16)


@pytest.mark.parametrize("n,k,m", [(1_000_000, 64, 13), (600_000, 64, 64)])
def test_a_gradient_in_fp32_between_boundaries(n, k, m):
    """What the backward pass of a concatenation gives: contiguous rows that start on any element.  Parts of half a gigabyte."""
    x, w, b, _, _ = make(n, k, m, torch.float32)
    wide = torch.randn(n * m + 1, device=DEV)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    dy = wide[1:].view(n, m)
    got = torch.autograd.grad(linear(*leaves), leaves, dy)
    want = torch.autograd.grad(linear(*leaves), leaves, dy.clone())
    assert dy.is_contiguous() and all(torch.equal(a, e) for a, e in zip(got, want))
    x, w = x.detach().double(), w.detach().double()
    for a, e in zip(got, (dy.double() @ w, dy.double().t() @ x, dy.double().sum(0))):
        assert off(a, e) <= 2e-6


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_boundaries(dtype):
    """Column blocks of wider buffers, starts on odd elements, every other row, transposed, repeated: as their copies."""
    g = torch.Generator().manual_seed(1)
    wide = torch.randn(300, 200, generator=g).to(dtype).to(DEV)
    w = torch.randn(48, 64, generator=g).to(dtype).to(DEV)
    for view in (wide[:, 8:72], wide[:, 3:67], wide[::2, 64:128], wide[:1, 5:69], wide.t()[:64, :64], wide[:1, :64].expand(40, 64)):
        for weight in (w, torch.cat([w, w], 1)[:, 64:], torch.cat([w, w], 1)[:, 7:71], w.t().contiguous().t()):
            lx, lw = view.detach().requires_grad_(True), weight.detach().requires_grad_(True)
            n = len(view)
            for r, dy in ((wide[:n, 40:88], wide[:n, 100:148]), (wide[:n, 41:89], wide[:n, 101:149]), (wide[:1, :48].expand(n, 48), wide[:1, :48].expand(n, 48))):
                for act in (None, "relu"):
                    got = linear(lx, lw, None, act, r)
                    grads = torch.autograd.grad(got, [lx, lw], dy)
                    cx, cw = view.detach().contiguous().requires_grad_(True), weight.detach().contiguous().requires_grad_(True)
                    want = linear(cx, cw, None, act, r.contiguous())
                    assert torch.equal(got, want) and got.is_contiguous()
                    assert all(torch.equal(p, q) for p, q in zip(grads, torch.autograd.grad(want, [cx, cw], dy.contiguous())))
    assert linear(wide[:0, :64], w).shape == (0, 48)
    lx, lw = wide[:0, :64].clone().requires_grad_(True), w.clone().requires_grad_(True)
    gx, gw = torch.autograd.grad(linear(lx, lw, None, "gelu", dropout_p=0.5).sum(), [lx, lw])
    assert gx.shape == (0, 64) and not gw.any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act,p", [(None, 0.0), ("gelu", 0.2)])
@pytest.mark.parametrize("n,k,m", [(20_001, 512, 400), (9_700, 1000, 776), (38_000, 768, 200)])
def test_two_blocks_to_a_tile_both_ways(dtype, act, p, n, k, m):
    """Forward, the gradient behind the activation and that of x, each with tiles cut at the rows' and the columns' end."""
    x, w, b, r, dy = make(n, k, m, dtype)
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    y = linear(x, w, b, act, r, p, 11)
    got = torch.autograd.grad(y, leaves, dy)
    x64, w64, b64, r64 = (t.detach().double() for t in leaves)
    keep = (dropout(torch.ones(n, m, device=DEV), p, 11) != 0).double() / (1 - round(65536 * p) / 65536) if p else 1.0
    a, slope = act64(x64 @ w64.t() + b64, act)
    dz = dy.double() * keep * slope
    assert off(y.detach(), r64 + keep * a) <= half(dtype)
    for t, e in zip(got, (dz @ w64, dz.t() @ x64, dz.sum(0), dy.double())):   # dz's rounding and the result's
        assert off(t, e) <= 2 * half(dtype)
    assert all(torch.equal(s, t) for s, t in zip(torch.autograd.grad(linear(x, w, b, act, r, p, 11), leaves, dy), got))
    check_device_status(DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k,m", [(45_000, 40, 13), (30_001, 64, 100), (9_000, 300, 20)])
def test_a_residual_on_boundaries_beside_a_result_that_is_not(dtype, n, k, m):
    """Columns of a wider buffer whose rows can be copied as a whole, results whose rows cannot."""
    x, w, b, r, _ = make(n, k, m, dtype)
    wide = torch.zeros(n, -(-m // 8) * 8, dtype=dtype, device=DEV)
    wide[:, :m] = r
    for act in (None, "gelu"):
        want = linear(x, w, b, act, r)
        assert all(torch.equal(linear(x, w, b, act, wide[:, :m]), want) for _ in range(3))
        z, _ = act64(x.double() @ w.double().t() + b.double(), act)
        assert off(want, z + r.double()) <= (half(dtype) if dtype != torch.float32 else 2e-6)


@pytest.mark.parametrize("dtype", DTYPES)
def test_numbers_that_are_none_stay_in_their_rows(dtype):
    x, w, b, r, dy = make(300, 64, 96, dtype)
    clean = linear(x, w, b, "gelu", r)
    bad = x.clone()
    bad[7, 3], bad[130, 0] = float("nan"), float("inf")
    y = linear(bad, w, b, "gelu", r)
    rows = [i for i in range(300) if i not in (7, 130)]
    assert torch.equal(y[rows], clean[rows]) and torch.isnan(y[7]).all() and not torch.isfinite(y[130]).all()
    lx = x.clone().requires_grad_(True)
    out = linear(lx, w, b, "relu", r)
    want = torch.autograd.grad(out, [lx], dy, retain_graph=True)[0]
    worse = dy.clone()
    worse[9] = float("nan")
    got = torch.autograd.grad(out, [lx], worse)[0]
    rows = [i for i in range(300) if i != 9]
    assert torch.equal(got[rows], want[rows]) and torch.isnan(got[9]).any()


def test_gradients_of_some_inputs():
    x, w, b, r, dy = make(500, 48, 80, torch.bfloat16)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    every = torch.autograd.grad(linear(leaves[0], leaves[1], leaves[2], "silu", leaves[3], 0.1, 4), leaves, dy)
    for i in range(4):
        args = [leaf if j == i else leaf.detach() for j, leaf in enumerate(leaves)]
        got, = torch.autograd.grad(linear(args[0], args[1], args[2], "silu", args[3], 0.1, 4), [leaves[i]], dy)
        assert torch.equal(got, every[i]) or (i == 1 and off(got, every[1].double()) <= 2 * half(torch.bfloat16))   # (dw alone is divided in other splits)


def test_captured_and_on_another_stream():
    x, w, b, r, dy = make(4000, 96, 200, torch.bfloat16)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    qx, sx = quantize_rows(x)
    qw, sw = quantize_rows(w)

    def step():
        y = linear(leaves[0], leaves[1], leaves[2], "gelu", leaves[3], 0.1, 4)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy), linear_8bit(qx, sx, qw, sw, b, "relu")]
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(there, want))
    graphs, results = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            results.append(step())
    for i in (0, 1, 0):   # two graphs' workspaces are their own
        for t in results[i][:4] + results[i][5:]:
            t.zero_()
        graphs[i].replay()
        assert all(torch.equal(p, q) for p, q in zip(results[i], want))


def test_graphs_of_the_gradient_and_transforms():
    x, w, b, r, dy = make(12, 8, 10, torch.float32)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    plain = torch.autograd.grad(linear(*leaves[:3], "gelu", leaves[3], 0.2, 3), leaves, dy)
    graph = torch.autograd.grad(linear(*leaves[:3], "gelu", leaves[3], 0.2, 3), leaves, dy, create_graph=True)
    assert all(torch.allclose(p, q, rtol=1e-4, atol=1e-5) for p, q in zip(plain, graph))
    second = torch.autograd.grad(graph[0].square().sum(), leaves[:2])
    keep = dropout(torch.ones(12, 10, device=DEV), 0.2, 3).double()
    X, W = x.double().requires_grad_(True), w.double().requires_grad_(True)
    first, = torch.autograd.grad(torch.nn.functional.gelu(X @ W.t() + b.double()) * keep, [X], dy.double(), create_graph=True)
    assert all(torch.allclose(p.double(), q, rtol=1e-4, atol=1e-4) for p, q in zip(second, torch.autograd.grad(first.square().sum(), [X, W])))
    tangent = torch.func.jvp(lambda t: linear(t, w, b, "silu"), (x,), (x,))[1]
    t64 = torch.func.jvp(lambda t: torch.nn.functional.silu(t @ w.double().t() + b.double()), (x.double(),), (x.double(),))[1]
    assert torch.allclose(tangent.double(), t64, rtol=1e-4, atol=1e-5)


def test_under_autocast():
    x, w, b, r, dy = make(200, 64, 72, torch.float32)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = linear(leaves[0], leaves[1], leaves[2], "gelu", leaves[3])
    low = [t.bfloat16() for t in (x, w, b, r)]
    assert y.dtype == torch.bfloat16 and torch.equal(y, linear(*low[:3], "gelu", low[3]))
    grads = torch.autograd.grad(y, leaves, dy.bfloat16())
    assert all(g.dtype == torch.float32 for g in grads)


@pytest.mark.parametrize("n,k,m", [(1, 16, 8), (1, 256, 1024), (300, 96, 384), (257, 100, 13), (129, 384, 96), (64, 1024, 520), (2000, 130, 40), (5, 33, 7), (9500, 1536, 512), (20001, 2000, 200)])
@pytest.mark.parametrize("out_dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act,residual", [(None, False), ("gelu", True), ("relu", True), ("silu", False)])
def test_eight_bits(n, k, m, out_dtype, act, residual):
    x, w, b, r, _ = make(n, k, m, out_dtype)
    qx, sx = quantize_rows(x)
    qw, sw = quantize_rows(w)
    y = linear_8bit(qx, sx, qw, sw, b, act, r if residual else None, out_dtype)
    X, W = qx.double() * sx.double()[:, None], qw.double() * sw.double()[:, None]
    z = X @ W.t() + b.double()
    a, _ = act64(z, act)
    want = a + (r.double() if residual else 0)
    terms = X.abs() @ W.abs().t()
    # 32 products at a time, sums cut; the two scales
    bound = half(out_dtype) * want.abs() + 1.13 * ((k / 32 + 8) * 2 * U + 4 * U) * (terms + b.double().abs()) + 2e-5 * a.abs() + 4 * U * want.abs() + 1e-10
    within(y, want, bound + (6e-8 if out_dtype == torch.float16 else 0))
    assert torch.equal(y, linear_8bit(torch.cat([qx.view(torch.uint8)] * 2, 1)[:, k:].view(torch.float8_e4m3fn), sx, qw, sw, b.float(), act, r if residual else None, out_dtype))
    check_device_status(DEV)


class expired:
    """The status word of a kernel that gave up waiting, set from the host."""

    def __enter__(self):
        device_status(DEV).fill_(-7)

    def __exit__(self, *exc):
        assert int(device_status(DEV)) == -7
        device_status(DEV).zero_()


def test_fp32_numbers_of_every_size():
    """Numbers without three bf16 parts (2^39 and more, infinities), small ones and subnormal ones: as others in their rows and columns."""
    g = torch.Generator().manual_seed(0)
    n, k, m = 400, 70, 50
    x, w = torch.randn(n, k, generator=g), torch.randn(m, k, generator=g) / 8
    x[3] *= 1e20
    x[200, 7] = 3e30
    x[5] *= 1e-30
    x[6] *= 1e-42
    w[9] *= 1e25
    dy = torch.randn(n, m, generator=g)
    dy[11] *= 1e15
    lx, lw = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    y = linear(lx, lw)
    dx, dw = torch.autograd.grad(y, [lx, lw], dy.to(DEV))
    X, W, D = x.double(), w.double(), dy.double()
    for got, want, terms, c in ((y, X @ W.t(), X.abs() @ W.t().abs(), k), (dx, D @ W, D.abs() @ W.abs(), m), (dw, D.t() @ X, D.t().abs() @ X.abs(), n)):
        got = got.detach().cpu()
        big = terms > 1e38
        assert not torch.isnan(got[~big]).any()
        d = (got.double() - want).abs()
        assert (d <= half(torch.float32) * want.abs() + sums(c, terms, torch.float32) + 2.0 ** -149 * c)[~big].all()


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_fp32_activations_over_their_whole_range(act):
    z = torch.cat([torch.linspace(-20, 20, 8001), torch.logspace(-6, 4, 300), -torch.logspace(-6, 4, 300)]).to(DEV)
    x, w = torch.zeros(1, 8, device=DEV), torch.zeros(len(z), 8, device=DEV)
    b = z.clone().requires_grad_(True)
    y = linear(x, w, b, act)
    slope_got, = torch.autograd.grad(y, [b], torch.ones_like(y))
    value, slope = act64(z.double(), act)
    within(y[0].detach(), value, 16 * U * value.abs() + 1e-37)
    # the slope is f + z f' of the function f that z is multiplied by, which for negative z is a difference: each term is some roundings
    # (of an exponential, a reciprocal, a polynomial, products) off in itself, and the result may be any part of them
    Z = z.double()
    p = torch.sigmoid(Z) if act == "silu" else normal64(Z)
    terms = p + Z.abs() * (p * torch.sigmoid(-Z) if act == "silu" else torch.exp(-Z * Z / 2) * 0.3989422804014327)
    within(slope_got, slope, 24 * U * terms + 1e-37)
    odd = torch.tensor([float("inf"), float("nan")], device=DEV)
    y = linear(x, w[:2], odd, act)
    assert float(y[0, 0]) == float("inf") and torch.isnan(y[0, 1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k,m", [(300, 96, 200), (1, 64, 40), (3000, 1024, 264), (130, 40, 33)])
def test_where_an_earlier_kernel_gave_up_waiting(dtype, n, k, m):
    x, w, b, r, dy = make(n, k, m, dtype)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    for act in (None, "gelu"):
        y = linear(*leaves, act, r)
        want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        with expired():
            assert torch.isnan(linear(x, w, b, act, r)).all()
            assert all(torch.isnan(t).all() for t in torch.autograd.grad(y, leaves, dy, retain_graph=True))
        assert torch.equal(linear(x, w, b, act, r), y) and all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, leaves, dy), want))


def test_refusals():
    x, w, b = torch.zeros(4, 8, device=DEV), torch.zeros(6, 8, device=DEV), torch.zeros(6, device=DEV)
    for bad in (lambda: linear(x[0], w), lambda: linear(x, w[:, :7]), lambda: linear(x, w[:0]), lambda: linear(x, w, b[:5]), lambda: linear(x, w.cpu()), lambda: linear(x, w, b.cpu()),
                lambda: linear(x.cpu(), w.cpu()), lambda: linear(x, w, b, "tanh"), lambda: linear(x, w, b, residual=x), lambda: linear(x, w, dropout_p=2.0),
                lambda: linear(x, w, dropout_p=0.5, seed=torch.tensor(1)), lambda: linear(torch.zeros(1, 32769, device=DEV), torch.zeros(1, 32769, device=DEV)),
                lambda: linear(x, w, residual=torch.zeros(4, 6, device=DEV).half())):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: linear(x, w.half()), lambda: linear(x, w, b.half()), lambda: linear(x.double(), w.double())):
        with pytest.raises(TypeError):
            bad()
    q, s = quantize_rows(x)
    qw, sw = quantize_rows(w)
    for bad in (lambda: linear_8bit(q, s[:3], qw, sw), lambda: linear_8bit(q, s, qw, sw.double()), lambda: linear_8bit(q, s, qw, sw, residual=torch.zeros(4, 6, device=DEV)),
                lambda: linear_8bit(q, s, qw, sw, b.clone().requires_grad_(True))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: linear_8bit(x, s, qw, sw), lambda: linear_8bit(q, s, qw, sw, out_dtype=torch.float32)):
        with pytest.raises(TypeError):
            bad()
