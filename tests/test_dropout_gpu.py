"""Dropout from a counter-based generator: which elements stay, values, gradients, seeds."""
import pytest
import torch

from warpconvnet_b200.nn.functional.dropout import dropout

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def bits_of(seed, row, col):
    """The 16 bits of one element, by the published rounds on Python's integers."""
    c, k = [col // 8, row & 0xFFFFFFFF, row >> 32, 0], [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(q >> 32) ^ c[1] ^ k[0], q & 0xFFFFFFFF, (p >> 32) ^ c[3] ^ k[1], p & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c[col % 8 // 2] >> (16 * (col % 2)) & 0xFFFF


def kept(seed, n, c, least):
    return torch.tensor([[bits_of(seed, i, j) >= least for j in range(c)] for i in range(n)], device=DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("n,c,p,seed", [(1, 1, 0.5, 3), (3, 8, 0.25, -1), (70, 13, 0.1, 2 ** 62 + 5), (33, 64, 0.9, -2 ** 63), (5, 1000, 0.333, 2 ** 63 - 1), (40, 100, 1.0, 7)])
def test_against_the_formula(dtype, residual, n, c, p, seed):
    g = torch.Generator().manual_seed(n * c)
    x, r, dy = ((torch.randn(n, c, generator=g) + 3).to(dtype).to(DEV) for _ in range(3))
    least = round(65536 * p)
    keep = kept(seed, n, c, least)
    lx, lr = x.clone().requires_grad_(True), r.clone().requires_grad_(True) if residual else None
    y = dropout(lx, p, seed, lr)
    rest = 1 - least / 65536
    want = torch.where(keep, x.double() / rest if rest else 0 * x.double(), 0.0)
    # the factor and the product are rounded in fp32, the sum and the result
    bound = lambda ref, terms: torch.finfo(dtype).eps / 2 * ref.abs() + 3 * 2.0 ** -24 * terms   # noqa: E731
    ref = want + r.double() if residual else want
    assert y.dtype == dtype and ((y.detach().double() - ref).abs() <= bound(ref, want.abs() + r.double().abs())).all()
    if not residual:
        assert torch.equal(y.detach() != 0, keep)
    grads = torch.autograd.grad(y, [t for t in (lx, lr) if t is not None], dy)
    ref = torch.where(keep, dy.double() / rest if rest else 0 * dy.double(), 0.0)
    assert ((grads[0].double() - ref).abs() <= bound(ref, ref.abs())).all() and torch.equal(grads[0] != 0, keep)
    assert not residual or torch.equal(grads[1], dy)
    assert torch.equal(dropout(x, p, torch.tensor([seed], device=DEV), r if residual else None), y.detach())


def test_large_matrices_and_rows_far_behind():
    """Places with more than 32 bits: the last rows of 2.2 thousand million elements."""
    n, c = 8_400_003, 264
    x = torch.ones(n, c, dtype=torch.bfloat16, device=DEV)
    y = dropout(x, 0.3, 11)
    del x
    rows = [0, 1, 4_000_000, n - 3, n - 2, n - 1]
    least = round(65536 * 0.3)
    want = torch.tensor([[bits_of(11, i, j) >= least for j in range(c)] for i in rows], device=DEV)
    assert torch.equal(y[rows] != 0, want)


def test_how_many_stay():
    n, c = 4000, 1000
    for p in (0.1, 0.5):
        share = float((dropout(torch.ones(n, c, device=DEV), p, 5) != 0).double().mean())
        assert abs(share - (1 - p)) <= 6 * (p * (1 - p) / (n * c)) ** 0.5   # six standard deviations


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    """By row and column alone: a column block of a wider buffer, or rows that start between boundaries, keep the same elements."""
    wide = torch.randn(50, 210, device=DEV).to(dtype)
    for view in (wide[:, 8:72], wide[:, 3:67], wide[::2, 64:128], wide[:1, 5:69], wide.t()[:64, :64].t()[:50], wide[:1, :64].expand(9, 64)):
        want = dropout(view.contiguous(), 0.4, 9)
        assert torch.equal(dropout(view, 0.4, 9), want)
        assert torch.equal(dropout(view, 0.4, 9, view), dropout(view.contiguous(), 0.4, 9, view.contiguous()))
    assert dropout(wide[:0], 0.5).shape == (0, 210) and dropout(wide[:, :0], 0.5).shape == (50, 0)


def test_what_is_dropped_is_zero_whatever_it_was():
    x = torch.full((64, 64), float("nan"), device=DEV)
    y = dropout(x, 0.5, 1)
    keep = kept(1, 64, 64, 32768)
    assert torch.isnan(y[keep]).all() and not y[~keep].any()
    assert not dropout(x, 1.0).any()
    assert dropout(x, 0.0) is x and dropout(x, 1e-6) is x
    assert torch.equal(dropout(torch.ones_like(x), 0.0, residual=torch.ones_like(x)), torch.full_like(x, 2.0))


def test_seeds():
    x = torch.ones(100, 100, device=DEV)
    torch.manual_seed(0)
    a, b = dropout(x), dropout(x)
    assert not torch.equal(a, b)
    torch.manual_seed(0)
    assert torch.equal(dropout(x), a)
    leaf = x.clone().requires_grad_(True)
    at = torch.tensor(4, device=DEV)
    y = dropout(leaf, 0.5, at)
    at += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_a_captured_step_has_other_elements_at_every_replay():
    leaf = torch.ones(300, 64, device=DEV, requires_grad=True)

    def step(seed=None):
        y = dropout(leaf, 0.5, seed)
        return y.detach(), torch.autograd.grad(y, [leaf], torch.ones_like(y))[0]
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = step()
    seen = []
    for _ in range(3):
        graph.replay()
        assert torch.equal(y, dx) and (y != 0).any()
        seen.append(y.clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])
    at = torch.tensor([5], device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = step(at)
    for seed in (5, -8):
        at.fill_(seed)
        graph.replay()
        assert torch.equal(y, dropout(leaf.detach(), 0.5, seed)) and torch.equal(y, dx)


def test_graphs_of_the_gradient_and_transforms():
    x = torch.randn(20, 12, device=DEV, requires_grad=True)
    y = dropout(x, 0.5, 3)
    u = torch.randn_like(x, requires_grad=True)
    g, = torch.autograd.grad(y, [x], u, create_graph=True)
    keep = kept(3, 20, 12, 32768)
    assert torch.equal(g, torch.where(keep, u * 2, 0.0))
    assert torch.equal(torch.autograd.grad(g.sum(), [u])[0], torch.where(keep, 2.0, 0.0))
    tangent = torch.func.jvp(lambda t: dropout(t, 0.5, 3), (x.detach(),), (torch.ones(20, 12, device=DEV),))[1]
    assert torch.equal(tangent, torch.where(keep, 2.0, 0.0))


def test_refusals():
    x = torch.zeros(4, 8, device=DEV)
    for bad in (lambda: dropout(x[0]), lambda: dropout(x, -0.1), lambda: dropout(x, 1.1), lambda: dropout(x, float("nan")), lambda: dropout(x, 0.5, 2 ** 63),
                lambda: dropout(x, 0.5, 0.5), lambda: dropout(x, 0.5, torch.tensor(1)), lambda: dropout(x, 0.5, torch.tensor([1, 2], device=DEV)),
                lambda: dropout(x, 0.5, torch.tensor(1.0, device=DEV)), lambda: dropout(x, residual=x[:2]), lambda: dropout(x, residual=x.half())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        dropout(x.double())
