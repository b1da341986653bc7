"""Group norm and linear cross entropy in graphs: of gradients, of CUDA, and under autocast with function transforms."""
import pytest
import torch

from warpconvnet_b200 import SegmentedGroupNorm, Voxels, linear_cross_entropy, segmented_group_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("which", [(1, 1, 1), (0, 1, 0), (0, 0, 1), (1, 0, 1)])
def test_a_graph_of_the_norms_gradient_without_rows(which):
    x, w, b = torch.zeros(0, 8, device=DEV), torch.ones(8, device=DEV), torch.ones(8, device=DEV)
    leaves = [t for t, need in zip((x, w, b), which) if t.requires_grad_(bool(need)).requires_grad]
    y = segmented_group_norm(x, [0, 0], 2, w, b)
    grads = torch.autograd.grad(y.sum(), leaves, create_graph=True)
    assert all(g.shape == t.shape and not g.any() for g, t in zip(grads, leaves))


@pytest.mark.parametrize("low", [torch.float16, torch.bfloat16])
def test_transforms_under_autocast_are_in_32_bits_too(low):
    """Inputs are brought to autocast's type once; what is computed from them is not."""
    g = torch.Generator().manual_seed(0)
    x, w, labels = torch.randn(200, 64, generator=g).to(DEV), torch.randn(30, 64, generator=g).to(DEV), torch.randint(0, 30, (200,), generator=g).to(DEV)
    want = linear_cross_entropy(x.to(low).double().float(), w.to(low).double().float(), labels)
    with torch.autocast("cuda", dtype=low):
        plain = linear_cross_entropy(x, w, labels)
        got, tangent = torch.func.jvp(lambda t: linear_cross_entropy(t, w, labels), (x,), (torch.ones_like(x),))
    # (sums of 64 products in another order)
    assert abs(float(plain) - float(want)) <= 2e-5 and abs(float(got) - float(want)) <= 2e-5


def test_a_captured_gradient_of_the_norm():
    x = torch.randn(5000, 32, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    w, dy = torch.rand(32, device=DEV, requires_grad=True), torch.randn(5000, 32, device=DEV, dtype=torch.bfloat16)

    def step():
        y = segmented_group_norm(x, [0, 100, 5000], 4, w, activation="gelu")
        return [y.detach(), *torch.autograd.grad(y, [x, w], dy)]
    want = step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        for t in got:
            t.zero_()
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_gradient_that_is_no_number_stays_in_its_scene_and_group(dtype, bad):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(100, 8, generator=g).to(dtype).to(DEV).requires_grad_(True)
    dy = torch.randn(100, 8, generator=g).to(dtype).to(DEV)
    w = torch.rand(8, generator=g).to(DEV).requires_grad_(True)
    y = segmented_group_norm(x, [0, 40, 100], 2, w, activation="silu")
    want = torch.autograd.grad(y, [x, w], dy, retain_graph=True)
    dy[50, 6] = bad
    got = torch.autograd.grad(y, [x, w], dy)
    assert not torch.isfinite(got[0][40:, 4:]).any()
    assert torch.equal(got[0][:40], want[0][:40]) and torch.equal(got[0][40:, :4], want[0][40:, :4])
    assert not torch.isfinite(got[1][6]) and torch.equal(got[1][[0, 1, 2, 3, 4, 5, 7]], want[1][[0, 1, 2, 3, 4, 5, 7]])


def test_a_batch_of_many_scenes_through_a_module():
    """2 900 of them: more than two launches take, some empty."""
    g = torch.Generator().manual_seed(0)
    sizes = torch.randint(0, 12, (2900,), generator=g)
    sizes[::50] = 0
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), sizes.cumsum(0)])
    n = int(offsets[-1])
    vox = Voxels(torch.arange(3 * n, dtype=torch.int32).view(n, 3).to(DEV), torch.randn(n, 16, generator=g).to(DEV), offsets=offsets)
    norm = SegmentedGroupNorm(4, 16, activation="relu").to(DEV)
    y = norm(vox).feature_tensor
    x = vox.feature_tensor.double().cpu()
    want = torch.zeros(n, 16, dtype=torch.float64)
    for lo, hi in zip(offsets.tolist(), offsets.tolist()[1:]):
        if hi > lo:
            xs = x[lo:hi].view(hi - lo, 4, 4)
            var, mean = torch.var_mean(xs, dim=(0, 2), keepdim=True, correction=0)
            want[lo:hi] = torch.relu((xs - mean) * torch.rsqrt(var + 1e-5)).reshape(hi - lo, 16)
    assert float((y.detach().double().cpu() - want).norm() / want.norm()) <= 2e-6
    y.square().sum().backward()
    assert all(torch.isfinite(p.grad).all() for p in norm.parameters())
