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
