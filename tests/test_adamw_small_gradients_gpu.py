"""Gradients so small that their squares are among the smallest numbers of fp32, with an epsilon of zero or far below them."""
import pytest
import torch

from warpconvnet_b200.optim import adamw_step, moment_slots

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-24, 1e-15, 1e-8])
@pytest.mark.parametrize("size", [1e-19, 3e-18, 1e-12, 1e-3])
def test_the_update_does_not_depend_on_the_gradients_size(size, eps):
    """The second moment of 1e-19 is 1e-41, a number of 13 bits: its root is known to 2^-14 of itself."""
    n = 1000
    g = size * (1 + torch.rand(n, generator=torch.Generator().manual_seed(0)))
    p, (m, v) = torch.zeros(n, device=DEV), (torch.zeros(moment_slots([n])[1], device=DEV) for _ in range(2))
    steps = torch.zeros(1, dtype=torch.int32, device=DEV)
    adamw_step([p], [g.to(DEV)], m, v, steps, lr=1e-2, eps=eps)
    # after one step the moments over their corrections are the gradient and its square
    want = -1e-2 * g.double() / (g.double().abs() + eps)
    assert float(((p.double().cpu() - want) / want).abs().max()) <= 2.0 ** -13
