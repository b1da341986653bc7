"""What the calls of group norm, linear cross entropy and AdamW are counted as: the kernels that they launched."""
import pytest
import torch

from warpconvnet_b200 import linear_cross_entropy, segmented_group_norm
from warpconvnet_b200._native import LAUNCH_COUNTS
from warpconvnet_b200.optim import adamw_step, moment_slots

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def counted(name, f):
    before = LAUNCH_COUNTS[name]
    result = f()
    return LAUNCH_COUNTS[name] - before, result


# (rows, channels, classes, dtype, bias): kernels forward; of all gradients; of x alone
CASES = [(300, 40, 20, torch.bfloat16, True, 1, 2, 1),         # losses in one kernel; gradients, and their sums joined
         (300, 40, 20, torch.float16, False, 1, 2, 1),
         (700, 64, 1000, torch.bfloat16, True, 3, 5, 2),       # bias, logits, losses; g and dx, dx joined, dw, joins of dw and db
         (700, 64, 1000, torch.bfloat16, False, 2, 4, 2),
         (300, 40, 70, torch.float32, True, 3, 6, 3)]          # bias, logits, losses; g, two products, joins of dx, dw and db


@pytest.mark.parametrize("n,c,v,dtype,bias,forward,backward,of_x", CASES)
def test_linear_cross_entropy(n, c, v, dtype, bias, forward, backward, of_x):
    x, w = (torch.randn(k, c, device=DEV).to(dtype).requires_grad_(True) for k in (n, v))
    b, labels = torch.randn(v, device=DEV).to(dtype).requires_grad_(True) if bias else None, torch.randint(0, v, (n,), device=DEV)
    launched, loss = counted("wcn_linear_ce", lambda: linear_cross_entropy(x, w, labels, b))
    assert launched == forward
    leaves = [t for t in (x, w, b) if t is not None]
    assert counted("wcn_linear_ce_backward", lambda: torch.autograd.grad(loss, leaves))[0] == backward
    loss = linear_cross_entropy(x, w.detach(), labels, None if b is None else b.detach())
    assert counted("wcn_linear_ce_backward", lambda: torch.autograd.grad(loss, [x]))[0] == of_x


@pytest.mark.parametrize("scenes,launches", [(0, 0), (1, 1), (1280, 1), (1281, 2), (4000, 4)])
def test_group_norm(scenes, launches):
    """A launch for every 1280 scenes that have rows."""
    offsets = [0, 0] + [3 * i for i in range(1, scenes + 1)]
    x = torch.randn(offsets[-1], 8, device=DEV, requires_grad=True)
    launched, y = counted("wcn_group_norm", lambda: segmented_group_norm(x, offsets, 2))
    assert launched == launches
    assert counted("wcn_group_norm_backward", lambda: torch.autograd.grad(y.sum(), [x]))[0] == launches


@pytest.mark.parametrize("sizes,launches", [([0, 0], 0), ([5], 1), ([3, 0, 700] * 320, 1), ([3, 0, 700] * 500, 2)])
def test_adamw(sizes, launches):
    """A launch for every 640 tensors that have elements."""
    params, grads = ([torch.zeros(n, device=DEV) for n in sizes] for _ in range(2))
    m, v = (torch.zeros(moment_slots(sizes)[1], device=DEV) for _ in range(2))
    steps = torch.zeros(len(sizes), dtype=torch.int32, device=DEV)
    assert counted("wcn_adamw_step", lambda: adamw_step(params, grads, m, v, steps, lr=1e-3))[0] == launches
