"""The example that trains with group norm per scene, the linear cross entropy and AdamW together."""
import math

import pytest
import torch

from warpconvnet_b200 import cat
from warpconvnet_b200._native import LAUNCH_COUNTS
from warpconvnet_b200.examples.train_segmentation import SegmentationNet, make_batch, train

from conftest import rel_l2

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype,state_bits", [(torch.float32, 32), (torch.float16, 32), (torch.bfloat16, 8)])
def test_the_loss_falls(dtype, state_bits):
    before = {k: LAUNCH_COUNTS[k] for k in ("wcn_group_norm_backward", "wcn_linear_ce_backward", "wcn_adamw_step")}
    losses, _ = train(scenes=2, voxels=6000, classes=27, steps=40, state_bits=state_bits, dtype=dtype)
    assert abs(losses[0] - math.log(27)) < 1.0 and all(math.isfinite(v) for v in losses)
    assert losses[-1] < 0.5 * losses[0]
    assert all(LAUNCH_COUNTS[k] > v for k, v in before.items())


def test_a_step_is_the_layers_one_by_one():
    """Loss and gradients of the network against torch's own norm, linear layer and loss on the same features."""
    torch.manual_seed(0)
    net = SegmentationNet(4, 27).to(DEV)
    vox, labels = make_batch(2, 5000, 27, 3, DEV)
    loss = net(vox, labels)
    grads = torch.autograd.grad(loss, [net.head.weight, net.head.bias, net.mix[1].weight])
    feats = net.mix[0](cat(net.up(net.down(net.stem(vox)), net.stem(vox)), net.stem(vox))).feature_tensor
    at, rows = vox.offsets.tolist(), []
    for lo, hi in zip(at, at[1:]):
        rows.append(torch.nn.functional.group_norm(feats[lo:hi].t()[None], 8, net.mix[1].weight, net.mix[1].bias)[0].t())
    x = torch.nn.functional.silu(torch.cat(rows))
    want = torch.nn.functional.cross_entropy(torch.nn.functional.linear(x, net.head.weight, net.head.bias), labels)
    wants = torch.autograd.grad(want, [net.head.weight, net.head.bias, net.mix[1].weight])
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-4
    for a, b in zip(grads, wants):
        assert rel_l2(a.cpu().numpy(), b.cpu().numpy()) < 1e-3
