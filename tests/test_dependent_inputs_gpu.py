"""Graphs of gradients (``create_graph=True``) where one input of an operator was made from another, or is it: the derivatives of the
operators' formulas, each input for itself."""
import pytest
import torch

from warpconvnet_b200 import SparseConv3d, Voxels, linear_cross_entropy, segmented_group_norm
from warpconvnet_b200.nn.functional import batch_norm, group_norm
from warpconvnet_b200.nn.functional.linear_cross_entropy import formula as cross_entropy
from warpconvnet_b200.nn.functional.sparse_conv import train_layer_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def leaves(*shapes):
    g = torch.Generator().manual_seed(0)
    return [torch.randn(s, generator=g).to(DEV).requires_grad_() for s in shapes]


def check(f, plain, inputs, bound=1e-5):
    """First gradients with a graph, and where that has one the gradients of their squares, against those of ``plain``.  (fp32 against fp32 in
    another order, some 30 roundings of sums of a thousand terms at most.)"""
    got, want = (torch.autograd.grad(h(*inputs), inputs, create_graph=True) for h in (f, plain))
    for a, e in zip(got, want):
        assert float((a - e).norm()) <= bound * float(e.norm())
    got, want = (torch.autograd.grad(sum(t.square().sum() for t in first), inputs) for first in (got, want))
    for a, e in zip(got, want):
        assert float((a - e).norm()) <= 10 * bound * float(e.norm())


def test_group_norm():
    a, w = leaves((60, 8), (8,))
    offsets = [0, 20, 60]

    def run(norm):
        return lambda a, w: norm(a + norm(a, w, None), w, w * 0.5).pow(3).sum()
    check(run(lambda x, w, b: segmented_group_norm(x, offsets, 2, w, b, activation="silu")),
          run(lambda x, w, b: group_norm.formula(x, offsets, 2, w, b, 1e-5, "silu")), [a, w])


def test_linear_cross_entropy():
    a, w = leaves((60, 16), (16, 16))
    labels = torch.randint(0, 16, (60,), generator=torch.Generator().manual_seed(1)).to(DEV)
    check(lambda a, w: linear_cross_entropy(a @ w, w, labels, w.sum(1)), lambda a, w: cross_entropy(a @ w, w, labels, w.sum(1), -100, "mean"), [a, w])


@pytest.mark.parametrize("relu", [False, True])
def test_batch_norm_with_residual(relu):
    a, m, dy = leaves((60, 16), (16, 16), (60, 16))
    bn = torch.nn.BatchNorm1d(16).to(DEV).train()
    for x in (lambda a, m: a, lambda a, m: a @ m):
        check(lambda a, m: (batch_norm.batch_norm_act(x(a, m), bn, relu, a) * dy * m.sum()).sum(),
              lambda a, m: (batch_norm.formula(x(a, m), bn.weight, bn.bias, a, bn.eps, relu) * dy * m.sum()).sum(), [a, m])


def test_a_convolution_with_norm_and_its_input_as_residual():
    g = torch.Generator().manual_seed(0)
    xyz = torch.unique(torch.randint(0, 12, (700, 3), generator=g, dtype=torch.int32), dim=0)
    feats, dy = (torch.randn(len(xyz), 32, generator=g).to(DEV) for _ in range(2))
    torch.manual_seed(0)
    layer, bn = SparseConv3d(32, 32, 3, bias=False).to(DEV).train(), torch.nn.BatchNorm1d(32).to(DEV).train()
    x = Voxels(xyz.to(DEV), feats, offsets=torch.tensor([0, len(xyz)]))
    a = feats.clone().requires_grad_()
    inputs = [a, layer.weight]

    def together(f):
        y = train_layer_norm(layer, bn, x.replace(batched_features=f), None, True, f)
        assert "LayerNorm" in type(y.feature_tensor.grad_fn).__name__
        return y.feature_tensor

    def apart(f):
        return batch_norm.formula(layer(x.replace(batched_features=f)).feature_tensor, bn.weight, bn.bias, f, bn.eps, True)
    for f in (lambda t: t, lambda t: t * 2):
        got, want = (torch.autograd.grad((h(f(a)) * dy).sum(), inputs, create_graph=True) for h in (together, apart))
        for p, q in zip(got, want):   # (the same kernels, sums in another order)
            assert float((p - q).norm()) <= 1e-5 * float(q.norm())
