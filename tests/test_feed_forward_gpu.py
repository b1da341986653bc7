"""The modules of a feed-forward block, and a block's operators together: against the formula in 64 bits, trained, captured, in 8 bits."""
import pytest
import torch

from warpconvnet_b200 import Dropout, FeedForward, Linear, LinearCrossEntropy, RMSNorm, Sequential, SparseConv3d, Voxels
from warpconvnet_b200._native import LAUNCH_COUNTS, check_device_status
from warpconvnet_b200.nn.functional.dropout import dropout
from warpconvnet_b200.optim import AdamW

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def voxels(n, c, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    side = int(n ** (1 / 3)) + 2
    xyz = torch.stack(torch.meshgrid(*[torch.arange(side)] * 3, indexing="ij"), -1).reshape(-1, 3)[:n].int()
    return Voxels(xyz.to(DEV), torch.randn(n, c, generator=g).to(dtype).to(DEV), offsets=torch.tensor([0, n // 3, n]))


def off(a, b):
    return float((a.detach().double() - b).norm() / b.norm())


def block64(block, x):
    h = x / torch.sqrt(x.square().mean(1, keepdim=True) + block.eps) * block.norm_weight.double()
    u = torch.nn.functional.gelu(h @ block.weight1.double().t() + block.bias1.double())
    return x + u @ block.weight2.double().t() + block.bias2.double()


# roundings of three results behind one another, each 0.58 of half a step in the mean, beside a sum in which the last two are halved or so
TOL = {torch.float32: 2e-6, torch.float16: 2 ** -11, torch.bfloat16: 2 ** -8}


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,c,hidden", [(1, 32, 128), (1000, 96, 384), (3001, 40, 100)])
def test_block_and_its_gradients(dtype, n, c, hidden):
    torch.manual_seed(n)
    block = FeedForward(c, hidden).to(DEV).to(dtype)
    vox = voxels(n, c, dtype)
    x = vox.feature_tensor.clone().requires_grad_(True)
    out = block(vox.replace(batched_features=x))
    assert isinstance(out, Voxels)
    y = out.feature_tensor
    dy = torch.randn(n, c, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    params = list(block.parameters())
    got = torch.autograd.grad(y, [x, *params], dy)
    x64 = x.detach().double().requires_grad_(True)
    want = block64(block, x64)
    ref = torch.autograd.grad(want, [x64, *params], dy.double())
    assert off(y, want.detach()) <= TOL[dtype]
    assert all(off(g, r.double()) <= 4 * TOL[dtype] for g, r in zip(got, ref))   # (of these some have gone through four roundings)
    assert torch.equal(block(x.detach()), y)   # features alone


def test_modules_of_one_operator():
    vox = voxels(500, 32, torch.bfloat16)
    x = vox.feature_tensor
    norm = RMSNorm(32).to(DEV)
    y, h = norm(vox, vox)
    assert torch.equal(h.feature_tensor, x + x)
    assert torch.equal(norm(h).feature_tensor, y.feature_tensor)
    layer = Linear(32, 48, activation="relu", dropout=0.5).to(DEV).bfloat16()
    layer.train()
    a, b = layer(vox).feature_tensor, layer(vox).feature_tensor
    assert not torch.equal(a, b)
    layer.eval()
    assert torch.equal(layer(vox).feature_tensor, layer(x))
    drop = Dropout(0.5)
    torch.manual_seed(3)
    a = drop(vox).feature_tensor
    torch.manual_seed(3)
    assert torch.equal(drop(x, x), dropout(x, 0.5, seed=int(torch.randint(-2 ** 63, 2 ** 63 - 1, (1,), dtype=torch.int64, generator=torch.Generator().manual_seed(3))), residual=x))
    assert (a == 0).float().mean() > 0.4
    drop.eval()
    assert drop(vox) is vox and torch.equal(drop(x, x), x + x)
    for bad in (lambda: Linear(4, 4, activation="tanh"), lambda: Linear(4, 4, dropout=1.5), lambda: Dropout(-1), lambda: RMSNorm(4, eps=0), lambda: FeedForward(4, 8, dropout=2)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_block_in_8_bits(dtype):
    torch.manual_seed(0)
    block = FeedForward(96, 384).to(DEV)
    vox = voxels(2000, 96, dtype)
    low = block.to_8bit()
    y = low(vox).feature_tensor
    want = block64(block, vox.feature_tensor.double()).detach()
    # e4m3 rounds by 2^-4 at most, 0.58 of it in the mean: two operands of each product, and the second product's rows once more
    change = want - vox.feature_tensor.double()
    assert y.dtype == dtype and off(y.double() - vox.feature_tensor.double(), change) <= 0.6 * 2 ** -4 * 3 ** 0.5 + 2 ** -7
    moved = low.half().to(DEV)
    assert moved.weight1.dtype == torch.float8_e4m3fn and moved.scale1.dtype == torch.float32 and torch.equal(moved(vox).feature_tensor, y)
    check_device_status(DEV)


def test_blocks_behind_a_convolution_are_trained():
    torch.manual_seed(0)
    vox = voxels(4000, 16, torch.float32)
    labels = torch.randint(0, 10, (4000,), device=DEV)
    net = torch.nn.ModuleList([Sequential(SparseConv3d(16, 64, 3, bias=False)), FeedForward(64, 256, dropout=0.1), FeedForward(64, 100, "silu"), LinearCrossEntropy(64, 10)]).to(DEV)
    opt = AdamW(net.parameters(), lr=2e-3)
    before = {k: LAUNCH_COUNTS[k] for k in ("wcn_linear", "wcn_linear_backward", "wcn_rms_norm", "wcn_rms_norm_backward")}
    for _ in range(4):
        opt.zero_grad()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = net[3](net[2](net[1](net[0](vox))), labels)
        loss.backward()
        assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in net.parameters())
        opt.step()
    assert all(LAUNCH_COUNTS[k] > v for k, v in before.items())
    check_device_status(DEV)


def test_a_captured_training_step():
    """Forward and backward in a graph: the same elements are dropped both ways, others at every replay."""
    torch.manual_seed(0)
    block = FeedForward(64, 256, dropout=0.25).to(DEV).bfloat16()
    x = torch.randn(3000, 64, device=DEV, dtype=torch.bfloat16)
    params = list(block.parameters())

    def step():
        y = block(x)
        return [y.detach(), *torch.autograd.grad(y, params, torch.ones_like(y))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    first = [t.clone() for t in got]
    graph.replay()
    assert not torch.equal(first[0], got[0]) and all(torch.isfinite(t).all() for t in got)
    # the last bias' gradient counts what is kept: 3000 of 4 / 3 each, less a quarter
    bias = got[1 + [n for n, _ in block.named_parameters()].index("bias2")].double()
    assert (bias / 3000 - 1).abs().max() <= 6 * (0.25 / 0.75 / 3000) ** 0.5 + 2 ** -8
    block.eval()
    want = step()
    assert all(torch.equal(p, q) for p, q in zip(step(), want))
