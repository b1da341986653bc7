"""Gradients through the nodes of csrc/autograd.cpp and through autograd functions in Python: the same bits, whatever lies how."""
import threading
import time

import pytest
import torch

from warpconvnet_b200 import _native
from warpconvnet_b200.nn.functional import dropout as dropout_module
from warpconvnet_b200.nn.functional import linear as linear_module
from warpconvnet_b200.nn.functional import rms_norm as norm_module

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def leaf(*shape, dtype):
    return torch.randn(*shape, device=DEV).to(dtype).requires_grad_()


def wide(t):
    """The same numbers as a column block of a wider buffer."""
    buffer = torch.empty(t.shape[0], t.shape[1] + 13, dtype=t.dtype, device=t.device)
    buffer[:, 5:5 + t.shape[1]] = t.detach()
    return buffer[:, 5:5 + t.shape[1]].requires_grad_()


def both(monkeypatch, call):
    """``call()``'s results through the nodes and through Python."""
    assert _native.graph_nodes() is not None
    one = call()
    with monkeypatch.context() as m:
        for module in (linear_module, dropout_module, norm_module):
            m.setattr(module, "graph_nodes", lambda: None)
        return one, call()


def same(one, two):
    assert len(one) == len(two)
    for a, b in zip(one, two):
        assert (a is None) == (b is None) and (a is None or (a.dtype == b.dtype and torch.equal(a, b)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, k, m", [(1, 8, 8), (300, 96, 20), (257, 13, 200), (130, 64, 384), (200, 384, 96)])
@pytest.mark.parametrize("lies", ["rows", "wide", "expanded"])
def test_linear(monkeypatch, dtype, n, k, m, lies):
    torch.manual_seed(0)
    x, w, b, r = leaf(n, k, dtype=dtype), leaf(m, k, dtype=dtype), leaf(m, dtype=dtype), leaf(n, m, dtype=dtype)
    dy = torch.randn(n, m, device=DEV).to(dtype)
    if lies == "wide":
        x, w, r, dy = wide(x), wide(w), wide(r), wide(dy).detach()
    elif lies == "expanded":
        dy = dy[:1, :1].expand(n, m)
    for activation, p, seed in ((None, 0.0, None), ("gelu", 0.25, 7), ("silu", 0.1, torch.tensor([11], device=DEV)), (None, 0.5, -3)):
        for inputs in ([x, w, b, r], [x], [w, b], [r]):
            same(*both(monkeypatch, lambda: torch.autograd.grad(linear_module.linear(x, w, b, activation, r, p, seed), inputs, dy)))
        same(*both(monkeypatch, lambda: torch.autograd.grad(linear_module.linear(x, w, None, activation, None, p, seed), [x, w], dy)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, c", [(1, 1), (300, 96), (77, 13), (9, 2048)])
@pytest.mark.parametrize("lies", ["rows", "wide", "expanded"])
def test_norm(monkeypatch, dtype, n, c, lies):
    torch.manual_seed(0)
    x, r = leaf(n, c, dtype=dtype), leaf(n, c, dtype=dtype)
    dy, dh = torch.randn(n, c, device=DEV).to(dtype), torch.randn(n, c, device=DEV).to(dtype)
    if lies == "wide":
        x, r, dy, dh = wide(x), wide(r), wide(dy).detach(), wide(dh).detach()
    elif lies == "expanded":
        dy, dh = dy[:1, :1].expand(n, c), dh[:1, :1].expand(n, c)
    for w in (leaf(c, dtype=torch.float32), leaf(c, dtype=dtype), None):
        some = [] if w is None else [w]
        same(*both(monkeypatch, lambda: torch.autograd.grad(norm_module.rms_norm(x, w), [x] + some, dy)))
        for inputs in ([x, r] + some, [r], some or [x]):
            same(*both(monkeypatch, lambda: torch.autograd.grad(norm_module.rms_norm(x, w, residual=r), inputs, [dy, dh])))
            same(*both(monkeypatch, lambda: torch.autograd.grad(norm_module.rms_norm(x, w, residual=r)[0], inputs, dy)))
        same(*both(monkeypatch, lambda: torch.autograd.grad(norm_module.rms_norm(x, w, residual=r)[1], [x, r], dh)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, c", [(0, 8), (1, 1), (300, 96), (77, 13)])
@pytest.mark.parametrize("lies", ["rows", "wide"])
def test_dropout(monkeypatch, dtype, n, c, lies):
    torch.manual_seed(0)
    x, r, dy = leaf(n, c, dtype=dtype), leaf(n, c, dtype=dtype), torch.randn(n, c, device=DEV).to(dtype)
    if lies == "wide":
        x, r, dy = wide(x), wide(r), wide(dy).detach()
    for p, seed in ((0.1, 5), (1.0, 5), (0.5, torch.tensor([-9], device=DEV))):
        for inputs in ([x, r], [x], [r]):
            same(*both(monkeypatch, lambda: torch.autograd.grad(dropout_module.dropout(x, p, seed, r), inputs, dy)))
        same(*both(monkeypatch, lambda: torch.autograd.grad(dropout_module.dropout(x, p, seed), [x], dy)))


def block(x, g, w1, b1, w2, seed):
    t = norm_module.rms_norm(x, g)
    t = linear_module.linear(t, w1, b1, "gelu", dropout_p=0.1, seed=seed)
    return dropout_module.dropout(linear_module.linear(t, w2), 0.2, seed, x)


def block_leaves(dtype=torch.bfloat16):
    torch.manual_seed(0)
    return leaf(500, 64, dtype=dtype), leaf(64, dtype=torch.float32), leaf(256, 64, dtype=dtype), leaf(256, dtype=dtype), leaf(64, 256, dtype=dtype)


def test_launches_are_counted():
    tensors = block_leaves()
    before = {k: _native.LAUNCH_COUNTS[k] for k in ("wcn_linear_backward", "wcn_rms_norm_backward", "wcn_dropout")}
    y = block(*tensors, 3)
    assert _native.LAUNCH_COUNTS["wcn_dropout"] == before["wcn_dropout"] + 1
    total = _native.launches_total()
    y.backward(torch.ones_like(y))
    assert _native.LAUNCH_COUNTS["wcn_dropout"] == before["wcn_dropout"] + 2
    assert all(_native.LAUNCH_COUNTS[k] > v for k, v in before.items()) and _native.launches_total() >= total + 5


def test_kept_graphs_checkpoints_streams_and_threads():
    tensors = list(block_leaves())
    dy = torch.randn(500, 64, device=DEV).bfloat16()
    want = torch.autograd.grad(block(*tensors, 3), tensors, dy)
    y = block(*tensors, 3)
    same(torch.autograd.grad(y, tensors, dy, retain_graph=True), want)
    same(torch.autograd.grad(y, tensors, dy), want)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, tensors, dy)
    y = torch.utils.checkpoint.checkpoint(block, *tensors, 3, use_reentrant=False)
    same(torch.autograd.grad(y, tensors, dy), want)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = torch.autograd.grad(block(*tensors, 3), tensors, dy)
    stream.synchronize()
    same(got, want)
    results = [None] * 4

    def work(i):
        for _ in range(5):
            with torch.cuda.stream(torch.cuda.Stream()):
                results[i] = torch.autograd.grad(block(*tensors, 3), tensors, dy)
                torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for got in results:
        same(got, want)


def test_other_threads_go_on_while_a_launch_waits():
    """The GPU is kept busy for half a second, and a thousand launches fill its queue: Python's other threads run meanwhile."""
    x, w = torch.randn(64, 64, device=DEV).bfloat16(), torch.randn(64, 64, device=DEV).bfloat16()
    q, s = norm_module.quantize_rows(x)
    qw, sw = norm_module.quantize_rows(w)
    for call in (lambda: linear_module.linear(x, w), lambda: norm_module.rms_norm(x), lambda: norm_module.rms_norm_8bit(x), lambda: dropout_module.dropout(x, 0.5, 3),
                 lambda: linear_module.linear_8bit(q, s, qw, sw)):
        call()
        torch.cuda.synchronize()
        longest, done = 0.0, threading.Event()

        def launch():
            torch.cuda._sleep(1_000_000_000)
            for _ in range(1500):
                call()
            done.set()
        thread = threading.Thread(target=launch)
        thread.start()
        last = time.perf_counter()
        while not done.wait(0.002):
            now = time.perf_counter()
            longest, last = max(longest, now - last), now
        thread.join()
        torch.cuda.synchronize()
        assert longest < 0.2, longest


def test_what_the_library_refuses_is_an_error_of_the_engine_s_thread():
    """A call without a status word is refused on the host; nothing runs."""
    nodes = _native.graph_nodes()
    for n, k, m in ((5, 4, 3), (1000, 64, 13)):
        x, w, b = (torch.randn(s, device=DEV, requires_grad=True) for s in ((n, k), (m, k), (m,)))
        y = nodes.linear(torch.empty(n, m, device=DEV), x, w, b, None, None, None, None, 0, 0, 0, 0, 0)
        with pytest.raises(RuntimeError, match=r"wcn_linear_backward failed: invalid parameters \(-5\)"):
            torch.autograd.grad(y, [x, w, b], torch.randn(n, m, device=DEV))


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_tensor_in_two_places(monkeypatch, dtype):
    x, w, dy = leaf(100, 64, dtype=dtype), leaf(64, 64, dtype=dtype), torch.randn(100, 64, device=DEV).to(dtype)

    def leaves(call):
        x.grad = w.grad = None
        results = call()
        results = results if isinstance(results, tuple) else (results,)
        torch.autograd.backward(results, [dy[:len(t)] for t in results])
        return [t for t in (x.grad, w.grad) if t is not None]
    for call in (lambda: norm_module.rms_norm(x, residual=x), lambda: linear_module.linear(x, w, activation="relu", residual=x), lambda: linear_module.linear(w, w),
                 lambda: dropout_module.dropout(x, 0.3, 1, x), lambda: norm_module.rms_norm(x * 2, residual=x)):
        one, two = both(monkeypatch, lambda: leaves(call))
        same(one, two)
        assert len({t.data_ptr() for t in one}) == len(one)


def test_gradient_of_the_gradient():
    x, w = leaf(20, 8, dtype=torch.float32), leaf(8, 8, dtype=torch.float32)
    first, = torch.autograd.grad(linear_module.linear(x, w, activation="gelu").sum(), [x], create_graph=True)
    got, = torch.autograd.grad(first.square().sum(), [w])
    first, = torch.autograd.grad(torch.nn.functional.gelu(x.double() @ w.double().t()).sum(), [x], create_graph=True)
    want, = torch.autograd.grad(first.double().square().sum(), [w])
    # sums of 20 x 8 terms, each of some ten fp32 operations, first in x's gradient (8 terms) and again in w's (20)
    assert (got - want).abs().max() <= 400 * 2 ** -24 * want.abs().max()


def test_captured_with_a_seed_on_the_device():
    tensors = block_leaves()
    seed = torch.tensor([5], device=DEV)
    dy = torch.randn(500, 64, device=DEV).bfloat16()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            torch.autograd.grad(block(*tensors, seed), tensors, dy)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(block(*tensors, seed), tensors, dy)
    for value in (5, 77):
        seed.fill_(value)
        graph.replay()
        torch.cuda.synchronize()
        same(got, torch.autograd.grad(block(*tensors, value), tensors, dy))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lies", ["rows", "wide", "off by one"])
def test_calls_without_gradient(monkeypatch, dtype, lies):
    """What the extension runs itself and what it leaves to Python is the same."""
    torch.manual_seed(0)
    x, w, b, r = (t.detach() for t in (leaf(77, 40, dtype=dtype), leaf(24, 40, dtype=dtype), leaf(24, dtype=dtype), leaf(77, 24, dtype=dtype)))
    g = torch.rand(40, device=DEV) + 0.5
    if lies == "wide":
        x, w, r = (wide(t).detach() for t in (x, w, r))
    elif lies == "off by one":   # contiguous, but not on a 16-byte boundary
        x, w, r = (torch.cat([t.flatten()[:1], t.flatten()])[1:].view_as(t) for t in (x, w, r))

    def call():
        return [linear_module.linear(x, w, b, "gelu", r, 0.3, 9), linear_module.linear(x, w), linear_module.linear(x, w, b, "relu"),
                norm_module.rms_norm(x, g), *norm_module.rms_norm(x, None, 1e-3, x), dropout_module.dropout(x, 0.4, 2), dropout_module.dropout(x, 0.4, 2, x)]
    same(*both(monkeypatch, call))
    with torch.no_grad():
        assert not any(t.requires_grad for t in call())
    with torch.autocast("cuda", dtype=torch.bfloat16):
        same(*both(monkeypatch, lambda: [linear_module.linear(x, w, b, "silu")]))
        assert linear_module.linear(x, w, b).dtype == torch.bfloat16


@pytest.mark.parametrize("dtype", DTYPES[1:])
@pytest.mark.parametrize("k, m", [(64, 24), (40, 24), (13, 7)])
def test_calls_in_8_bits(monkeypatch, dtype, k, m):
    torch.manual_seed(0)
    x, w, r, g = torch.randn(77, k, device=DEV).to(dtype), torch.randn(m, k, device=DEV), torch.randn(77, m, device=DEV).to(dtype), torch.rand(k, device=DEV)
    (q, s), (wq, ws) = norm_module.quantize_rows(x), norm_module.quantize_rows(w)
    other = torch.float16 if dtype == torch.bfloat16 else torch.bfloat16

    def call():
        got = [*norm_module.rms_norm_8bit(x, g), *norm_module.rms_norm_8bit(x, residual=x)]
        got = [t.view(torch.uint8) if t.dtype == norm_module.E4M3 else t for t in got]
        return got + [linear_module.linear_8bit(q, s, wq, ws, r[0], "gelu", r, dtype), linear_module.linear_8bit(q, s, wq, ws, out_dtype=dtype),
                      linear_module.linear_8bit(q, s, wq, ws, r[0], out_dtype=other), linear_module.linear_8bit(q[::2], s[::2], wq, ws, residual=r[::2], out_dtype=dtype)]
    same(*both(monkeypatch, call))
    before = _native.LAUNCH_COUNTS["wcn_linear_8bit"]
    linear_module.linear_8bit(q, s, wq, ws)
    assert _native.LAUNCH_COUNTS["wcn_linear_8bit"] == before + 1
    for bad in (lambda: linear_module.linear_8bit(q, s[:3], wq, ws), lambda: linear_module.linear_8bit(q, s.requires_grad_(), wq, ws),
                lambda: linear_module.linear_8bit(q, s.detach(), wq, ws, residual=r, out_dtype=other)):
        with pytest.raises(ValueError):
            bad()


def test_refusals_are_python_s():
    x, w = leaf(4, 8, dtype=torch.float32), leaf(8, 8, dtype=torch.float32)
    for bad in (lambda: linear_module.linear(x, w[:, :4]), lambda: linear_module.linear(x, w, residual=x[:2]), lambda: linear_module.linear(x.cpu(), w),
                lambda: linear_module.linear(x, w, activation="tanh"),
                lambda: linear_module.linear(x, w, dropout_p=2.0), lambda: linear_module.linear(x, w, dropout_p=0.5, seed=2 ** 63),
                lambda: linear_module.linear(x, w, seed=2 ** 63), lambda: norm_module.rms_norm_8bit(x), lambda: norm_module.rms_norm_8bit(x, eps=0.0),
                lambda: norm_module.rms_norm(x, w[0, :4]), lambda: norm_module.rms_norm(x, eps=float("nan")), lambda: norm_module.rms_norm(x, eps=0.0),
                lambda: norm_module.rms_norm(x, residual=x.double()), lambda: dropout_module.dropout(x, 0.5, 2 ** 63),
                lambda: dropout_module.dropout(x, 0.5, 1, x[:, :4]), lambda: dropout_module.dropout(x[0], 0.5, 1)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        linear_module.linear(x, w.half())
    with pytest.raises(TypeError):
        norm_module.rms_norm(x.double())


def test_forward_mode_and_transforms_go_through_torch():
    x, w = torch.randn(6, 8, device=DEV), torch.randn(8, 8, device=DEV)
    t = torch.randn(6, 8, device=DEV)
    _, got = torch.func.jvp(lambda v: linear_module.linear(v, w), (x,), (t,))
    torch.testing.assert_close(got, t @ w.t(), rtol=2 ** -18, atol=2 ** -18)
    stacked = torch.vmap(lambda v: norm_module.rms_norm(v))(torch.stack([x, t]))
    torch.testing.assert_close(stacked[1], norm_module.rms_norm(t), rtol=2 ** -20, atol=2 ** -20)
