"""Nodes of autograd's graph in the extension (csrc/autograd.cpp): what they pass on to Python, and what stands in for them."""
import copy
import gc
import os
import subprocess
import sys
from collections import Counter

import pytest
import torch

from warpconvnet_b200 import _native
from warpconvnet_b200.nn.functional import dropout as dropout_module
from warpconvnet_b200.nn.functional import linear as linear_module
from warpconvnet_b200.nn.functional import rms_norm as norm_module

nodes = _native.graph_nodes()
built = pytest.mark.skipif(nodes is None, reason="the extension was not built here")


def test_the_extension_is_built_where_its_compiler_is():
    assert nodes is not None or not os.path.isfile(_native.AUTOGRAD_PATH)


def test_without_the_extension_functions_in_python_stand_in(monkeypatch, tmp_path):
    monkeypatch.setattr(_native, "AUTOGRAD_PATH", str(tmp_path / "_autograd.so"))
    assert _native._load_nodes() is None
    (tmp_path / "_autograd.so").write_bytes(b"no library")
    assert _native._load_nodes() is None


@built
def test_another_torch_does_not_load_it():
    """Its nodes are laid out as one version of torch has them; a build for another one is made anew."""
    from warpconvnet_b200.csrc import build
    assert build._autograd_is_built(torch.__version__) and not build._autograd_is_built("1.2.3")
    code = "import torch\nfrom warpconvnet_b200 import _native\ntorch.__version__ = {!r}\nprint(_native.graph_nodes() is None)"
    root = os.path.dirname(os.path.dirname(os.path.abspath(_native.__file__)))
    for version, refused in ((torch.__version__, "False"), ("1.2.3", "True")):
        out = subprocess.run([sys.executable, "-c", code.format(str(version))], cwd=root, capture_output=True, text=True, timeout=300)
        assert out.stdout.strip() == refused, out.stderr


@built
def test_the_extension_has_no_cpp_library_of_its_own():
    """(Two in a process, and the text of the first error ended it.)"""
    with open(_native.AUTOGRAD_PATH, "rb") as f:
        assert b"\0libstdc++.so" in f.read()


@built
def test_what_the_library_refuses_is_an_error_with_its_number():
    x, w = leaves((5, 4), (3, 4))
    y = nodes.linear(torch.empty(5, 3), x, w, None, None, None, None, None, 9, 0, 0, 0, 0)   # no such activation
    with pytest.raises(RuntimeError, match=r"invalid parameters \(-5\)"):
        torch.autograd.grad(y, [x], torch.ones(5, 3))


def leaves(*shapes):
    torch.manual_seed(0)
    return [torch.randn(s, requires_grad=True) for s in shapes]


def linear(x, w, b, r, act=2):
    with torch.no_grad():
        y = linear_module.formula(x, w, b, linear_module._NAMES[act], r, 0, 0)
    return nodes.linear(y, x, w, b, r, None, None, None, act, 0, 0, 0, 0)


@built
def test_a_graph_of_the_gradient_is_the_formula_s():
    x, w, b, r = leaves((5, 4), (3, 4), (3,), (5, 3))
    y = linear(x, w, b, r)
    assert y.grad_fn.name() == "LinearBackward"
    first = torch.autograd.grad(y.square().sum(), [x, w, b, r], create_graph=True)
    want = torch.autograd.grad(linear_module.formula(x, w, b, "silu", r, 0, 0).square().sum(), [x, w, b, r], create_graph=True)
    for a, e in zip(first, want):
        torch.testing.assert_close(a, e, rtol=0, atol=0)
    second = torch.autograd.grad(first[0].square().sum(), [w], create_graph=True)
    torch.testing.assert_close(second, torch.autograd.grad(want[0].square().sum(), [w], create_graph=True), rtol=2 ** -18, atol=2 ** -18)


@built
def test_norm_and_dropout():
    x, r, g = leaves((5, 4), (5, 4), (4,))
    with torch.no_grad():
        y, h = norm_module.formula(x, g, 1e-6, r)
    nodes.norm(y, h, x, r, g, torch.ones(5), 1e-6, 0)
    got = torch.autograd.grad(y.square().sum() + h.sum(), [x, r, g], create_graph=True)
    a, b = norm_module.formula(x, g, 1e-6, r)
    torch.testing.assert_close(got, torch.autograd.grad(a.square().sum() + b.sum(), [x, r, g]))
    with torch.no_grad():
        y, h = norm_module.formula(x, g, 1e-6, r)
    nodes.norm(y, h, x, r, g, torch.ones(5), 1e-6, 0)
    assert all((t == 1).all() for t in torch.autograd.grad(h.sum(), [x, r]))   # the sum alone was used
    with torch.no_grad():
        y = dropout_module.formula(x, 20000, 5, r)
    nodes.dropout(y, x, r, None, 20000, 5, 0)
    dx, dr = torch.autograd.grad(y.sum(), [x, r], create_graph=True)
    assert torch.equal(dx, dropout_module.formula(torch.ones(5, 4), 20000, 5, None)) and (dr == 1).all()


@built
@pytest.mark.parametrize("f", [lambda layer, a, w: layer(layer(a, w, None, a), w, None, a), lambda layer, a, w: layer(a, a, None, None),
                               lambda layer, a, w: layer(a, w, w.sum(1), a), lambda layer, a, w: layer(a @ w, w, None, None)],
                         ids=["one weight twice", "one tensor twice", "a bias of the weight", "rows of the weight"])
def test_a_graph_of_a_linear_layer_s_gradient_where_inputs_depend_on_each_other(f):
    a, w = leaves((5, 4), (4, 4))

    def gradients(layer):
        y = f(layer, a, w)
        first = torch.autograd.grad(y.square().sum(), [a, w], create_graph=True, allow_unused=True)
        return first + torch.autograd.grad(sum(t.square().sum() for t in first if t is not None), [a, w], create_graph=True, allow_unused=True)
    want = gradients(lambda x, w, b, r: linear_module.formula(x, w, b, "silu", r, 0, 0))
    for got, e in zip(gradients(linear), want):
        if e is None:
            assert got is None
        else:
            torch.testing.assert_close(got, e, rtol=2 ** -18, atol=2 ** -18 * float(e.abs().max()))


def norm(x, g, r):
    with torch.no_grad():
        results = norm_module.formula(x, g, 1e-6, r)
    y, h = (results, None) if r is None else results
    nodes.norm(y, h, x, r, g, torch.ones(x.shape[0]), 1e-6, 0)
    return results


@built
@pytest.mark.parametrize("inputs", [lambda a, m: (a, a), lambda a, m: (a * 1.5, a), lambda a, m: (a @ m, a), lambda a, m: (a, a @ m)])
def test_a_graph_of_the_norm_s_gradient_where_inputs_depend_on_each_other(inputs):
    a, m, g = leaves((5, 4), (4, 4), (4,))

    def gradients(f):
        x, r = inputs(a, m)
        y, h = f(x, g, r)
        first = torch.autograd.grad(y.square().sum() + h.pow(3).sum(), [a, g], create_graph=True)
        return first + torch.autograd.grad(first[0].square().sum() + first[1].square().sum(), [a, g], create_graph=True)
    want = gradients(lambda x, g, r: norm_module.formula(x, g, 1e-6, r))
    for got, e in zip(gradients(norm), want):   # the same sums in fp32, in another order
        torch.testing.assert_close(got, e, rtol=2 ** -18, atol=2 ** -18 * float(e.abs().max()))


@built
def test_a_graph_of_a_norm_s_gradient_behind_the_same_weight():
    a, g = leaves((5, 4), (4,))

    def gradients(f):
        first = torch.autograd.grad(f(f(a, g, None) + a.square(), g, None).pow(3).sum(), [a, g], create_graph=True)
        return first + torch.autograd.grad(first[0].square().sum() + first[1].square().sum(), [a, g], create_graph=True)
    want = gradients(lambda x, g, r: norm_module.formula(x, g, 1e-6, r))
    for got, e in zip(gradients(norm), want):
        torch.testing.assert_close(got, e, rtol=2 ** -18, atol=2 ** -18 * float(e.abs().max()))


@built
def test_errors_are_the_engine_s(monkeypatch):
    x, w, b, r = leaves((5, 4), (3, 4), (3,), (5, 3))
    y = linear(x, w, b, r)

    def refuses(*_):
        raise ValueError("not today")
    with monkeypatch.context() as m:
        m.setattr(linear_module, "formula", refuses)
        with pytest.raises(ValueError, match="not today"):
            torch.autograd.grad(y.sum(), [x], create_graph=True)
    y = linear(x, w, b, r)
    with torch.no_grad():
        w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), [x], create_graph=True)
    y = linear(x, w, b, r)
    torch.autograd.grad(y.sum(), [x], create_graph=True, retain_graph=False)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y.sum(), [x], create_graph=True)


@built
def test_what_a_node_keeps_goes_with_it():
    x, w, b = leaves((5, 4), (3, 4), (3,))
    kept = [0]

    class Packed:
        def __init__(self, t):
            self.t = t
            kept[0] += 1

        def __del__(self):
            kept[0] -= 1
    with torch.autograd.graph.saved_tensors_hooks(Packed, lambda p: p.t):
        y = linear(x, w, b, None)
    assert kept[0] == 3
    torch.autograd.grad(y.sum(), [x], create_graph=True, retain_graph=True)
    del y
    gc.collect()
    assert kept[0] == 0


def test_launches_of_the_extension_are_counted_however_they_are_read(monkeypatch):
    class Nodes:
        left = 0

        def launches(self):
            n, self.left = self.left, 0
            return (0, 0, n, 0, 0, 0)
    nodes = Nodes()
    monkeypatch.setattr(_native, "_nodes", nodes)
    counts = _native.LAUNCH_COUNTS
    monkeypatch.setattr(_native, "LAUNCH_COUNTS", counts := type(counts)())
    reads = [lambda: counts["wcn_dropout"], lambda: counts.get("wcn_dropout"), lambda: dict(counts)["wcn_dropout"], lambda: dict(counts.items())["wcn_dropout"],
             lambda: sum(counts.values()), lambda: counts.total(), lambda: counts.copy()["wcn_dropout"], lambda: (counts - Counter())["wcn_dropout"],
             lambda: copy.deepcopy(counts)["wcn_dropout"], lambda: counts.most_common(1)[0][1], lambda: {**counts}["wcn_dropout"], lambda: list(counts.elements()).count("wcn_dropout"),
             lambda: 10 * len(counts), lambda: 10 * ("wcn_dropout" in counts), lambda: 10 * len(list(counts)), lambda: 10 * len(counts.keys()), lambda: counts.pop("wcn_dropout"),
             _native.launches_total]
    for read in reads:
        counts.clear()
        nodes.left = 3
        before = counts["wcn_dropout"]   # (3 of them are in)
        nodes.left = 7
        assert before == 3 and read() == 10
    nodes.left = 5
    taken = counts.copy()
    nodes.left = 2
    assert taken["wcn_dropout"] == counts["wcn_dropout"] - 2   # (a copy takes nothing away)
    counts.clear()
    nodes.left = 5   # (what was launched before goes with the others)
    counts.clear()
    assert counts["wcn_dropout"] == 0
