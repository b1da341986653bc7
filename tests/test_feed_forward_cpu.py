"""What needs no GPU of the feed-forward operators: the published values of the generator, and what the C entry points refuse on the
host (nothing is launched, the addresses are made up)."""
import ctypes

import pytest
import torch

from warpconvnet_b200 import _native
from warpconvnet_b200.nn.functional.dropout import dropout, kept_factor
from warpconvnet_b200.nn.functional.rms_norm import rms_norm
from warpconvnet_b200.nn.functional.rms_norm import check_eps

BASE = 1 << 20   # stands for aligned device memory
INVALID = -5
ONE = 0x3F800000


def test_published_values():
    """Counter and key of zeros give 6627e8d5 e169c58d bc57ac4c 9b00dbd8."""
    bits = [0xE8D5, 0x6627, 0xC58D, 0xE169, 0xAC4C, 0xBC57, 0xDBD8, 0x9B00]
    for i, b in enumerate(bits):
        assert kept_factor(0, 1, 8, b, torch.device("cpu"))[0, i] > 0
        assert kept_factor(0, 1, 8, b + 1, torch.device("cpu"))[0, i] == 0
    assert torch.equal(kept_factor(-1, 9, 20, 3000, torch.device("cpu")), kept_factor(torch.tensor(-1), 9, 20, 3000, torch.device("cpu")))


def test_no_cpu_path():
    for f in (lambda: rms_norm(torch.zeros(2, 4)), lambda: dropout(torch.zeros(2, 4))):
        with pytest.raises(ValueError, match="CUDA"):
            f()


def norm(n=4, c=8, dtype=0, x=BASE, x_ld=8, residual=None, res_ld=0, eps=ONE, h=None, y=BASE, q=None, scale=None):
    return _native.lib().wcn_rms_norm(x, x_ld, residual, res_ld, n, c, dtype, None, eps, h, y, None, q, scale, None)


@pytest.mark.parametrize("bad", [dict(n=-1), dict(n=2 ** 31), dict(c=0), dict(c=8193), dict(dtype=3), dict(x=None), dict(x_ld=7), dict(residual=BASE, res_ld=8), dict(y=None),
                                 dict(residual=BASE, res_ld=7, h=BASE), dict(q=BASE, scale=BASE), dict(y=None, q=BASE), dict(eps=0), dict(eps=0x7FC00000)])
def test_rms_norm_refuses(bad):
    assert norm(**bad) == INVALID
    assert norm(n=0) == 0


def test_rms_norms_gradient_refuses():
    size = _native.query_bytes("wcn_rms_norm_workspace_bytes", 100, 64)
    call = lambda n=100, c=64, ws=BASE, bytes_=size, h_ld=64, dx=BASE, dw=BASE: _native.lib().wcn_rms_norm_backward(   # noqa: E731
        BASE, h_ld, BASE, 64, None, 0, n, c, 0, None, BASE, dx, dw, ws, bytes_, None)
    for bad in (dict(n=0), dict(c=9000), dict(ws=None), dict(ws=BASE + 2), dict(bytes_=size - 1), dict(h_ld=63), dict(dx=None, dw=None)):
        assert call(**bad) == INVALID
    out = ctypes.c_int64()
    assert _native.lib().wcn_rms_norm_workspace_bytes(10, 9000, ctypes.byref(out)) == INVALID


def test_codes_and_dropout_refuse():
    codes = lambda n=4, c=8, ld=8, q=BASE, s=BASE: _native.lib().wcn_quantize_rows(BASE, ld, n, c, 0, q, s, None)   # noqa: E731
    assert codes(n=0) == 0 and all(codes(**b) == INVALID for b in (dict(c=0), dict(ld=7), dict(q=None), dict(s=None)))
    drop = lambda n=4, c=8, ld=8, least=5, dtype=0, y=BASE, res=None, res_ld=0: _native.lib().wcn_dropout(BASE, ld, res, res_ld, n, c, dtype, least, 1, None, y, None)   # noqa: E731
    assert drop(n=0) == 0
    assert all(drop(**b) == INVALID for b in (dict(n=-1), dict(c=0), dict(ld=7), dict(least=-1), dict(least=65537), dict(dtype=5), dict(y=None), dict(res=BASE, res_ld=3)))


def layer(n=4, k=8, m=16, dtype=_native.WCN_BF16, act=0, x=BASE, x_ld=8, w_ld=8, y=BASE, least=0, res=None, res_ld=0, ws=None, size=0, status=BASE):
    return _native.lib().wcn_linear(x, x_ld, n, k, BASE, w_ld, m, dtype, None, act, res, res_ld, least, 1, None, y, ws, size, status, None)


@pytest.mark.parametrize("bad", [dict(n=-1), dict(n=2 ** 31 - 2 ** 17 + 1), dict(k=0), dict(k=32769), dict(m=0), dict(m=2 ** 20 + 1), dict(dtype=7), dict(act=4), dict(act=-1), dict(x=None),
                                 dict(x=BASE + 2), dict(x_ld=12), dict(x_ld=0), dict(w_ld=4), dict(y=None), dict(least=65537), dict(res=BASE, res_ld=15), dict(status=None),
                                 dict(dtype=_native.WCN_F32), dict(dtype=_native.WCN_F32, ws=BASE + 16, size=1 << 40), dict(dtype=_native.WCN_F32, ws=BASE, size=100)])
def test_linear_refuses(bad):
    assert layer(**bad) == INVALID
    assert layer(n=0) == 0


def test_linears_gradient_and_codes_refuse():
    def gradient(n=100, k=64, m=40, dtype=_native.WCN_BF16, act=1, ws=BASE, less=0, what=7, dy=BASE, dy_ld=40, x_ld=64):
        size = _native.query_bytes("wcn_linear_workspace_bytes", 100, 64, 40, dtype, 7, 1, 0, 1)
        out = [BASE if what >> i & 1 else None for i in range(3)]
        return _native.lib().wcn_linear_backward(BASE, x_ld, n, k, BASE, 64, m, dtype, None, act, dy, dy_ld, 0, 0, None, *out, ws, size - less, BASE, None)
    for dtype in (_native.WCN_F32, _native.WCN_F16, _native.WCN_BF16):
        for bad in (dict(n=0), dict(act=9), dict(ws=None), dict(ws=BASE + 16), dict(less=1), dict(what=0), dict(dy=None), dict(dy_ld=39), dict(x_ld=63)):
            assert gradient(dtype=dtype, **bad) == INVALID
    eight = lambda x_ld=16, w_ld=16, out=_native.WCN_F16, scale=BASE, n=4, k=16: _native.lib().wcn_linear_8bit(   # noqa: E731
        BASE, x_ld, scale, n, k, BASE, w_ld, BASE, 8, out, None, 0, None, 0, BASE, BASE, None)
    assert eight(n=0) == 0
    assert all(eight(**b) == INVALID for b in (dict(x_ld=8), dict(w_ld=24), dict(out=_native.WCN_F32), dict(scale=None), dict(k=0)))
    out = ctypes.c_int64()
    for args in ((0, 8, 8, 1, 1, 0, 0, 0), (10, 0, 8, 1, 1, 0, 0, 0), (10, 8, 8, 5, 1, 0, 0, 0), (10, 8, 8, 1, 8, 0, 0, 0), (10, 8, 8, 1, 1, 4, 0, 0)):
        assert _native.lib().wcn_linear_workspace_bytes(*args, ctypes.byref(out)) == INVALID
    # the gradient behind the activation in pieces of 512 MB: whatever the rows are, the workspace stays bounded
    for dtype in (_native.WCN_F32, _native.WCN_BF16):
        assert _native.query_bytes("wcn_linear_workspace_bytes", 2 ** 31 - 2 ** 17, 64, 1000, dtype, 1, 1, 0, 0) <= (512 << 20) + (1 << 20)


@pytest.mark.parametrize("n,k,m", [(1_000_000, 64, 13), (600_000, 64, 64), (2_200_000, 96, 20), (100, 8, 8)])
def test_a_workspace_for_a_gradient_in_fp32_does_not_go_by_where_it_lies(n, k, m):
    """The gradient is taken wherever its numbers are: what was asked for one between boundaries has to do for what the call makes of it."""
    for what in range(1, 8):
        for act, least in ((0, 0), (0, 100), (3, 0)):
            sizes = {_native.query_bytes("wcn_linear_workspace_bytes", n, k, m, _native.WCN_F32, what, act, least, aligned) for aligned in (0, 1)}
            assert len(sizes) == 1


@pytest.mark.parametrize("n,k,m,dtype,act,aligned", [(5000, 8, 1 << 20, _native.WCN_BF16, 1, 1), (300, 64, 60_000, _native.WCN_F32, 3, 1), (5000, 64, 1 << 19, _native.WCN_F16, 0, 0),
                                                     (100_000_000, 8, 13, _native.WCN_F16, 0, 0), (20_000_000, 64, 100, _native.WCN_BF16, 2, 0)])
def test_workspaces_stay_bounded(n, k, m, dtype, act, aligned):
    """Pieces of 512 MB (or 128 rows), also for many outputs and for a gradient between boundaries; what the weight's parts take beside them is its own."""
    size = _native.query_bytes("wcn_linear_workspace_bytes", n, k, m, dtype, 1, act, 0, aligned)
    assert size <= (512 << 20) + (1 << 20) + (6 * k * m if dtype == _native.WCN_F32 else 0)


def test_an_eps_that_fp32_does_not_hold_is_refused():
    assert norm(eps=0x7F800000) == INVALID
    assert check_eps(3.4e38) == 3.4e38
    for eps in (3.5e38, float("inf"), float("nan"), 0.9e-30):
        with pytest.raises(ValueError, match="eps"):
            check_eps(eps)
