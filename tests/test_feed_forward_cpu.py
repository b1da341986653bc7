"""What needs no GPU of the feed-forward operators: the published values of the generator, and what the C entry points refuse on the
host (nothing is launched, the addresses are made up)."""
import ctypes

import pytest
import torch

from warpconvnet_b200 import _native
from warpconvnet_b200.nn.functional.dropout import dropout, kept_factor
from warpconvnet_b200.nn.functional.rms_norm import rms_norm

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
