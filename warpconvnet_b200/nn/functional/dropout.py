"""Dropout of feature rows from a counter-based generator, with the residual's addition, in a native kernel (``csrc/dropout.cu``):
the gradient makes the same random bits again, and no mask is kept.

An addition to the reference, which uses ``nn.Dropout``."""
from __future__ import annotations

from typing import Optional, Union

import torch
from torch import Tensor

from ..._native import check, dtype_code, graph_nodes, lib, on_device, ptr, require_cuda, stream_ptr
from .batch_norm import reverse_mode_only
from .group_norm import _rows
from .rms_norm import check_residual

_MOST, _MOST_COLUMNS = 0x7FFFFEFF, 1 << 30
_WORD = 0xFFFFFFFF


def check_probability(p: float) -> int:
    """What the random 16 bits of an element that stays are not below."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"the probability to drop an element lies between 0 and 1, got {p}")
    return round(65536 * p)


def check_seed(seed: Union[int, Tensor, None], device: torch.device) -> None:
    if isinstance(seed, Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != device:
            raise ValueError(f"a seed in a tensor must be one int64 on {device}, got {tuple(seed.shape)} {seed.dtype} on {seed.device}")
    elif seed is not None and (not isinstance(seed, int) or not -2 ** 63 <= seed < 2 ** 63):
        raise ValueError(f"seed must be a 64-bit integer, an int64 tensor of one element or None, got {seed!r}")


def new_seed(device: torch.device) -> Union[int, Tensor]:
    """A seed from torch's generators: the host's, or the device's while a graph is captured, which then has another one at every
    replay."""
    if torch.cuda.is_current_stream_capturing():
        return torch.randint(-2 ** 63, 2 ** 63 - 1, (1,), dtype=torch.int64, device=device)
    return int(torch.randint(-2 ** 63, 2 ** 63 - 1, (1,), dtype=torch.int64))


def kept_factor(seed: Union[int, Tensor], n: int, c: int, least: int, device: torch.device) -> Tensor:
    """0, or what is kept is multiplied by, of every element of ``[n, c]``, through torch."""
    a = torch.arange(-(-c // 8), device=device).expand(n, -1)
    row = torch.arange(n, device=device)[:, None].expand_as(a)
    b, d, e = row & _WORD, row >> 32, torch.zeros_like(a)
    seed = seed.reshape(()) if isinstance(seed, Tensor) else seed
    k0, k1 = seed & _WORD, (seed >> 32) & _WORD
    for _ in range(10):
        u, v = a * 0xD2511F53, d * 0xCD9E8D57
        a, b, d, e = ((v >> 32) & _WORD) ^ b ^ k0, v & _WORD, ((u >> 32) & _WORD) ^ e ^ k1, u & _WORD
        k0, k1 = (k0 + 0x9E3779B9) & _WORD, (k1 + 0xBB67AE85) & _WORD
    words = torch.stack([a, b, d, e], dim=2)
    bits = torch.stack([words & 0xFFFF, words >> 16], dim=3).view(n, 8 * a.shape[1])[:, :c]
    return torch.where(bits >= least, 65536 / max(1, 65536 - least), 0.0).float()


def formula(x: Tensor, least: int, seed: Union[int, Tensor], residual: Optional[Tensor]) -> Tensor:
    """The same through torch: for a graph of the gradient, forward-mode differentiation and function transforms."""
    factor = kept_factor(seed, *x.shape, least, x.device)
    y = torch.where(factor > 0, x.float() * factor, 0.0)
    return (y if residual is None else y + residual.float()).to(x.dtype)


def _run(x: Tensor, least: int, seed: Union[int, Tensor], residual: Optional[Tensor]) -> Tensor:
    n, c = x.shape
    dev = x.device
    y = x.new_empty((n, c))
    if n and c:
        x, x_ld = (x, c) if x.is_contiguous() else _rows(x)
        res_ld = c
        if residual is not None and not residual.is_contiguous():
            residual, res_ld = _rows(residual)
        number, at = (0, seed.data_ptr()) if isinstance(seed, Tensor) else (seed, None)
        with on_device(dev):
            check(lib().wcn_dropout(ptr(x), x_ld, ptr(residual), res_ld, n, c, dtype_code(x.dtype), least, number, at, ptr(y), stream_ptr(dev)), "wcn_dropout")
    return y


def gradients(seed: Optional[Tensor], least: int, number: int, needs, dy: Tensor):
    """Those of x and residual.  ``seed``: a tensor, or None where it is ``number``."""
    need_x, need_r = needs
    seed = number if seed is None else seed
    dx = None
    if need_x:
        dx = formula(dy, least, seed, None) if torch.is_grad_enabled() else _run(dy, least, seed, None)
    return dx, dy if need_r else None


class _Dropout(torch.autograd.Function):
    """What a graph's node of ``csrc/autograd.cpp`` is, where that was not built."""

    @staticmethod
    def forward(ctx, x: Tensor, residual: Optional[Tensor], least: int, seed: Union[int, Tensor]):
        ctx.call = least, 0 if isinstance(seed, Tensor) else seed
        ctx.save_for_backward(seed if isinstance(seed, Tensor) else None)   # (one that was changed meanwhile is an error)
        return _run(x, least, seed, residual)

    @staticmethod
    def backward(ctx, dy: Tensor):
        return gradients(*ctx.saved_tensors, *ctx.call, ctx.needs_input_grad[:2], dy) + (None, None)


def dropout(x: Tensor, p: float = 0.5, seed: Union[int, Tensor, None] = None, residual: Optional[Tensor] = None) -> Tensor:
    """``residual + keep * x / (1 - p)`` of ``x [N, C]`` (float32, float16 or bfloat16), rounded once.

    Each element is dropped with probability ``p``, which is taken to the nearest multiple of 2^-16; what is dropped is 0 whatever it
    was.  ``seed``: a 64-bit integer, or an int64 tensor of one element on ``x``'s device, that fixes which elements those are (by
    row and column alone); None: one from torch's generator on the host (while a graph is captured, the device's, another one at
    every replay).  Rows of ``x`` and of the residual may be column blocks of wider buffers."""
    least = check_probability(p)
    nodes, transformed = graph_nodes(), not reverse_mode_only()
    if nodes is not None and not transformed and least and type(seed) is int and -2 ** 63 <= seed < 2 ** 63 and isinstance(x, Tensor):
        y = nodes.run_dropout(x, residual, least, seed, _MOST, _MOST_COLUMNS)
        if y is not None:
            return y
    if x.dim() != 2:
        raise ValueError(f"x must be [N, C], got {tuple(x.shape)}")
    require_cuda(x, "x")
    dtype_code(x.dtype)
    if x.shape[0] > _MOST or x.shape[1] > _MOST_COLUMNS:
        raise ValueError(f"at most {_MOST} rows and {_MOST_COLUMNS} columns are taken, got {tuple(x.shape)}")
    check_residual(residual, x.shape, x.dtype, x.device)
    check_seed(seed, x.device)
    if not least and residual is None:
        return x
    seed = new_seed(x.device) if seed is None else seed
    if transformed:
        return formula(x, least, seed, residual)
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        if nodes is None:
            return _Dropout.apply(x, residual, least, seed)
        with torch.no_grad():
            y = _run(x, least, seed, residual)
        at, number = (seed, 0) if isinstance(seed, Tensor) else (None, seed)
        nodes.dropout(y, x, residual, at, least, number, dtype_code(x.dtype))
        return y
    return _run(x, least, seed, residual)
