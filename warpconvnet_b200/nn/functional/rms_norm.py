"""Root-mean-square norm of feature rows with the residual's addition before it, in native kernels (``csrc/rms_norm.cu``).

An addition to the reference, whose norms are torch's layers over ``[N, C]`` rows (warpconvnet/nn/modules/normalizations.py)."""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch import Tensor

from ..._native import check, count_training_launches, dtype_code, graph_nodes, lib, on_device, ptr, query_bytes, require_cuda, stream_ptr
from .batch_norm import _bits, apart, reverse_mode_only
from .group_norm import _rows, _vector

_MOST, _MOST_CHANNELS = 0x7FFFFEFF, 8192
_LEAST_EPS, _MOST_EPS = 1e-30, torch.finfo(torch.float32).max
E4M3 = torch.float8_e4m3fn


def check_eps(eps: float) -> float:
    if not _LEAST_EPS <= eps <= _MOST_EPS:
        raise ValueError(f"eps must be a number of at least {_LEAST_EPS} that fp32 holds, got {eps}")
    return eps


def check_rows(x: Tensor, name: str = "x") -> int:
    """``x`` as the row kernels take it; its dtype's code."""
    if x.dim() != 2:
        raise ValueError(f"{name} must be [N, C], got {tuple(x.shape)}")
    require_cuda(x, name)
    code = dtype_code(x.dtype)
    if not 1 <= x.shape[1] <= _MOST_CHANNELS or x.shape[0] > _MOST:
        raise ValueError(f"1 to {_MOST_CHANNELS} channels and at most {_MOST} rows are taken, got {tuple(x.shape)}")
    return code


def check_residual(residual: Optional[Tensor], shape, dtype: torch.dtype, device: torch.device) -> None:
    if residual is not None and (residual.shape != shape or residual.dtype != dtype or residual.device != device):
        raise ValueError(f"residual must be {tuple(shape)} {dtype} on {device}, got {tuple(residual.shape)} {residual.dtype} on {residual.device}")


def _check(x: Tensor, weight: Optional[Tensor], eps: float, residual: Optional[Tensor]) -> int:
    code = check_rows(x)
    check_eps(eps)
    if weight is not None and (weight.shape != x.shape[1:] or weight.device != x.device or not weight.is_floating_point()):
        raise ValueError(f"weight must be {x.shape[1]} floating-point numbers on {x.device}, got {tuple(weight.shape)} {weight.dtype} on {weight.device}")
    if residual is not None:
        check_residual(residual, x.shape, x.dtype, x.device)
    return code


def _forward(x: Tensor, weight: Optional[Tensor], eps: float, residual: Optional[Tensor], code: int, eight: bool, keep: bool):
    """(y, or codes and scales; h, or None; 1 / root mean square of each row, or None)"""
    n, c = x.shape
    dev = x.device
    h = x.new_empty((n, c)) if residual is not None else None
    y = torch.empty((n, c), dtype=E4M3, device=dev) if eight else x.new_empty((n, c))
    scale = torch.empty(n, dtype=torch.float32, device=dev) if eight else None
    rstd = torch.empty(n, dtype=torch.float32, device=dev) if keep else None
    if n:
        x, x_ld = (x, c) if x.is_contiguous() else _rows(x)
        res_ld = c
        if residual is not None and not residual.is_contiguous():
            residual, res_ld = _rows(residual)
        with on_device(dev):
            check(lib().wcn_rms_norm(ptr(x), x_ld, ptr(residual), res_ld, n, c, code, ptr(weight), _bits(eps), ptr(h), None if eight else ptr(y),
                                     ptr(rstd), ptr(y) if eight else None, ptr(scale), stream_ptr(dev)), "wcn_rms_norm")
    return (y, scale) if eight else y, h, rstd


def formula(x: Tensor, weight: Optional[Tensor], eps: float, residual: Optional[Tensor]):
    """The same through torch: for a graph of the gradient, forward-mode differentiation and function transforms."""
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    t = h.float()
    y = t * torch.rsqrt(t.square().mean(dim=1, keepdim=True) + eps)
    y = (y if weight is None else y * weight.float()).to(x.dtype)
    return y if residual is None else (y, h)


def gradients(x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor], h: Optional[Tensor], rstd: Tensor, eps: float, needs, dy: Optional[Tensor],
              dh: Optional[Tensor] = None):
    """Those of x, residual and weight."""
    need_x, need_r, need_w = needs
    if torch.is_grad_enabled():  # a graph of the gradient is wanted: the same formulas through torch
        x, residual, weight = apart(x, residual, weight)
        results = formula(x, weight, eps, residual)
        pairs = [(t, g) for t, g in zip(results if residual is not None else (results,), (dy, dh)) if g is not None]
        wanted = [t for t, need in zip((x, residual, weight), (need_x, need_r, need_w)) if need]
        got = iter(torch.autograd.grad([t for t, _ in pairs], wanted, [g for _, g in pairs], create_graph=True, allow_unused=True) if pairs else
                   [None] * len(wanted))
        return tuple(next(got) if need else None for need in (need_x, need_r, need_w))
    if dy is None:   # the sum alone was used
        return dh if need_x else None, dh if need_r else None, None
    n, c = x.shape
    dev, code = x.device, dtype_code(x.dtype)
    h, h_ld = _rows(x if h is None else h)
    dy, dy_ld = (dy, c) if dy.is_contiguous() else _rows(dy)
    dh_ld = c
    if dh is not None and not dh.is_contiguous():
        dh, dh_ld = _rows(dh)
    dx = x.new_empty((n, c)) if need_x or need_r else None
    dw = (torch.empty if n else torch.zeros)(c, dtype=torch.float32, device=dev) if need_w else None
    if n:
        ws = torch.empty(query_bytes("wcn_rms_norm_workspace_bytes", n, c), dtype=torch.uint8, device=dev) if need_w else None
        gamma = _vector(weight)
        with on_device(dev):
            check(lib().wcn_rms_norm_backward(ptr(h), h_ld, ptr(dy), dy_ld, ptr(dh), dh_ld, n, c, code, ptr(gamma), ptr(rstd), ptr(dx), ptr(dw),
                                              ptr(ws), ws.numel() if need_w else 0, stream_ptr(dev)), "wcn_rms_norm_backward")
            count_training_launches("wcn_rms_norm_backward")
    return dx if need_x else None, dx if need_r else None, (dw if weight.dtype == torch.float32 else dw.to(weight.dtype)) if need_w else None


class _RMSNorm(torch.autograd.Function):
    """What a graph's node of ``csrc/autograd.cpp`` is, where that was not built."""

    @staticmethod
    def forward(ctx, x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor], eps: float, code: int):
        y, h, rstd = _forward(x, _vector(weight), eps, residual, code, False, True)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, residual, weight, h, rstd)
        return y if residual is None else (y, h)

    @staticmethod
    def backward(ctx, dy: Optional[Tensor], dh: Optional[Tensor] = None):
        return gradients(*ctx.saved_tensors, ctx.eps, ctx.needs_input_grad[:3], dy, dh) + (None, None)


def rms_norm(x: Tensor, weight: Optional[Tensor] = None, eps: float = 1e-6, residual: Optional[Tensor] = None) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """``h / sqrt(mean(h ** 2) + eps) * weight`` of each row of ``x [N, C]`` (float32, float16 or bfloat16; at most 8192 channels),
    computed in fp32 and rounded once.

    Without a residual ``h`` is ``x`` and the norm is the result.  With one, ``h = x + residual`` rounded to their dtype, and the
    result is ``(norm, h)``: ``h`` is what the next residual connection adds to.  ``eps`` is at least 1e-30.  Rows of ``x`` and of
    the residual may be column blocks of wider buffers."""
    nodes, transformed = graph_nodes(), not reverse_mode_only()
    if nodes is not None and not transformed and isinstance(x, Tensor):
        results = nodes.run_norm(x, weight, eps, residual, False, _LEAST_EPS, _MOST, _MOST_CHANNELS)
        if results is not None:
            return results
    code = _check(x, weight, eps, residual)
    if transformed:
        return formula(x, weight, eps, residual)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        if nodes is None:
            return _RMSNorm.apply(x, residual, weight, eps, code)
        with torch.no_grad():
            y, h, rstd = _forward(x, _vector(weight), eps, residual, code, False, True)
        nodes.norm(y, h, x, residual, weight, rstd, eps, code)
        return y if residual is None else (y, h)
    y, h, _ = _forward(x, _vector(weight), eps, residual, code, False, False)
    return y if residual is None else (y, h)


def no_gradient(what: str, *tensors: Optional[Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{what} has no gradient: call it under torch.no_grad()")


def rms_norm_8bit(x: Tensor, weight: Optional[Tensor] = None, eps: float = 1e-6, residual: Optional[Tensor] = None):
    """:func:`rms_norm` with the norm in 8 bits: ``(q, scale)``, and ``h`` behind them where a residual is given.

    ``q [N, C]`` are e4m3 numbers and ``scale [N]`` fp32, the largest magnitude of a row's norm / 448 (2^-126 at least), so that
    ``q * scale`` is the norm.  A row with a number that is not finite is NaN, scale and all.  No gradient."""
    nodes = graph_nodes()
    if nodes is not None and isinstance(x, Tensor) and reverse_mode_only():
        results = nodes.run_norm(x, weight, eps, residual, True, _LEAST_EPS, _MOST, _MOST_CHANNELS)
        if results is not None:
            return results
    code = _check(x, weight, eps, residual)
    no_gradient("rms_norm_8bit", x, weight, residual)
    (q, scale), h, _ = _forward(x, _vector(weight), eps, residual, code, True, False)
    return (q, scale) if residual is None else (q, scale, h)


def quantize_rows(x: Tensor) -> Tuple[Tensor, Tensor]:
    """Rows in 8 bits with a scale each, ``(q, scale)`` as :func:`rms_norm_8bit` gives them: weights and activations of
    :func:`linear_8bit`.  No gradient."""
    code = check_rows(x)
    no_gradient("quantize_rows", x)
    n, c = x.shape
    dev = x.device
    q, scale = torch.empty((n, c), dtype=E4M3, device=dev), torch.empty(n, dtype=torch.float32, device=dev)
    if n:
        x, ld = _rows(x)
        with on_device(dev):
            check(lib().wcn_quantize_rows(ptr(x), ld, n, c, code, ptr(q), ptr(scale), stream_ptr(dev)), "wcn_quantize_rows")
    return q, scale
