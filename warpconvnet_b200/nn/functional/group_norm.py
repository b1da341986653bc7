"""Group norm with statistics per scene and the activation behind it, in native kernels (``csrc/group_norm.cu``).

An addition to the reference, whose ``GroupNorm`` is ``nn.GroupNorm`` of ``[N, C]`` rows (statistics per row)."""
from __future__ import annotations

import ctypes
from array import array
from typing import Optional, Sequence, Union

import torch
from torch import Tensor

from ..._native import check, count_training_launches, device_status, dtype_code, lib, on_device, ptr, query_bytes, require_cuda, stream_ptr
from .batch_norm import _bits, _counter, apart, reverse_mode_only

_ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3}


def check_activation(activation: Optional[str]) -> int:
    try:
        return _ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"activation is one of {list(_ACTIVATIONS)}, got {activation!r}") from None


def _host_offsets(offsets: Union[Tensor, Sequence[int], None], n: int) -> array:
    """[scenes + 1] 64-bit integers on the host."""
    if offsets is None:
        return array("q", (0, n))
    if isinstance(offsets, Tensor):
        if offsets.dim() != 1 or offsets.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"offsets must be a 1-d integer tensor [scenes + 1], got {tuple(offsets.shape)} {offsets.dtype}")
        offsets = offsets.detach().to(device="cpu", dtype=torch.int64).numpy().tobytes()
    try:
        at = array("q", offsets)
    except (TypeError, OverflowError):
        raise ValueError("offsets must be integers [scenes + 1]") from None
    if not at or at[-1] != n:
        raise ValueError(f"offsets must end at the {n} rows of x, got {list(at[-4:])}")
    return at


def _rows(t: Tensor):
    """``t`` with unit stride along the channels, and the elements from row to row."""
    n, c = t.shape
    if (t.stride(1) != 1 and c > 1) or (n > 1 and t.stride(0) < c):
        t = t.contiguous()
    return t, max(t.stride(0), c)


def _workspace(offsets: array, c: int, groups: int, dtype: int, backward: bool, device) -> Tensor:
    size = ctypes.c_int64(0)
    if lib().wcn_group_norm_workspace_bytes(offsets.buffer_info()[0], len(offsets) - 1, c, groups, dtype, int(backward), ctypes.addressof(size)):
        raise ValueError(f"offsets must rise from 0, and at most 4096 channels are taken: got {list(offsets[:8])} ... and {c} channels")
    return torch.empty(max(16, size.value), dtype=torch.uint8, device=device)


def _sync(device, stream: int) -> Tensor:
    return _counter(device, stream, query_bytes("wcn_group_norm_sync_bytes") // 4)


def _forward(x: Tensor, offsets: array, groups: int, weight, bias, eps: float, act: int, keep: bool):
    """(y, mean and 1 / std of each scene and group, or None)"""
    n, c = x.shape
    dev, dc = x.device, dtype_code(x.dtype)
    ws = _workspace(offsets, c, groups, dc, False, dev)
    y = torch.empty((n, c), dtype=x.dtype, device=dev)
    scenes = len(offsets) - 1
    saved = torch.empty((2, scenes, groups), dtype=torch.float32, device=dev) if keep else None
    x, ld = _rows(x)
    at, stream = saved.data_ptr() if keep else None, stream_ptr(dev)
    with on_device(dev):
        check(lib().wcn_group_norm(ptr(x), ld, offsets.buffer_info()[0], scenes, c, groups, dc, ptr(weight), ptr(bias), _bits(eps), act, ptr(y),
                                   at, at + 4 * scenes * groups if keep else None, ptr(ws), ws.numel(), ptr(_sync(dev, stream)),
                                   ptr(device_status(dev)), stream), "wcn_group_norm")
        count_training_launches("wcn_group_norm")
    return y, saved


def formula(x: Tensor, offsets: Sequence[int], groups: int, weight, bias, eps: float, activation: Optional[str]) -> Tensor:
    """The same through torch, scene by scene: for a graph of the gradient, forward-mode differentiation and function transforms."""
    out = [x.float()[:0]]   # (no rows: the result hangs on all inputs all the same)
    for lo, hi in zip(offsets, offsets[1:]):
        if hi > lo:
            xs = x[lo:hi].float().reshape(hi - lo, groups, -1)
            var, mean = torch.var_mean(xs, dim=(0, 2), keepdim=True, correction=0)
            out.append(((xs - mean) * torch.rsqrt(var + eps)).reshape(hi - lo, -1))
    z = torch.cat(out)
    z = z if weight is None else z * weight.float()
    z = z if bias is None else z + bias.float()
    act = {None: lambda t: t, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[activation]
    return act(z).to(x.dtype)


class _SegmentedGroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], offsets: array, groups: int, eps: float, activation):
        y, saved = _forward(x, offsets, groups, _vector(weight), _vector(bias), eps, _ACTIVATIONS[activation], True)
        ctx.save_for_backward(x, weight, bias, saved)
        ctx.offsets, ctx.groups, ctx.eps, ctx.activation = offsets, groups, eps, activation
        return y

    @staticmethod
    def backward(ctx, dy: Tensor):
        x, weight, bias, saved = ctx.saved_tensors
        if torch.is_grad_enabled():  # a graph of the gradient is wanted: the same formulas through torch
            x, weight, bias = apart(x, weight, bias)
            y = formula(x, ctx.offsets, ctx.groups, weight, bias, ctx.eps, ctx.activation)
            wanted = [t for t, need in zip((x, weight, bias), ctx.needs_input_grad) if need]
            got = iter(torch.autograd.grad(y, wanted, dy, create_graph=True))
            return tuple(next(got) if need else None for need in ctx.needs_input_grad[:3]) + (None,) * 4
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        n, c = x.shape
        dev, dc, scenes = x.device, dtype_code(x.dtype), len(ctx.offsets) - 1
        x, x_ld = _rows(x)
        dy, dy_ld = _rows(dy)
        dx = torch.empty((n, c), dtype=x.dtype, device=dev) if need_x else None
        sums = torch.empty((2, c), dtype=torch.float32, device=dev) if need_w or need_b else None
        ws = _workspace(ctx.offsets, c, ctx.groups, dc, True, dev)
        gamma, beta, at, stream = _vector(weight), _vector(bias), saved.data_ptr(), stream_ptr(dev)
        with on_device(dev):
            check(lib().wcn_group_norm_backward(ptr(x), x_ld, ptr(dy), dy_ld, ctx.offsets.buffer_info()[0], scenes, c, ctx.groups, dc, ptr(gamma),
                                                ptr(beta), at, at + 4 * scenes * ctx.groups, _ACTIVATIONS[ctx.activation], ptr(dx), ptr(sums),
                                                ptr(ws), ws.numel(), ptr(_sync(dev, stream)), ptr(device_status(dev)), stream), "wcn_group_norm_backward")
            count_training_launches("wcn_group_norm_backward")
        return (dx, sums[1].to(weight.dtype) if need_w else None, sums[0].to(bias.dtype) if need_b else None) + (None,) * 4


def _vector(t: Optional[Tensor]) -> Optional[Tensor]:
    if t is None or (t.dtype == torch.float32 and t.is_contiguous()):
        return t
    return t.detach().float().contiguous()


def segmented_group_norm(x: Tensor, offsets: Union[Tensor, Sequence[int], None], num_groups: int, weight: Optional[Tensor] = None,
                         bias: Optional[Tensor] = None, eps: float = 1e-5, activation: Optional[str] = None) -> Tensor:
    """``act(weight * (x - mean) / sqrt(var + eps) + bias)`` of ``x [N, C]`` (float32, float16 or bfloat16), rounded once.

    ``mean`` and the biased ``var`` are taken over the rows ``offsets[b] .. offsets[b + 1]`` of a scene and the
    ``C / num_groups`` channels of a group, in fp32.  ``offsets`` rise from 0 to N, best on the CPU as a ``Voxels`` has them
    (on a device they are read back); None: one scene.  ``activation``: None, ``"relu"``, ``"silu"`` or ``"gelu"`` (of the error
    function).  Rows of ``x`` may be a column block of a wider buffer."""
    act = check_activation(activation)
    if x.dim() != 2:
        raise ValueError(f"x must be [N, C], got {tuple(x.shape)}")
    require_cuda(x, "x")
    dtype_code(x.dtype)
    n, c = x.shape
    if num_groups < 1 or c < 1 or c % num_groups:
        raise ValueError(f"{c} channels are not divisible into {num_groups} groups")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None and (t.shape != (c,) or t.device != x.device or not t.is_floating_point()):
            raise ValueError(f"{name} must be {c} floating-point numbers on {x.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    offsets = _host_offsets(offsets, n)
    if not reverse_mode_only():
        return formula(x, offsets, num_groups, weight, bias, eps, activation)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _SegmentedGroupNorm.apply(x, weight, bias, offsets, num_groups, eps, activation)
    return _forward(x, offsets, num_groups, _vector(weight), _vector(bias), eps, act, False)[0]
