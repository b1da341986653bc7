"""Linear layers over feature rows with bias, activation, dropout and residual in one native kernel (``csrc/linear.cu``), in fp32, 16
bits and, for inference, of operands in 8 bits.

An addition to the reference, whose ``Linear`` and MLP blocks (warpconvnet/nn/modules/mlp.py) run torch's layers one after the other."""
from __future__ import annotations

from typing import Optional, Union

import torch
from torch import Tensor

from ..._native import WCN_F32, check, count_training_launches, device_status, dtype_code, graph_nodes, lib, on_device, ptr, query_bytes, require_cuda, stream_ptr
from .batch_norm import apart, reverse_mode_only
from .dropout import check_probability, check_seed, kept_factor, new_seed
from .group_norm import _ACTIVATIONS, _rows, check_activation
from .linear_cross_entropy import _matrix
from .rms_norm import E4M3, check_residual, no_gradient

_MOST, _MOST_INPUTS, _MOST_OUTPUTS = 0x7FFE0000, 32768, 1 << 20
_NAMES = {code: name for name, code in _ACTIVATIONS.items()}


def _check_shapes(x: Tensor, weight: Tensor, bias: Optional[Tensor]) -> None:
    if x.dim() != 2 or weight.dim() != 2 or x.shape[1] != weight.shape[1] or not weight.numel():
        raise ValueError(f"x must be [N, K] and weight [M, K], got {tuple(x.shape)} and {tuple(weight.shape)}")
    if x.shape[0] > _MOST or x.shape[1] > _MOST_INPUTS or weight.shape[0] > _MOST_OUTPUTS:
        raise ValueError(f"at most {_MOST} rows, {_MOST_INPUTS} inputs and {_MOST_OUTPUTS} outputs are taken, got {tuple(x.shape)} and {tuple(weight.shape)}")
    require_cuda(x, "x")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"bias must be [{weight.shape[0]}], got {tuple(bias.shape)}")
    if weight.device != x.device or (bias is not None and bias.device != x.device):
        raise ValueError(f"all tensors must be on {x.device}")


def _operand(t: Tensor, whole: int, c: int = 0):
    """``t`` as the kernels read it and the elements from row to row (``_matrix``, without its questions where they have an answer)."""
    if t.is_contiguous() and t.data_ptr() % 16 == 0 and t.shape[1] % whole == 0:
        return t, t.shape[1]
    return _matrix(t, c)


def _forward(x: Tensor, weight: Tensor, bias: Optional[Tensor], act: int, residual: Optional[Tensor], least: int, seed, code: int):
    """(y, the matrices as the kernels read them)"""
    (n, k), m, dev = x.shape, weight.shape[0], x.device
    y = x.new_empty((n, m))
    whole = 1 if code == WCN_F32 else 8
    x, x_ld = _operand(x, whole)
    weight, w_ld = _operand(weight, whole)
    res_ld = m
    if residual is not None and not residual.is_contiguous():
        residual, res_ld = _rows(residual)
    number, at = (0, seed.data_ptr()) if isinstance(seed, Tensor) else (seed, None)
    size = query_bytes("wcn_linear_workspace_bytes", n, k, m, code, 0, act, least, 0) if code == WCN_F32 else 0
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    with on_device(dev):
        check(lib().wcn_linear(x.data_ptr(), x_ld, n, k, weight.data_ptr(), w_ld, m, code, ptr(bias), act, ptr(residual), res_ld, least, number, at,
                               y.data_ptr(), ptr(ws), size, device_status(dev).data_ptr(), stream_ptr(dev)), "wcn_linear")
        count_training_launches("wcn_linear")
    return y, x, weight


def formula(x: Tensor, weight: Tensor, bias: Optional[Tensor], activation: Optional[str], residual: Optional[Tensor], least: int, seed) -> Tensor:
    """The same through torch: for a graph of the gradient, forward-mode differentiation and function transforms."""
    with torch.autocast("cuda", enabled=False):
        z = x.float() @ weight.float().t()
    z = z if bias is None else z + bias.float()
    y = {None: lambda t: t, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[activation](z)
    if least:
        factor = kept_factor(seed, *z.shape, least, z.device)
        y = torch.where(factor > 0, y * factor, 0.0)
    return (y if residual is None else y + residual.float()).to(x.dtype)


def gradients(x: Tensor, weight: Tensor, bias: Optional[Tensor], seed, x_rows: Optional[Tensor], w_rows: Optional[Tensor], act: int, least: int,
              number: int, code: int, needs, dy: Tensor):
    """Those of x, weight, bias and residual.  ``seed``: a tensor, or None where it is ``number``; ``x_rows``, ``w_rows``: copies that the
    forward call has made."""
    seed = number if seed is None else seed
    need_x, need_w, need_b, need_r = needs
    d_residual = dy if need_r else None
    if torch.is_grad_enabled():  # a graph of the gradient is wanted: the same formulas through torch
        x, weight, bias = apart(x, weight, bias)
        y = formula(x, weight, bias, _NAMES[act], None, least, seed)
        wanted = [t for t, need in zip((x, weight, bias), (need_x, need_w, need_b)) if need]
        got = iter(torch.autograd.grad(y, wanted, dy, create_graph=True) if wanted else ())
        return tuple(next(got) if need else None for need in (need_x, need_w, need_b)) + (d_residual,)
    if not (need_x or need_w or need_b):
        return None, None, None, d_residual
    (n, k), m, dev = x.shape, weight.shape[0], x.device
    dx = x.new_empty((n, k)) if need_x else None
    dw = weight.new_empty((m, k)) if need_w else None
    db = weight.new_empty(m) if need_b else None
    dy, dy_ld = (dy, m) if dy.is_contiguous() else _rows(dy)
    whole = 1 if code == WCN_F32 else 8
    aligned = dy_ld % whole == 0 and dy.data_ptr() % (2 * whole) == 0
    x, x_ld = _operand(x if x_rows is None else x_rows, whole, k)
    weight, w_ld = _operand(weight if w_rows is None else w_rows, whole, k)
    bias = None if bias is None else bias.contiguous()
    number, at = (0, seed.data_ptr()) if isinstance(seed, Tensor) else (seed, None)
    size = query_bytes("wcn_linear_workspace_bytes", n, k, m, code, need_x + 2 * need_w + 4 * need_b, act, least, int(aligned))
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    with on_device(dev):
        check(lib().wcn_linear_backward(x.data_ptr(), x_ld, n, k, weight.data_ptr(), w_ld, m, code, ptr(bias), act, dy.data_ptr(), dy_ld, least, number, at,
                                        ptr(dx), ptr(dw), ptr(db), ptr(ws), size, device_status(dev).data_ptr(), stream_ptr(dev)),
              "wcn_linear_backward")
        count_training_launches("wcn_linear_backward")
    return dx, dw, db, d_residual


class _Linear(torch.autograd.Function):
    """What a graph's node of ``csrc/autograd.cpp`` is, where that was not built."""

    @staticmethod
    def forward(ctx, x: Tensor, weight: Tensor, bias: Optional[Tensor], residual: Optional[Tensor], act: int, least: int, seed, code: int):
        y, x_rows, w_rows = _forward(x, weight, None if bias is None else bias.contiguous(), act, residual, least, seed, code)
        ctx.call = act, least, 0 if isinstance(seed, Tensor) else seed, code
        # (matrices that had to be copied are kept with them: there are not two copies to be made)
        ctx.save_for_backward(x, weight, bias, seed if isinstance(seed, Tensor) else None, None if x_rows is x else x_rows, None if w_rows is weight else w_rows)
        return y

    @staticmethod
    def backward(ctx, dy: Tensor):
        return gradients(*ctx.saved_tensors, *ctx.call, ctx.needs_input_grad[:4], dy) + (None, None, None, None)


def linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, activation: Optional[str] = None, residual: Optional[Tensor] = None,
           dropout_p: float = 0.0, seed: Union[int, Tensor, None] = None) -> Tensor:
    """``residual + dropout(act(x @ weight.T + bias))`` of ``x [N, K]`` and ``weight [M, K]``, summed in fp32 and rounded once.

    All tensors are of one dtype, float32, float16 or bfloat16 (under autocast they are brought to its dtype).  ``activation``: None,
    ``"relu"``, ``"silu"`` or ``"gelu"`` (of the error function).  ``dropout_p`` and ``seed`` as in :func:`dropout`; a probability of 0
    drops nothing.  The gradient computes the activation's argument again; beside its results it takes fp32 sums of ``weight``'s
    gradient (parts of the rows have their own, as many as there are multiprocessors and in 16 bits one for 8192 rows at least) and, for
    wider layers, the gradient behind the activation in pieces of at most 512 MB or 128 rows.  In 16 bits that gradient, without
    dropout's factor, is rounded to ``x``'s dtype before its products (float16 ends at 65 504, which a slope of up to 1.13 reaches
    from 58 000 on).  In fp32 the operands are made into sums of three bf16 numbers, 6 bytes for each, in pieces of at most 512 MB or
    128 rows too.  At most 32 768 inputs and 2^20 outputs."""
    act = check_activation(activation)
    least = check_probability(dropout_p) if dropout_p else 0
    nodes, transformed = graph_nodes(), not reverse_mode_only()
    if nodes is not None and not transformed and isinstance(x, Tensor) and (type(seed) is int and -2 ** 63 <= seed < 2 ** 63 or seed is None and not least):
        y = nodes.run_linear(x, weight, bias, residual, act, least, seed if least else 0, _MOST, _MOST_INPUTS, _MOST_OUTPUTS)
        if y is not None:
            return y
    _check_shapes(x, weight, bias)
    if torch.is_autocast_enabled():
        dtype = torch.get_autocast_dtype("cuda")
        x, weight = x.to(dtype), weight.to(dtype)
        bias, residual = (t if t is None else t.to(dtype) for t in (bias, residual))
    code = dtype_code(x.dtype)
    if weight.dtype != x.dtype or (bias is not None and bias.dtype != x.dtype):
        raise TypeError(f"x is {x.dtype}, weight {weight.dtype}{'' if bias is None else f', bias {bias.dtype}'}: they must be of one dtype")
    if residual is not None:
        check_residual(residual, (x.shape[0], weight.shape[0]), x.dtype, x.device)
    if seed is not None:
        check_seed(seed, x.device)
    seed = new_seed(x.device) if least and seed is None else 0 if not least else seed
    if transformed or not x.shape[0]:
        return formula(x, weight, bias, activation, residual, least, seed)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        if nodes is None:
            return _Linear.apply(x, weight, bias, residual, act, least, seed, code)
        with torch.no_grad():
            y, x_rows, w_rows = _forward(x, weight, None if bias is None else bias.contiguous(), act, residual, least, seed, code)
        at, number = (seed, 0) if isinstance(seed, Tensor) else (None, seed)
        return nodes.linear(y, x, weight, bias, residual, at, None if x_rows is x else x_rows, None if w_rows is weight else w_rows, act, least,
                            number, code, device_status(x.device).data_ptr())
    return _forward(x, weight, None if bias is None else bias.contiguous(), act, residual, least, seed, code)[0]


def _codes(t: Tensor):
    """8-bit rows as the kernels read them, and the bytes from row to row."""
    n, k = t.shape
    if (t.stride(1) == 1 or k == 1) and t.data_ptr() % 16 == 0 and (n == 1 or (t.stride(0) >= k and t.stride(0) % 16 == 0)):
        return t, t.stride(0) if n > 1 else -(-k // 16) * 16
    rows = torch.empty((n, -(-k // 16) * 16), dtype=torch.uint8, device=t.device)
    rows[:, :k].copy_(t.view(torch.uint8))
    return rows, rows.shape[1]


def _check_scale(scale: Tensor, rows: int, device: torch.device, name: str) -> None:
    if scale.shape != (rows,) or scale.dtype != torch.float32 or scale.device != device:
        raise ValueError(f"{name} must be {rows} float32 numbers on {device}, got {tuple(scale.shape)} {scale.dtype} on {scale.device}")


def linear_8bit(x: Tensor, x_scale: Tensor, weight: Tensor, weight_scale: Tensor, bias: Optional[Tensor] = None, activation: Optional[str] = None,
                residual: Optional[Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """:func:`linear` of e4m3 numbers with a scale a row, as ``rms_norm_8bit`` and ``quantize_rows`` give them: products in 8 bits, summed in
    fp32, times the scales.  ``residual`` and the result are of ``out_dtype`` (float16 or bfloat16), to which the bias is brought.  No
    gradient."""
    act = check_activation(activation)
    nodes = graph_nodes()
    if nodes is not None and (out_dtype is torch.bfloat16 or out_dtype is torch.float16) and isinstance(x, Tensor) and reverse_mode_only():
        y = nodes.run_linear_8bit(x, x_scale, weight, weight_scale, bias, act, residual, dtype_code(out_dtype), _MOST, _MOST_INPUTS, _MOST_OUTPUTS)
        if y is not None:
            return y
    _check_shapes(x, weight, bias)
    if x.dtype != E4M3 or weight.dtype != E4M3:
        raise TypeError(f"x and weight must be {E4M3}, got {x.dtype} and {weight.dtype}")
    if out_dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"out_dtype must be float16 or bfloat16, got {out_dtype}")
    (n, k), m, dev = x.shape, weight.shape[0], x.device
    _check_scale(x_scale, n, dev, "x_scale")
    _check_scale(weight_scale, m, dev, "weight_scale")
    check_residual(residual, (n, m), out_dtype, dev)
    no_gradient("linear_8bit", x, x_scale, weight, weight_scale, bias, residual)
    y = torch.empty((n, m), dtype=out_dtype, device=dev)
    if not n:
        return y
    x, x_ld = _codes(x)
    weight, w_ld = _codes(weight)
    res_ld = 0
    if residual is not None:
        residual, res_ld = _rows(residual)
    bias = None if bias is None else bias.to(out_dtype).contiguous()
    x_scale, weight_scale = x_scale.contiguous(), weight_scale.contiguous()
    with on_device(dev):
        check(lib().wcn_linear_8bit(ptr(x), x_ld, ptr(x_scale), n, k, ptr(weight), w_ld, ptr(weight_scale), m, dtype_code(out_dtype), ptr(bias), act,
                                    ptr(residual), res_ld, ptr(y), ptr(device_status(dev)), stream_ptr(dev)), "wcn_linear_8bit")
        count_training_launches("wcn_linear_8bit")
    return y
