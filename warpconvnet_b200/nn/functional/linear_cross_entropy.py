"""Cross entropy of a linear layer's logits, which are never kept, in native kernels (``csrc/linear_ce.cu``).

An addition to the reference, whose networks end in a 1x1x1 convolution (examples/mink_unet.py:405-413) with
``torch.nn.functional.cross_entropy`` behind it: there the logits of all rows and classes and their gradient are in memory."""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from ..._native import check, count_training_launches, device_status, dtype_code, lib, on_device, ptr, query_bytes, require_cuda, stream_ptr
from .batch_norm import _counter, reverse_mode_only

_MOST, _MOST_CHANNELS = 0x7FFFFEFF, 32768   # rows, classes; channels (row numbers of the kernels are 32-bit)
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def check_reduction(reduction: str) -> int:
    try:
        return _REDUCTIONS[reduction]
    except (KeyError, TypeError):
        raise ValueError(f"reduction is one of {list(_REDUCTIONS)}, got {reduction!r}") from None


def _matrix(t: Tensor, c: int = 0):
    """``t`` as the kernels read it (unit stride along the channels; in 16 bits rows on 16-byte boundaries) and the elements from
    row to row.  Copied where it is not so already.  ``c``: the channels of a copy that this function has made (rows may be longer)."""
    n, c = t.shape[0], c or t.shape[1]
    whole = 1 if t.dtype == torch.float32 else 8
    padded = -(-c // whole) * whole
    one_row = n == 1
    if (t.stride(1) == 1 or c == 1) and (one_row or (t.stride(0) >= c and t.stride(0) % whole == 0)) and t.data_ptr() % (2 * whole) == 0:
        return t, padded if one_row else t.stride(0)
    rows = torch.empty((n, padded), dtype=t.dtype, device=t.device)
    rows[:, :c].copy_(t[:, :c])
    return rows, padded


def _workspace(n: int, c: int, v: int, code: int, what: int, device) -> Tensor:
    return torch.empty(query_bytes("wcn_linear_ce_workspace_bytes", n, c, v, code, what), dtype=torch.uint8, device=device)


def _kept(n: int, v: int, bias: bool):
    """Places of the count and of the bias in what is kept, and its length."""
    at_bias = (2 * n + 1 + 3) // 4 * 4
    return 2 * n, at_bias, at_bias + (-(-v // 256) * 256 + 256 if bias else 0)


def _forward(x: Tensor, weight: Tensor, labels: Tensor, bias: Optional[Tensor], ignore_index: int, reduction: int, keep: bool):
    """(loss or losses, what the backward pass needs: log-sum-exp and loss of each row, the count, the bias in units of ln 2; the
    matrices as the kernels read them)"""
    (n, c), v, dev = x.shape, weight.shape[0], x.device
    code, stream = dtype_code(x.dtype), stream_ptr(dev)
    x, x_ld = _matrix(x)
    weight, w_ld = _matrix(weight)
    at_count, at_bias, length = _kept(n, v, bias is not None)
    kept = torch.empty(length, dtype=torch.float32, device=dev)
    loss = torch.empty((), dtype=torch.float32, device=dev)
    rows = torch.empty(n, dtype=torch.float32, device=dev) if not (keep or reduction) else kept[n:2 * n]   # (a result holds no more than itself)
    base = kept.data_ptr()
    ws = _workspace(n, c, v, code, 0, dev)
    with on_device(dev):
        check(lib().wcn_linear_ce(ptr(x), x_ld, n, c, ptr(weight), w_ld, v, ptr(bias), dtype_code(bias.dtype) if bias is not None else 0,
                                  ptr(labels), ignore_index, code, reduction, base, ptr(rows), base + 4 * at_bias if bias is not None else None,
                                  base + 4 * at_count, ptr(loss), ptr(ws), ws.numel(), ptr(_counter(dev, stream)), ptr(device_status(dev)), stream),
              "wcn_linear_ce")
        count_training_launches("wcn_linear_ce")
    return (loss if reduction else rows), kept, x, weight


def formula(x: Tensor, weight: Tensor, labels: Tensor, bias: Optional[Tensor], ignore_index: int, reduction: str) -> Tensor:
    """The same through torch, logits and all: for a graph of the gradient, forward-mode differentiation and function transforms."""
    with torch.autocast("cuda", enabled=False):   # (what the inputs were brought to counts, not what a product would be)
        z = x.float() @ weight.float().t()
    labels = torch.where((labels >= 0) & (labels < weight.shape[0]), labels, ignore_index)
    return torch.nn.functional.cross_entropy(z if bias is None else z + bias.float(), labels, ignore_index=ignore_index, reduction=reduction)


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: Tensor, weight: Tensor, bias: Optional[Tensor], labels: Tensor, ignore_index: int, reduction: str):
        ctx.ignore_index, ctx.reduction = ignore_index, reduction
        loss, kept, x_rows, w_rows = _forward(x.detach(), weight.detach(), labels, None if bias is None else bias.detach().contiguous(),
                                              ignore_index, _REDUCTIONS[reduction], True)
        # (matrices that had to be copied are kept with them: there are not two copies to be made)
        copied = tuple(None if rows.data_ptr() == given.data_ptr() else rows for rows, given in ((x_rows, x), (w_rows, weight)))
        ctx.save_for_backward(x, weight, bias, labels, kept, *copied)
        return loss.clone() if reduction == "none" else loss   # (the row losses are kept: the caller's are its own)

    @staticmethod
    def backward(ctx, grad: Tensor):
        x, weight, bias, labels, kept, x_rows, w_rows = ctx.saved_tensors
        if torch.is_grad_enabled():  # a graph of the gradient is wanted
            loss = formula(x, weight, labels, bias, ctx.ignore_index, ctx.reduction)
            wanted = [t for t, need in zip((x, weight, bias), ctx.needs_input_grad) if need]
            got = iter(torch.autograd.grad(loss, wanted, grad, create_graph=True))
            return tuple(next(got) if need else None for need in ctx.needs_input_grad[:3]) + (None,) * 3
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        (n, c), v, dev = x.shape, weight.shape[0], x.device
        code = dtype_code(x.dtype)
        dx = torch.empty((n, c), dtype=x.dtype, device=dev) if need_x else None
        dw = torch.empty((v, c), dtype=x.dtype, device=dev) if need_w else None
        db = torch.empty(v, dtype=bias.dtype, device=dev) if need_b else None
        grad = grad.float().contiguous()
        at_count, at_bias, _ = _kept(n, v, bias is not None)
        base = kept.data_ptr()
        # (numbers beside which the others keep their precision: what is no number stays with its row, as does a row that does not count)
        row_max = torch.where(torch.isfinite(grad) & (labels != ctx.ignore_index), grad.abs(), 0.0).amax() if ctx.reduction == "none" else None
        x, x_ld = _matrix(x if x_rows is None else x_rows, c)
        weight, w_ld = _matrix(weight if w_rows is None else w_rows, c)
        ws = _workspace(n, c, v, code, need_x + 2 * need_w + 4 * need_b, dev)
        with on_device(dev):
            check(lib().wcn_linear_ce_backward(ptr(x), x_ld, n, c, ptr(weight), w_ld, v, base + 4 * at_bias if bias is not None else None,
                                               ptr(labels), ctx.ignore_index, code, base, base + 4 * n,
                                               base + 4 * at_count if ctx.reduction == "mean" else None, ptr(grad),
                                               ptr(row_max), ptr(dx), ptr(dw), ptr(db), dtype_code(bias.dtype) if need_b else 0, ptr(ws),
                                               ws.numel(), ptr(device_status(dev)), stream_ptr(dev)), "wcn_linear_ce_backward")
            count_training_launches("wcn_linear_ce_backward")
        return dx, dw, db, None, None, None


def linear_cross_entropy(x: Tensor, weight: Tensor, labels: Tensor, bias: Optional[Tensor] = None, ignore_index: int = -100,
                         reduction: str = "mean") -> Tensor:
    """``cross_entropy(x @ weight.T + bias, labels)`` in fp32 without the logits, for any number of classes
    (below 2^31, as the rows; at most 32 768 channels).

    ``x [N, C]`` and ``weight [V, C]`` are float32, float16 or bfloat16 and of one dtype (under autocast they are brought to its
    dtype); ``bias [V]`` may be of any of the three.  ``labels`` are N integers: a row labelled ``ignore_index`` does not count.
    A label that names no class counts as one and is reported by ``check_device_status``.  ``reduction``: ``"mean"`` over the rows that
    count, ``"sum"``, or ``"none"`` for the row losses.  Gradients come in the inputs' dtypes.  With up to 256 classes and a few
    hundred channels in 16 bits that of the logits is in no memory; else it is made and used in pieces of at most 512 MB, beside
    which the sums of a piece take fp32 memory of about two copies of its rows (240 000 rows x 256 channels x 1 000 classes bf16:
    955 MB in all).  In 16 bits it is rounded to x's dtype before the factor of the reduction, with the rows' weights over the
    largest of those that count (in fp16 ``x``'s gradient takes them afterwards)."""
    how = check_reduction(reduction)
    if x.dim() != 2 or weight.dim() != 2 or x.shape[1] != weight.shape[1] or not weight.numel():
        raise ValueError(f"x must be [N, C] and weight [V, C], got {tuple(x.shape)} and {tuple(weight.shape)}")
    if max(x.shape[0], weight.shape[0]) > _MOST or x.shape[1] > _MOST_CHANNELS:
        raise ValueError(f"at most {_MOST} rows and classes and {_MOST_CHANNELS} channels are taken, got {tuple(x.shape)} and {tuple(weight.shape)}")
    if labels.shape != x.shape[:1] or labels.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"labels must be {x.shape[0]} integers, got {tuple(labels.shape)} {labels.dtype}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"bias must be [{weight.shape[0]}], got {tuple(bias.shape)}")
    require_cuda(x, "x")
    if any(t.device != x.device for t in (weight, labels) + (() if bias is None else (bias,))):
        raise ValueError(f"all tensors must be on {x.device}")
    if torch.is_autocast_enabled():
        dtype = torch.get_autocast_dtype("cuda")
        x, weight = x.to(dtype), weight.to(dtype)
    if x.dtype != weight.dtype:
        raise TypeError(f"x is {x.dtype}, weight {weight.dtype}: they must be of one dtype")
    dtype_code(x.dtype)
    if bias is not None:
        dtype_code(bias.dtype)
    labels = labels.long().contiguous()
    if not reverse_mode_only() or not x.shape[0]:
        return formula(x, weight, labels, bias, ignore_index, reduction)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LinearCrossEntropy.apply(x, weight, bias, labels, ignore_index, reduction)
    return _forward(x, weight, labels, None if bias is None else bias.contiguous(), ignore_index, how, False)[0]
