"""AdamW over many tensors in one launch (``csrc/adamw.cu``), moments in 32 bits or in 8.

The moments of all tensors are one flat tensor each: a tensor's moments begin at its *slot*, a multiple of 256 elements, and fill
whole blocks of 256.  With 8 bits they are codes of a logarithmic scale, 8 values to an octave, with one int16 base per block:
the code ``k > 0`` stands for the fp32 number with the bits ``(k + base) << 20``, 0 for zero; the first moment has a sign in its
top bit.  Numbers are rounded to a neighbouring code at random (a hash of the tensor's step and the element's place), so that the
second moment, which moves by a thousandth per step, keeps its mean.
"""
from __future__ import annotations

import functools
import struct
from array import array
from itertools import accumulate, chain
from operator import attrgetter, eq
from typing import List, Optional, Sequence, Tuple, Union

import torch
from torch import Tensor

from .._native import check, count_training_launches, dtype_code, lib, on_device, ptr, require_cuda, stream_ptr
from ..nn.functional.batch_norm import _counter

BLOCK = 256


@functools.lru_cache(maxsize=256)
def _bits(value: float) -> int:
    """A number as the 64 bits of a double (calls pass integers only)."""
    return struct.unpack("<q", struct.pack("<d", value))[0]


def moment_slots(sizes: Sequence[int]) -> Tuple[List[int], int]:
    """(first element of each tensor's moments, length of the flat moments) for tensors of these sizes in order."""
    out = list(accumulate([-(-n // BLOCK) * BLOCK for n in sizes], initial=0))
    return out[:-1], out[-1]


_dtype, _shape = attrgetter("dtype"), attrgetter("shape")
_BOUNDS = -8   # a status of the library


def _at(a: Optional[array]) -> Optional[int]:
    return None if a is None else a.buffer_info()[0]


def _one(kinds: set, what: str):
    if len(kinds) != 1:
        raise ValueError(f"{what} differ: {sorted(map(str, kinds))}")
    return kinds.pop()


def _scalar(t: Optional[Tensor], name: str, device: torch.device) -> Optional[int]:
    if t is None:
        return None
    if t.device != device or t.dtype != torch.float32 or t.numel() != 1:
        raise ValueError(f"{name} must be one float32 on {device}, got {t.numel()} x {t.dtype} on {t.device}")
    return t.data_ptr()


def _moments(m: Tensor, v: Tensor, m_base: Optional[Tensor], v_base: Optional[Tensor], device: torch.device) -> int:
    """The length of the flat moments, which are checked."""
    if (m_base is None) != (v_base is None):
        raise ValueError("both moments have bases (8 bits) or none (32 bits)")
    dtype = torch.float32 if m_base is None else torch.uint8
    n = m.numel()
    for t, name in ((m, "exp_avg"), (v, "exp_avg_sq")):
        if t.dtype != dtype or t.device != device or t.dim() != 1 or not t.is_contiguous() or t.numel() != n or n % BLOCK or t.data_ptr() % 32:
            raise ValueError(f"{name} must be a contiguous, 32-byte aligned 1-d {dtype} tensor of a multiple of {BLOCK} elements on {device}, "
                             f"as long as the other moment; got {tuple(t.shape)} {t.dtype} on {t.device}")
    for t, name in ((m_base, "exp_avg_base"), (v_base, "exp_avg_sq_base")):
        if t is not None and (t.dtype != torch.int16 or t.device != device or t.numel() != n // BLOCK or not t.is_contiguous()):
            raise ValueError(f"{name} must be {n // BLOCK} contiguous int16 on {device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    return n


def adamw_step(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avg: Tensor, exp_avg_sq: Tensor, steps: Tensor, *,
               lr: Union[float, Tensor], betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
               exp_avg_base: Optional[Tensor] = None, exp_avg_sq_base: Optional[Tensor] = None, slots: Optional[Sequence[int]] = None,
               step_index: Optional[Sequence[int]] = None, grad_scale: Optional[Tensor] = None, found_inf: Optional[Tensor] = None) -> None:
    """One AdamW step of ``params`` in place, computed in fp32.

    ``params`` (contiguous, one dtype) and ``grads`` (one dtype, which may be another) are float32, float16 or bfloat16 CUDA
    tensors of one device.  ``exp_avg`` / ``exp_avg_sq`` are the flat moments: float32, or uint8 codes with their int16 bases
    (zeros to begin with).  ``slots`` are the tensors' places in them, one after the other (:func:`moment_slots`) where not
    given.  ``steps`` (int32, on the device) counts each tensor's steps and is advanced; ``step_index`` are the tensors' places
    in it.  ``lr`` may be a float32 device tensor, which a captured step reads at every replay.  Gradients are divided by
    ``grad_scale``; the step is cancelled where ``found_inf`` is not zero."""
    if len(params) != len(grads):
        raise ValueError(f"{len(params)} parameters but {len(grads)} gradients")
    if not params:
        return
    # (a network has hundreds of tensors: each look at all of them is one pass of a C function)
    device, dtype = params[0].device, _one(set(map(_dtype, params)), "dtypes of the parameters")
    require_cuda(params[0], "params")
    grad_dtype = _one(set(map(_dtype, grads)), "dtypes of the gradients")
    codes = dtype_code(dtype), dtype_code(grad_dtype)
    if set(map(Tensor.get_device, params)) != {device.index} or set(map(Tensor.get_device, grads)) != {device.index}:
        raise ValueError(f"all parameters and gradients must be on {device}")
    if not all(map(eq, map(_shape, params), map(_shape, grads))):
        raise ValueError("a gradient has another shape than its parameter")
    try:
        if not all(map(Tensor.is_contiguous, params)):
            raise ValueError("parameters must be contiguous: they are updated in place")
        if not all(map(Tensor.is_contiguous, grads)):
            grads = [g.detach().contiguous() for g in grads]
        at_params, at_grads = array("q", map(Tensor.data_ptr, params)), array("q", map(Tensor.data_ptr, grads))
    except (NotImplementedError, RuntimeError):
        if all(t.layout == torch.strided for t in chain(params, grads)):
            raise
        raise TypeError("parameters and gradients must be dense") from None
    sizes = array("q", map(Tensor.numel, params))
    length = _moments(exp_avg, exp_avg_sq, exp_avg_base, exp_avg_sq_base, device)
    for places, name in ((slots, "slots"), (step_index, "step_index")):
        if places is not None and len(places) != len(params):
            raise ValueError(f"{name} has {len(places)} places for {len(params)} tensors")
    if slots is not None:
        slots = array("q", slots)
        if any([s % BLOCK or s < 0 for s in slots]):
            raise ValueError(f"slots must be multiples of {BLOCK}")
    if step_index is not None:
        step_index = array("q", step_index)
        if min(step_index) < 0:
            raise ValueError("step_index must not be negative")
    if steps.dtype != torch.int32 or steps.device != device or not steps.is_contiguous():
        raise ValueError(f"steps must be contiguous int32 on {device}, got {steps.dtype} on {steps.device}")
    lr_at = None
    if isinstance(lr, Tensor):
        if lr.is_cuda:
            lr_at, lr = _scalar(lr, "lr", device), 0.0
        else:
            lr = float(lr)
    stream = stream_ptr(device)
    with on_device(device):
        status = lib().wcn_adamw_step(_at(at_params), _at(at_grads), _at(sizes), _at(slots), _at(step_index), len(params), *codes, ptr(exp_avg),
                                      ptr(exp_avg_base), ptr(exp_avg_sq), ptr(exp_avg_sq_base), length, ptr(steps), steps.numel(), _bits(lr),
                                      _bits(betas[0]), _bits(betas[1]), _bits(eps), _bits(weight_decay), lr_at,
                                      _scalar(grad_scale, "grad_scale", device), _scalar(found_inf, "found_inf", device),
                                      ptr(_counter(device, stream)), stream)
    count_training_launches("wcn_adamw_step")
    if status == _BOUNDS:
        raise ValueError(f"the tensors need more than the {length} elements of the moments or the {steps.numel()} of steps")
    check(status, "wcn_adamw_step")
    torch.autograd.graph.increment_version(params)


def decode_moments(exp_avg: Tensor, exp_avg_base: Tensor, exp_avg_sq: Tensor, exp_avg_sq_base: Tensor) -> Tuple[Tensor, Tensor]:
    """The numbers that 8-bit moments stand for, as flat fp32 tensors."""
    require_cuda(exp_avg, "exp_avg")
    device = exp_avg.device
    n = _moments(exp_avg, exp_avg_sq, exp_avg_base, exp_avg_sq_base, device)
    m, v = (torch.empty(n, dtype=torch.float32, device=device) for _ in range(2))
    with on_device(device):
        check(lib().wcn_adamw_decode(ptr(exp_avg), ptr(exp_avg_base), ptr(exp_avg_sq), ptr(exp_avg_sq_base), n, ptr(m), ptr(v),
                                     stream_ptr(device)), "wcn_adamw_decode")
    return m, v


def _check_rule(group: dict) -> None:
    """Flags of torch's optimizers for steps that this one does not make."""
    asked = [k for k, plain in (("maximize", False), ("amsgrad", False), ("decoupled_weight_decay", True)) if group.get(k, plain) != plain]
    if asked:
        raise ValueError(f"a group with {', '.join(f'{k}={group[k]}' for k in asked)} is not AdamW's")


def _beside(t: Optional[Tensor], p: Tensor) -> Optional[Tensor]:
    """``t`` on the device of ``p`` (a scaler has one number for all devices)."""
    return t if t is None or t.device == p.device else t.to(p.device, non_blocking=True)


class _Arena:
    """The flat moments and step counts of some parameters."""

    def __init__(self, params: Sequence[Tensor], bits: int):
        device = params[0].device
        slots, length = moment_slots([p.numel() for p in params])
        dtype = torch.float32 if bits == 32 else torch.uint8
        self.exp_avg, self.exp_avg_sq = (torch.zeros(length, dtype=dtype, device=device) for _ in range(2))
        self.exp_avg_base = self.exp_avg_sq_base = None
        if bits == 8:
            self.exp_avg_base, self.exp_avg_sq_base = (torch.zeros(length // BLOCK, dtype=torch.int16, device=device) for _ in range(2))
        self.steps = torch.zeros(len(params), dtype=torch.int32, device=device)
        self.place = {p: (i, s) for i, (p, s) in enumerate(zip(params, slots))}

    def state(self, p: Tensor) -> dict:
        """Views of what is kept for a parameter."""
        i, s = self.place[p]
        blocks = -(-p.numel() // BLOCK)
        if self.exp_avg_base is None:
            return {"step": self.steps[i], "exp_avg": self.exp_avg[s:s + p.numel()].view(p.shape), "exp_avg_sq": self.exp_avg_sq[s:s + p.numel()].view(p.shape)}
        base = slice(s // BLOCK, s // BLOCK + blocks)
        return {"step": self.steps[i], "exp_avg": self.exp_avg[s:s + blocks * BLOCK], "exp_avg_base": self.exp_avg_base[base],
                "exp_avg_sq": self.exp_avg_sq[s:s + blocks * BLOCK], "exp_avg_sq_base": self.exp_avg_sq_base[base]}


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` as one launch per group and dtype.

    ``state_bits``: 32, or 8 for moments of a byte each (a quarter of the memory, and 16 instead of 28 bytes of traffic per
    fp32 parameter).  The moments live in flat tensors; ``state[p]`` are views of them.  Nothing is read back to the host:
    steps can be captured in a CUDA graph (with a float32 device tensor as ``lr`` where that changes), and ``torch.amp.GradScaler``
    hands its scale and its infinity flag to the kernel.  Parameters are float32, float16 or bfloat16, contiguous and on CUDA
    devices at the first step."""

    _step_supports_amp_scaling = True

    def __init__(self, params, lr: Union[float, Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, state_bits: int = 32):
        if not isinstance(lr, Tensor) and not 0.0 <= lr:
            raise ValueError(f"invalid learning rate: {lr}")
        if isinstance(lr, Tensor) and lr.numel() != 1:
            raise ValueError("a learning rate is one number")
        if not 0.0 <= eps:
            raise ValueError(f"invalid epsilon: {eps}")
        if not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"invalid betas: {betas}")
        if not 0.0 <= weight_decay:
            raise ValueError(f"invalid weight decay: {weight_decay}")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits is 8 or 32, got {state_bits}")
        self._arena_of: dict = {}
        self.state_bits = state_bits
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits))

    def add_param_group(self, group):
        super().add_param_group(group)
        try:
            if self.param_groups[-1]["state_bits"] != self.state_bits:
                raise ValueError(f"all groups of this optimizer have moments of {self.state_bits} bits")
            _check_rule(self.param_groups[-1])
        except ValueError:
            self.param_groups.pop()
            raise

    def _rooms(self, params: Sequence[Tensor]) -> dict:
        """``{parameter: its arena}``, new ones."""
        by_device: dict = {}
        for p in params:
            by_device.setdefault(p.device, []).append(p)
        return {p: arena for group in by_device.values() for arena in (_Arena(group, self.state_bits),) for p in group}

    def _make_room(self, params: Sequence[Tensor]) -> None:
        """Moments for the parameters that have none."""
        for p, arena in self._rooms(params).items():
            self._arena_of[p] = arena
            self.state[p] = arena.state(p)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        scale, found = getattr(self, "grad_scale", None), getattr(self, "found_inf", None)
        for group in self.param_groups:
            buckets: dict = {}
            params = [p for p in group["params"] if p.grad is not None]
            missing = [p for p in params if p not in self._arena_of]
            if missing:
                self._make_room([p for p in group["params"] if p not in self._arena_of])
            for p in params:
                buckets.setdefault((id(self._arena_of[p]), p.dtype, p.grad.dtype), []).append(p)
            for (_, _, _), some in buckets.items():
                arena = self._arena_of[some[0]]
                places = [arena.place[p] for p in some]
                adamw_step(some, [p.grad for p in some], arena.exp_avg, arena.exp_avg_sq, arena.steps, lr=group["lr"], betas=group["betas"],
                           eps=group["eps"], weight_decay=group["weight_decay"], exp_avg_base=arena.exp_avg_base,
                           exp_avg_sq_base=arena.exp_avg_sq_base, slots=[s for _, s in places], step_index=[i for i, _ in places],
                           grad_scale=_beside(scale, some[0]), found_inf=_beside(found, some[0]))
        return loss

    # -- what is kept travels as the views of ``state``: copies are put into flat tensors again

    def _filled(self, state: dict) -> dict:
        """``{parameter: its arena}`` with the moments and steps of ``{parameter: entries}``; what is kept so far stays as it is."""
        known = [p for g in self.param_groups for p in g["params"] if p in state]
        for p in known:
            if not p.is_cuda:
                raise ValueError("move the parameters to their device before their optimizer's state is loaded")
        rooms = self._rooms(known)
        for p in known:
            mine = rooms[p].state(p)
            if set(mine) != set(state[p]):
                raise ValueError(f"state with {sorted(state[p])} cannot be loaded into an optimizer with moments of {self.state_bits} bits")
            for name, view in mine.items():
                value = torch.as_tensor(state[p][name])
                if value.numel() != view.numel():
                    raise ValueError(f"{name} of a parameter with {p.numel()} elements has {value.numel()}")
                view.copy_(value.to(view.device).view(view.shape))
        return rooms

    def _put(self, rooms: dict) -> None:
        """Arenas in the place of those so far."""
        self._arena_of = rooms
        self.state.clear()
        for p, arena in rooms.items():
            self.state[p] = arena.state(p)

    def load_state_dict(self, state_dict):
        """Takes the state of an optimizer of this class with the same ``state_bits``, and with 32 bits one of ``torch.optim.AdamW``.
        A state that is refused leaves everything as it was."""
        saved = state_dict["param_groups"]
        if len(saved) != len(self.param_groups):
            raise ValueError("loaded state dict has a different number of parameter groups")
        if any(len(own["params"]) != len(g["params"]) for own, g in zip(self.param_groups, saved)):
            raise ValueError("loaded state dict contains a parameter group that doesn't match the size of optimizer's group")
        bits = {g.get("state_bits", 32) for g in saved}
        if bits - {self.state_bits}:
            raise ValueError(f"moments of {sorted(bits)} bits cannot be loaded into an optimizer with moments of {self.state_bits} bits")
        for g in saved:
            _check_rule(g)
        params = [p for g in self.param_groups for p in g["params"]]
        names = [i for g in saved for i in g["params"]]
        rooms = self._filled({p: state_dict["state"][i] for p, i in zip(params, names) if i in state_dict["state"]})
        groups = [{**{k: v for k, v in own.items() if k != "params"}, **g} for own, g in zip(self.param_groups, saved)]
        super().load_state_dict({"state": {}, "param_groups": groups})
        self._put(rooms)

    def __setstate__(self, state):
        super().__setstate__(state)
        self.state_bits = self.defaults["state_bits"]
        self._arena_of = {}
        if "state" in state:
            self._put(self._filled({p: dict(entries) for p, entries in self.state.items()}))
