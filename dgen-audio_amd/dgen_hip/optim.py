"""The optimiser's step on device tensors (include/dgen_hip.h, "optimiser step
on device tensors"): AdamW over all of a model's tensors in one launch for each
fifty-two of them.

``adamw`` is one step from tensors to tensors; :class:`AdamW` keeps a model's
moments and steps in place.  Tensors are contiguous torch tensors on one GPU;
work is enqueued on torch's current stream and the calls return without
waiting.  A wrong argument raises ``ValueError``, a failing launch ``HIPError``.

The reference's Adam (Sources/DGenLazy/Optimizers.swift:164-204) has no weight
decay and no bound on the gradients' norm.
"""
from __future__ import annotations

import ctypes
import operator
import struct
from typing import Optional, Sequence

import torch

from . import sequence as Q
from .runtime import load_library
from .sequence import HIPError

try:
    from ._tensor_args import table
except ImportError:  # the library was built without PyTorch's headers: the same in Python
    from ._tensor_args_python import table

_ADAMW = struct.Struct("@Iiq Q dddddd q Q Q")  # struct dgen_hip_adamw, but for the workspace
_ADAMW_SIZE = _ADAMW.size + 16
_F32, _BF16 = 0, 1
_NAMES = ("params", "grads", "exp_avg", "exp_avg_sq", "out[0]", "out[1]", "out[2]", "copies")


def _table(lists, types, device) -> bytes:
    """The tensors' addresses and sizes, or what is wrong with one."""
    rows = []
    for name, tensors in zip(_NAMES, lists):
        if tensors is not None and len(tensors) != len(lists[0]):
            raise ValueError(f"{name}: {len(lists[0])} tensors expected, got {len(tensors)}")
    for k, like in enumerate(lists[0]):
        row = []
        if not isinstance(like, torch.Tensor):
            raise Q._wrong(f"params[{k}]", like, "a float32 tensor")
        for name, ty, tensors in zip(_NAMES, types, lists):
            want = torch.bfloat16 if ty == _BF16 else torch.float32
            if tensors is None:
                row.append(0)
                continue
            t = tensors[k]
            if t is None and name == "copies":
                row.append(0)
                continue
            if not isinstance(t, torch.Tensor) or t.dtype is not want or t.shape != like.shape or t.device != device:
                raise Q._wrong(f"{name}[{k}]", t, f"{tuple(like.shape)} {want} on {device}")
            if not t.is_contiguous():
                raise ValueError(f"{name}[{k}]: must be contiguous")
            row.append(t.data_ptr())
        rows.append(struct.pack(f"@{len(row)}Qq", *row, like.numel()))
    return b"".join(rows)


def _list(x, name: str):
    try:
        return None if x is None else list(x)
    except TypeError:
        raise ValueError(f"{name}: a list of tensors expected, got {type(x).__name__}") from None


def _whole(step) -> int:
    """A count of steps that the descriptor holds (its size is tested there)."""
    try:
        n = int(step) if isinstance(step, float) and step.is_integer() else operator.index(step)
    except TypeError:
        n = -1
    if not 0 <= n < 1 << 63:
        raise ValueError(f"step {step!r}: a whole number from 1 on, or one int64 on the device, expected")
    return n


def adamw(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avg: Sequence[torch.Tensor],
          exp_avg_sq: Sequence[torch.Tensor], step, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999),
          eps: float = 1e-8, weight_decay: float = 1e-2, max_norm: Optional[float] = None,
          copies: Optional[Sequence[torch.Tensor]] = None, out=None) -> Optional[torch.Tensor]:
    """One step of AdamW over float32 ``params`` with their moments ``exp_avg``
    and ``exp_avg_sq`` (float32) and ``grads`` (all float32 or all bfloat16).
    ``step`` counts from 1: a number, or an int64 tensor on the device, which is
    read when the work runs (for a step that is captured and replayed).

        m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2
        p = (1 - lr weight_decay) p - lr (m / (1 - beta1^step)) / (sqrt(v / (1 - beta2^step)) + eps)

    Results replace params and moments, or go to ``out`` (three lists: params,
    exp_avg, exp_avg_sq).  ``copies`` (bfloat16, or None for a tensor without
    one) receive the new params rounded, for the next pass.  With ``max_norm`` the gradients are scaled by min(1,
    max_norm / (norm + 1e-6)), and the result is their norm before that, on the
    device; else None."""
    out = (params, exp_avg, exp_avg_sq) if out is None else _list(out, "out")
    if len(out) != 3:
        raise ValueError("out: three lists expected")
    lists = [_list(x, name) for x, name in zip((params, grads, exp_avg, exp_avg_sq, *out, copies), _NAMES)]
    if not lists[0]:
        raise ValueError("params: no tensors")
    Q._type(lists[0][0], "params[0]")
    dev = lists[0][0].device
    half = bool(lists[1]) and isinstance(lists[1][0], torch.Tensor) and lists[1][0].dtype is torch.bfloat16
    types = (_F32, _BF16 if half else _F32, _F32, _F32, _F32, _F32, _F32, _BF16)
    rows = table(tuple(lists), types, dev.index) or _table(lists, types, dev)
    at = 0
    if isinstance(step, torch.Tensor):
        if step.dtype is not torch.int64 or step.numel() != 1 or step.device != dev:
            raise Q._wrong("step", step, f"a number, or one int64 on {dev}")
        at, step = step.data_ptr(), 0
    else:
        step = _whole(step)
    bound = 0.0 if max_norm is None else Q._number(max_norm, "max_norm")
    if max_norm is not None and not bound > 0:
        raise ValueError(f"max_norm {max_norm}: a positive number expected")
    norm = torch.empty((), dtype=torch.float32, device=dev) if bound else None
    betas = _list(betas, "betas")
    if betas is None or len(betas) != 2:
        raise ValueError("betas: two numbers expected")
    numbers = [Q._number(x, name) for x, name in zip((lr, *betas, eps, weight_decay), ("lr", "betas[0]", "betas[1]", "eps", "weight_decay"))]
    # (the rows of dgen_hip_adamw_tensor, copies before the number of elements)
    host = ctypes.create_string_buffer(rows, len(rows))
    d = _ADAMW.pack(_ADAMW_SIZE, types[1], len(lists[0]), ctypes.addressof(host), *numbers, bound, step, at,
                    0 if norm is None else norm.data_ptr())
    _run(d, dev, norm is not None)
    return norm


def _run(d: bytes, dev: torch.device, scratch: bool) -> None:
    L, tail = _library(), Q._NO_WORKSPACE
    if scratch:
        need = ctypes.c_uint64(0)
        _check(L, L.dgen_hip_adamw_workspace(dev.index, d + tail, ctypes.byref(need)))
        if need.value:
            ws = torch.empty(need.value, dtype=torch.uint8, device=dev)
            tail = Q._WORKSPACE.pack(ws.data_ptr(), need.value)
    _check(L, L.dgen_hip_adamw_step(dev.index, d + tail, Q._raw_stream(dev.index)))


def _check(L, rc: int) -> None:
    if rc:
        raise (ValueError if rc in (-1, -4) else HIPError)(L.dgen_hip_last_error().decode(errors="replace"))


def _library() -> ctypes.CDLL:
    Q._op("rms_norm")  # (refuses a second HIP runtime)
    return load_library()


class AdamW:
    """AdamW over a model's float32 tensors, in place: their moments, the count
    of steps, and ``copies`` (bfloat16, one for each tensor or None) that are
    kept equal to the rounded parameters, from the start on.  The count lies on the device, so a
    captured step counts on when it is replayed."""

    def __init__(self, params: Sequence[torch.Tensor], lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, max_norm: Optional[float] = None,
                 copies: Optional[Sequence[torch.Tensor]] = None):
        self.params, self.copies = list(params), None if copies is None else list(copies)
        if not self.params:
            raise ValueError("params: no tensors")
        if self.copies is not None:
            self._fill()
        self.lr, self.betas, self.eps, self.weight_decay, self.max_norm = lr, betas, eps, weight_decay, max_norm
        self.exp_avg, self.exp_avg_sq = ([torch.zeros_like(p) for p in self.params] for _ in range(2))
        self.count = torch.zeros((), dtype=torch.int64, device=self.params[0].device)

    @torch.no_grad()
    def _fill(self) -> None:
        """The copies, for a pass before the first step."""
        if len(self.copies) != len(self.params):
            raise ValueError(f"copies: {len(self.params)} tensors expected, got {len(self.copies)}")
        for k, (p, c) in enumerate(zip(self.params, self.copies)):
            if c is not None and (not isinstance(c, torch.Tensor) or c.dtype is not torch.bfloat16 or c.shape != p.shape):
                raise Q._wrong(f"copies[{k}]", c, f"{tuple(p.shape)} {torch.bfloat16}")
        for p, c in zip(self.params, self.copies):
            if c is not None:
                c.copy_(p)

    @torch.no_grad()
    def step(self, grads: Sequence[torch.Tensor]) -> Optional[torch.Tensor]:
        """One step; the gradients' norm where it is held to a bound.  A step that
        is refused does not count."""
        self.count += 1
        try:
            return adamw(self.params, grads, self.exp_avg, self.exp_avg_sq, self.count, self.lr, self.betas, self.eps,
                         self.weight_decay, self.max_norm, self.copies)
        except Exception:
            self.count -= 1
            raise
