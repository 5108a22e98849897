"""Sequence operators on device tensors: the parts of a recurrent control
decoder (include/dgen_hip.h, "sequence operators on device tensors").

- ``rms_norm`` / ``rms_norm_backward``: root-mean-square norm with the
  residual's addition;
- ``causal_conv`` / ``causal_conv_backward``: short depthwise causal
  convolution with SiLU;
- ``selective_scan`` / ``selective_scan_backward``: selective state space scan
  with skip and gate;
- ``gated_mlp`` / ``gated_mlp_backward``: gated feed-forward block.

Tensors are torch tensors on one GPU (float32 or bfloat16; parameters of the
first three float32), possibly views of wider ones: the last axis is
contiguous, and batch and time have any stride, as rows have (leading axes of
the norms and the gated block that are one axis of rows).  Work is enqueued on
torch's current stream and the calls return without waiting; results and
scratch come from torch's allocator on that stream.  Nothing is recorded for
autograd: a program calls the backward functions itself, and an operand that
requires a gradient brings a warning unless gradients are switched off.  A
wrong argument raises ``ValueError``, a failing launch ``HIPError``.

Results that the caller gives a place for (``out``, ``sum_out``, ``state_out``)
may lie over the operands: where the operator would overwrite what it still
reads, it writes to a tensor of its own, which is copied there afterwards.
What may be replaced in place without one: x, residual, ds, s and dy in the
norms, x, dt and z in the scan, the state by ``state_out``.  Two results must
not share memory.

Clips of unequal length: ``lengths`` ([batch] int32) ends each sequence; later
frames are not read, and their outputs and gradients are 0.  Streaming: the
state that a call leaves (``state_out``) is the next call's ``state``, the
same tensor if wanted; a call with one frame is the form for live voices.

No counterpart in the reference, whose decoder sees one frame at a time
(Examples/HarmonicE2E/Model.swift:96-120).
"""
from __future__ import annotations

import ctypes
import os
import struct
import sys
import warnings
from typing import NamedTuple, Optional

import torch

from .runtime import HIPError, load_library

try:
    from ._tensor_args import covers, dense, rows, sequence
except ImportError:  # the library was built without PyTorch's headers: the same in Python
    from ._tensor_args_python import covers, dense, rows, sequence

_TYPES = {torch.float32: 0, torch.bfloat16: 1}
_F32, _INT32 = 0, 2  # as the native tests name them
_ACTS = {"silu": 0, "gelu": 1}


def _descriptor(fields: str) -> struct.Struct:
    """A descriptor of dgen_hip.h in native layout but for its last two
    fields, the workspace's address and size.  p: address, v: address and
    stride of rows, s: address and two strides of a sequence tensor."""
    return struct.Struct("@" + fields.replace("p", "Q").replace("v", "Qq").replace("s", "Qqq"))


# (packed as bytes: a ctypes structure took 3 us more a call)
_NORM = _descriptor("Iiif qq p v v v v v v v p")           # struct dgen_hip_norm
_CONV = _descriptor("Iiii qqq ppp s s pp s s pp")          # struct dgen_hip_conv
_SCAN = _descriptor("Ii qqqq pppppp ssssssssssss ppp")     # struct dgen_hip_scan
_MLP = _descriptor("Iiii qqq vvvvvvvv")                    # struct dgen_hip_mlp
_WORKSPACE = struct.Struct("@QQ")
_NO_WORKSPACE = _WORKSPACE.pack(0, 0)
# the descriptors' struct_size
_NORM_SIZE, _CONV_SIZE, _SCAN_SIZE, _MLP_SIZE = (d.size + 16 for d in (_NORM, _CONV, _SCAN, _MLP))
_NONE, _NO_ROWS = (0, 0, 0), (0, 0)


def _current_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# (the same handle without a Stream object: 0.1 instead of 2 us a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _current_stream)


def _one_runtime(L: ctypes.CDLL) -> bool:
    """Whether the library and PyTorch call the same HIP runtime.  PyTorch
    brings its own, which the library uses too if that is there first; if the
    library comes first it takes the system's, and PyTorch loads a second one."""
    try:
        theirs = ctypes.CDLL("libc10_hip.so", mode=os.RTLD_NOW | os.RTLD_NOLOAD)
        a, b = (ctypes.cast(lib.hipGetDevice, ctypes.c_void_p).value for lib in (L, theirs))
    except (OSError, AttributeError):  # a PyTorch without HIP has no tensors to pass
        return True
    return a == b


class _Op:
    """One operator's C entries."""

    def __init__(self, name: str):
        L = load_library()
        if not _one_runtime(L):
            raise HIPError("two HIP runtimes in this process: PyTorch's streams and memory are unknown to the one that the "
                           "library uses; import torch (or dgen_hip.sequence) before the library is loaded")
        self.forward, self.backward = getattr(L, f"dgen_hip_{name}"), getattr(L, f"dgen_hip_{name}_backward")
        self.workspace = getattr(L, f"dgen_hip_{name}_workspace")
        self.error = L.dgen_hip_last_error

    def __call__(self, desc: bytes, device: torch.device, backward: bool, scratch: bool) -> None:
        index, tail = device.index, _NO_WORKSPACE
        if scratch:
            need = ctypes.c_uint64(0)
            self._check(self.workspace(index, desc + tail, int(backward), ctypes.byref(need)))
            if need.value:
                ws = torch.empty(need.value, dtype=torch.uint8, device=device)
                tail = _WORKSPACE.pack(ws.data_ptr(), need.value)
        rc = (self.backward if backward else self.forward)(index, desc + tail, _raw_stream(index))
        if rc:
            self._check(rc)

    def _check(self, rc: int) -> None:
        if rc:
            msg = self.error().decode(errors="replace")
            raise (ValueError if rc in (-1, -4) else HIPError)(msg)


_OPS: dict[str, _Op] = {}


def _op(name: str) -> _Op:
    op = _OPS.get(name)
    if op is None:
        op = _OPS[name] = _Op(name)
    return op


def _wrong(name: str, t, want: str):
    got = f"{tuple(t.shape)} {t.dtype} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
    return ValueError(f"{name}: {want} expected, got {got}")


def _type(x, name: str) -> int:
    ty = _TYPES.get(x.dtype) if isinstance(x, torch.Tensor) and x.is_cuda else None
    if ty is None:
        raise _wrong(name, x, "a float32 or bfloat16 tensor on a GPU")
    return ty


# Tests of an argument: dense, rows and sequence (csrc/tensor_args.cpp) give its
# address and strides; what they turn down comes to the functions here, which
# say what is wrong with it, or take it after all.
def _is(t, name: str, shape, dtype, device) -> bool:
    try:
        if not (t.dtype is dtype and t.shape == shape and t.device == device):
            return False
    except AttributeError:  # not a tensor
        return False
    if t.requires_grad and torch.is_grad_enabled():
        caller, up = sys._getframe(1), 2
        while caller.f_back and caller.f_code.co_filename == __file__:
            caller, up = caller.f_back, up + 1
        warnings.warn(f"{name} requires a gradient, which the sequence operators do not record: call them under "
                      "torch.no_grad() and their backward functions, or give them detached tensors", stacklevel=up)
    return True


def _seq(t, name: str, shape, dtype, device):
    """(address, batch stride, time stride) of a [batch][time][channel] tensor."""
    if not _is(t, name, shape, dtype, device):
        raise _wrong(name, t, f"{tuple(shape)} {dtype} on {device}")
    sb, st, sc = t.stride()
    if sc != 1 and shape[2] != 1:
        raise ValueError(f"{name}: the last axis must be contiguous")
    return t.data_ptr(), sb, st


def _dense(t, name: str, shape, dtype, device):
    """Address of a contiguous tensor (0 for None)."""
    if t is None:
        return 0
    if not _is(t, name, shape, dtype, device):
        raise _wrong(name, t, f"{tuple(shape)} {dtype} on {device}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")
    return t.data_ptr()


def _rows(t, name: str, shape, dtype, device):
    """(address, row stride) of a tensor whose leading axes are rows."""
    if not _is(t, name, shape, dtype, device):
        raise _wrong(name, t, f"{tuple(shape)} {dtype} on {device}")
    if len(shape) != 2:
        if t.is_contiguous():
            return t.data_ptr(), shape[-1]
        try:
            t = t.view(-1, shape[-1])
        except RuntimeError:
            raise ValueError(f"{name}: its leading axes must be one axis of rows (contiguous, or a view of rows)") from None
    rs, cs = t.stride()
    if cs != 1 and shape[-1] != 1:
        raise ValueError(f"{name}: the last axis must be contiguous")
    return t.data_ptr(), rs


def _fresh(like, out, name: str, shape):
    """A result in rows, given or made: the tensor, its address and row stride
    (one that is made here needs no test)."""
    if out is None:
        out = torch.empty_like(like, memory_format=torch.contiguous_format)
        return out, (out.data_ptr(), shape[-1])
    return out, (rows(out, shape, _TYPES[like.dtype], like.get_device())
                 or _rows(out, name, shape, like.dtype, like.device))


def _fresh_seq(like, out, shape):
    """The same of a sequence tensor."""
    if out is None:
        out = torch.empty_like(like, memory_format=torch.contiguous_format)
        return out, (out.data_ptr(), shape[1] * shape[2], shape[2])
    return out, (sequence(out, shape, _TYPES[like.dtype], like.get_device())
                 or _seq(out, "out", shape, like.dtype, like.device))


def _given(target, written):
    """A result in the place that the caller gave."""
    return written if target is written else target.copy_(written)


def _two_results(a: str, x, b: str, y) -> None:
    if y is not None and covers(0, x, y):
        raise ValueError(f"{a} and {b}: the two results share memory")


def _count(shape) -> int:
    n = 1
    for s in shape[:-1]:
        n *= s
    return n


# -------------------------------------------------------------------- norm
def rms_norm(x, weight, residual=None, eps: float = 1e-5, out=None, sum_out=None):
    """y = s / sqrt(mean(s^2) + eps) * weight over the last axis, s = x +
    residual.  Without a residual, s = x and the result is y; with one (of x's
    type or float32) the result is (y, s), s in the residual's type, ready to be
    the next residual.  ``sum_out`` may be the residual itself."""
    ty, shape, dev = _type(x, "x"), x.shape, x.device
    if x.dim() < 1:
        raise _wrong("x", x, "at least one axis")
    if x.dim() == 1:
        raise _wrong("x", x, "rows ([..., width])")
    i = dev.index
    xp = rows(x, shape, ty, i) or _rows(x, "x", shape, x.dtype, dev)
    w = dense(weight, shape[-1:], _F32, i) or _dense(weight, "weight", shape[-1:], torch.float32, dev)
    y, yp = _fresh(x, out, "out", shape)
    rp = sp = _NO_ROWS
    st = ty
    if residual is not None:
        st = _type(residual, "residual")
        rp = rows(residual, shape, st, i) or _rows(residual, "residual", shape, residual.dtype, dev)
        s, sp = _fresh(residual, sum_out, "sum_out", shape)
        if sum_out is not None and covers(2, s, residual, x, weight):
            s, sp = _fresh(residual, None, "sum_out", shape)
    elif sum_out is not None:
        raise ValueError("sum_out: only with a residual")
    if out is not None:
        _two_results("out", out, "sum_out", sum_out)
        if covers(2, out, x, residual, weight):
            y, yp = _fresh(x, None, "out", shape)
    d = _NORM.pack(_NORM_SIZE, ty, st, eps, _count(shape), shape[-1], w, *xp, *rp, *yp, *sp, 0, 0, 0, 0, 0, 0, 0)
    _op("rms_norm")(d, dev, False, False)
    if out is not None:
        y = _given(out, y)
    if residual is None:
        return y
    return y, s if sum_out is None else _given(sum_out, s)


def rms_norm_backward(dy, s, weight, ds=None, eps: float = 1e-5, out=None):
    """(dx, dweight) from the gradient of y and the stored sum ``s`` (x itself
    where there was no residual).  dx, in the sum's type, is the gradient of x
    and of the residual alike; ``ds``, the gradient that reaches the stored sum
    from elsewhere, is added to it."""
    ty, st, shape, dev = _type(dy, "dy"), _type(s, "s"), s.shape, s.device
    if s.dim() < 2:
        raise _wrong("s", s, "rows ([..., width])")
    i, width = dev.index, shape[-1:]
    dx, op = _fresh(s, out, "out", shape)
    if out is not None and covers(3, out, s, dy, ds, weight):
        dx, op = _fresh(s, None, "out", shape)
    dw = s.new_empty(shape[-1], dtype=torch.float32)
    d = _NORM.pack(_NORM_SIZE, ty, st, eps, _count(shape), shape[-1],
                   dense(weight, width, _F32, i) or _dense(weight, "weight", width, torch.float32, dev),
                   0, 0, 0, 0, 0, 0, *(rows(s, shape, st, i) or _rows(s, "s", shape, s.dtype, dev)),
                   *(rows(dy, shape, ty, i) or _rows(dy, "dy", shape, dy.dtype, dev)),
                   *(_NO_ROWS if ds is None else rows(ds, shape, st, i) or _rows(ds, "ds", shape, s.dtype, dev)),
                   *op, dw.data_ptr())
    _op("rms_norm")(d, dev, True, True)
    return (dx if out is None else _given(out, dx)), dw


# -------------------------------------------------------------- convolution
def _conv_parts(x, weight, bias, state, lengths):
    ty = _type(x, "x")
    if x.dim() != 3:
        raise _wrong("x", x, "[batch][time][channel]")
    B, T, D = shape = x.shape
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise _wrong("weight", weight, "[channel][width]")
    W, dev, f32, before = weight.shape[1], x.device, torch.float32, (B, weight.shape[1] - 1, D)
    i = dev.index
    head = (ty, (B, T, D), dense(weight, (D, W), _F32, i) or _dense(weight, "weight", (D, W), f32, dev),
            dense(bias, (D,), _F32, i) or _dense(bias, "bias", (D,), f32, dev),
            dense(lengths, (B,), _INT32, i) or _dense(lengths, "lengths", (B,), torch.int32, dev),
            sequence(x, shape, ty, i) or _seq(x, "x", shape, x.dtype, dev),
            dense(state, before, ty, i) or _dense(state, "state", before, x.dtype, dev))
    return W, dev, head


def causal_conv(x, weight, bias=None, silu: bool = True, state=None, state_out=None, lengths=None, out=None):
    """y[t] = silu(bias + sum_i weight[:, i] x[t - W + 1 + i]) per channel of
    x [batch][time][D], weight [D][W] (W up to 8).  The frames before the
    first are ``state`` ([batch][W-1][D], x's type, oldest first) or 0;
    ``state_out`` receives the last W-1 frames of each sequence.  A call takes
    up to 65535 sequences."""
    W, dev, (ty, (B, T, D), w, b, n, xs, st) = _conv_parts(x, weight, bias, state, lengths)
    y, ys = _fresh_seq(x, out, x.shape)
    if out is not None:
        _two_results("out", out, "state_out", state_out)
        if covers(0, out, x, weight, bias, state, lengths):
            y, ys = _fresh_seq(x, None, x.shape)
    after, left = (B, W - 1, D), state_out
    so = dense(state_out, after, ty, dev.index) or _dense(state_out, "state_out", after, x.dtype, dev)
    if so and covers(1, state_out, state, x, weight, bias, lengths):
        left = torch.empty_like(state_out)
        so = left.data_ptr()
    d = _CONV.pack(_CONV_SIZE, ty, 1 if silu else 0, W, B, T, D, w, b, n, *xs, *ys, st, so, 0, 0, 0, 0, 0, 0, 0, 0)
    _op("causal_conv")(d, dev, False, False)
    if left is not state_out:
        state_out.copy_(left)
    return y if out is None else _given(out, y)


def causal_conv_backward(dy, x, weight, bias=None, silu: bool = True, state=None, lengths=None, out=None):
    """(dx, dweight, dbias) of ``causal_conv`` (dbias None without a bias);
    the state counts as given."""
    W, dev, (ty, (B, T, D), w, b, n, xs, st) = _conv_parts(x, weight, bias, state, lengths)
    dx, ds = _fresh_seq(x, out, x.shape)
    if out is not None and covers(0, out, dy, x, weight, bias, state, lengths):
        dx, ds = _fresh_seq(x, None, x.shape)
    dw = weight.new_empty((D, W))
    db = None if bias is None else bias.new_empty(D)
    d = _CONV.pack(_CONV_SIZE, ty, 1 if silu else 0, W, B, T, D, w, b, n, *xs, 0, 0, 0, st, 0,
                   *(sequence(dy, x.shape, ty, dev.index) or _seq(dy, "dy", x.shape, x.dtype, dev)), *ds,
                   dw.data_ptr(), 0 if db is None else db.data_ptr())
    _op("causal_conv")(d, dev, True, True)
    return (dx if out is None else _given(out, dx)), dw, db


# --------------------------------------------------------------------- scan
class ScanGrads(NamedTuple):
    """Gradients of ``selective_scan``; None for what was not given."""
    dx: torch.Tensor
    ddt: torch.Tensor
    dA: torch.Tensor
    dB: torch.Tensor
    dC: torch.Tensor
    dD: Optional[torch.Tensor]
    dz: Optional[torch.Tensor]
    ddt_bias: Optional[torch.Tensor]


def _scan_parts(x, dt, A, B, C, D, z, dt_bias, state, lengths):
    """(device, sizes, the descriptor's first fields, those of the inputs)."""
    ty = _type(x, "x")
    if x.dim() != 3:
        raise _wrong("x", x, "[batch][time][channel]")
    if not isinstance(A, torch.Tensor) or A.dim() != 2:
        raise _wrong("A", A, "[channel][state]")
    shape, dev, f32, et = x.shape, x.device, torch.float32, x.dtype
    n, T, ch = shape
    N = A.shape[1]
    bc, per, states, i = (n, T, N), (ch,), (n, ch, N), dev.index
    head = (_SCAN_SIZE, ty, n, T, ch, N, dense(A, (ch, N), _F32, i) or _dense(A, "A", (ch, N), f32, dev),
            dense(D, per, _F32, i) or _dense(D, "D", per, f32, dev),
            dense(dt_bias, per, _F32, i) or _dense(dt_bias, "dt_bias", per, f32, dev),
            dense(lengths, (n,), _INT32, i) or _dense(lengths, "lengths", (n,), torch.int32, dev),
            dense(state, states, _F32, i) or _dense(state, "state", states, f32, dev))
    return dev, (n, T, ch, N), head, (*(sequence(x, shape, ty, i) or _seq(x, "x", shape, et, dev)),
                                      *(sequence(dt, shape, ty, i) or _seq(dt, "dt", shape, et, dev)),
                                      *(_NONE if z is None else
                                        sequence(z, shape, ty, i) or _seq(z, "z", shape, et, dev)),
                                      *(sequence(B, bc, ty, i) or _seq(B, "B", bc, et, dev)),
                                      *(sequence(C, bc, ty, i) or _seq(C, "C", bc, et, dev)))


_NO_SCAN_GRADS = (0,) * 21


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, state=None, state_out=None, lengths=None, out=None):
    """The selective scan over x [batch][time][channels]: with step =
    softplus(dt + dt_bias), h[t] = exp(step A) h[t-1] + step x[t] B[t] per
    channel ([channels][N] states, N up to 64), y[t] = (C[t].h[t] + D x[t])
    silu(z[t]).  B and C are [batch][time][N]; A, D, dt_bias and the states
    ([batch][channels][N]) are float32; D, z and dt_bias may be left out.
    Results of a sequence can differ in rounding with the number of sequences
    and channels in the call, which decide how time is cut."""
    dev, (n, T, ch, N), head, ins = _scan_parts(x, dt, A, B, C, D, z, dt_bias, state, lengths)
    y, ys = _fresh_seq(x, out, x.shape)
    if out is not None:
        _two_results("out", out, "state_out", state_out)
        if covers(3, out, x, dt, z, A, B, C, D, dt_bias, state, lengths):
            y, ys = _fresh_seq(x, None, x.shape)
    after, left = (n, ch, N), state_out
    so = dense(state_out, after, _F32, dev.index) or _dense(state_out, "state_out", after, torch.float32, dev)
    if so and covers(1, state_out, state, x, dt, z, A, B, C, D, dt_bias, lengths):
        left = torch.empty_like(state_out)
        so = left.data_ptr()
    d = _SCAN.pack(*head, so, *ins, *ys, *_NO_SCAN_GRADS)
    # (a call of few frames is one launch without scratch)
    _op("selective_scan")(d, dev, False, T > 32)
    if left is not state_out:
        state_out.copy_(left)
    return y if out is None else _given(out, y)


def selective_scan_backward(dy, x, dt, A, B, C, D=None, z=None, dt_bias=None, state=None, lengths=None) -> ScanGrads:
    """Gradients of ``selective_scan``; the state counts as given."""
    dev, (n, T, ch, N), head, ins = _scan_parts(x, dt, A, B, C, D, z, dt_bias, state, lengths)

    def new(like):
        return None if like is None else torch.empty_like(like, memory_format=torch.contiguous_format)

    g = ScanGrads(new(x), new(dt), new(A), new(B), new(C), new(D), new(z), new(dt_bias))
    wide, narrow = (T * ch, ch), (T * N, N)
    d = _SCAN.pack(*head, 0, *ins, 0, 0, 0,
                   *(sequence(dy, x.shape, head[1], dev.index) or _seq(dy, "dy", x.shape, x.dtype, dev)), g.dx.data_ptr(), *wide,
                   g.ddt.data_ptr(), *wide, *(_NONE if g.dz is None else (g.dz.data_ptr(), *wide)), g.dB.data_ptr(),
                   *narrow, g.dC.data_ptr(), *narrow, g.dA.data_ptr(), 0 if g.dD is None else g.dD.data_ptr(),
                   0 if g.ddt_bias is None else g.ddt_bias.data_ptr())
    _op("selective_scan")(d, dev, True, True)
    return g


# ------------------------------------------------------ gated feed-forward
def _mlp_parts(x, w_gate, w_up, activation):
    """(device, hidden, the descriptor's fields up to the weights)."""
    ty = _type(x, "x")
    if x.dim() < 2:
        raise _wrong("x", x, "rows ([..., width])")
    act = _ACTS.get(activation)
    if act is None:
        raise ValueError(f"activation {activation!r}: one of {sorted(_ACTS)}")
    if not isinstance(w_gate, torch.Tensor) or w_gate.dim() != 2:
        raise _wrong("w_gate", w_gate, "[width][hidden]")
    dev, shape, ws = x.device, x.shape, w_gate.shape
    if ws[0] != shape[-1]:
        raise _wrong("w_gate", w_gate, f"[{shape[-1]}][hidden]")
    i, et = dev.index, x.dtype
    return dev, ws[1], (_MLP_SIZE, ty, act, 0, _count(shape), ws[0], ws[1],
                        *(rows(x, shape, ty, i) or _rows(x, "x", shape, et, dev)),
                        *(rows(w_gate, ws, ty, i) or _rows(w_gate, "w_gate", ws, et, dev)),
                        *(rows(w_up, ws, ty, i) or _rows(w_up, "w_up", ws, et, dev)))


def gated_mlp(x, w_gate, w_up, activation: str = "silu", out=None):
    """act(x w_gate) * (x w_up) for x [..., width] and weights
    [width][hidden] of x's type; act is "silu" or "gelu" (tanh form).  Products
    of bfloat16 are accumulated in float32; float32 operands are multiplied as
    accurately as in float32 (infinities and numbers past bfloat16's largest
    take a slower way there)."""
    dev, hidden, head = _mlp_parts(x, w_gate, w_up, activation)
    shape = (*x.shape[:-1], hidden)
    h, hp = out, None
    if out is not None:
        hp = rows(out, shape, head[1], dev.index) or _rows(out, "out", shape, x.dtype, dev)
    if out is None or covers(0, out, x, w_gate, w_up):
        h = x.new_empty(shape)
        hp = h.data_ptr(), hidden
    d = _MLP.pack(*head, *hp, 0, 0, 0, 0, 0, 0, 0, 0)
    # (up to 16 rows of a block that is not very wide take no scratch)
    _op("gated_mlp")(d, dev, False, head[4] > 16 or hidden > 8192)
    return h if out is None else _given(out, h)


def gated_mlp_backward(dh, x, w_gate, w_up, activation: str = "silu"):
    """(dx, dw_gate, dw_up) of ``gated_mlp``; the projections are formed
    again, so nothing is kept between the passes.  The gradients of the
    projections, between the products, have the operands' type."""
    dev, hidden, head = _mlp_parts(x, w_gate, w_up, activation)
    dx, dg, du = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (x, w_gate, w_up))
    shape = (*x.shape[:-1], hidden)
    dhp = rows(dh, shape, head[1], dev.index) or _rows(dh, "dh", shape, x.dtype, dev)
    d = _MLP.pack(*head, 0, 0, *dhp, dx.data_ptr(), x.shape[-1],
                  dg.data_ptr(), hidden, du.data_ptr(), hidden)
    _op("gated_mlp")(d, dev, True, True)
    return dx, dg, du
