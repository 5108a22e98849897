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
contiguous, the others have any stride.  Work is enqueued on torch's current
stream and the calls return without waiting; results and scratch come from
torch's allocator on that stream.  Nothing is recorded for autograd: a program
calls the backward functions itself.  A wrong argument raises ``ValueError``, a
failing launch ``HIPError``.

Clips of unequal length: ``lengths`` ([batch] int32) ends each sequence; later
frames are not read, and their outputs and gradients are 0.  Streaming: the
state that a call leaves (``state_out``) is the next call's ``state``, the
same tensor if wanted; a call with one frame is the form for live voices.

No counterpart in the reference, whose decoder sees one frame at a time
(Examples/HarmonicE2E/Model.swift:96-120).
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from .runtime import HIPError, load_library

_TYPES = {torch.float32: 0, torch.bfloat16: 1}
_ACTS = {"silu": 0, "gelu": 1}
_VP, _I32, _I64, _U32, _U64, _F = (ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_uint32, ctypes.c_uint64,
                                   ctypes.c_float)


class CSeq(ctypes.Structure):
    _fields_ = [("data", _VP), ("stride_b", _I64), ("stride_t", _I64)]


class CNorm(ctypes.Structure):
    _fields_ = [("struct_size", _U32), ("x_type", _I32), ("s_type", _I32), ("eps", _F), ("rows", _I64), ("width", _I64),
                ("weight", _VP), ("x", _VP), ("x_stride", _I64), ("residual", _VP), ("residual_stride", _I64),
                ("y", _VP), ("y_stride", _I64), ("s", _VP), ("s_stride", _I64), ("dy", _VP), ("dy_stride", _I64),
                ("ds", _VP), ("ds_stride", _I64), ("dx", _VP), ("dx_stride", _I64), ("dweight", _VP),
                ("workspace", _VP), ("workspace_bytes", _U64)]


class CConv(ctypes.Structure):
    _fields_ = [("struct_size", _U32), ("type", _I32), ("silu", _I32), ("width", _I32), ("batch", _I64), ("T", _I64),
                ("D", _I64), ("weight", _VP), ("bias", _VP), ("lengths", _VP), ("x", CSeq), ("y", CSeq),
                ("state", _VP), ("state_out", _VP), ("dy", CSeq), ("dx", CSeq), ("dweight", _VP), ("dbias", _VP),
                ("workspace", _VP), ("workspace_bytes", _U64)]


class CScan(ctypes.Structure):
    _fields_ = [("struct_size", _U32), ("type", _I32), ("batch", _I64), ("T", _I64), ("D", _I64), ("N", _I64),
                ("A", _VP), ("skip", _VP), ("dt_bias", _VP), ("lengths", _VP), ("state", _VP), ("state_out", _VP),
                ("x", CSeq), ("dt", CSeq), ("z", CSeq), ("B", CSeq), ("C", CSeq), ("y", CSeq), ("dy", CSeq),
                ("dx", CSeq), ("ddt", CSeq), ("dz", CSeq), ("dB", CSeq), ("dC", CSeq), ("dA", _VP), ("dskip", _VP),
                ("ddt_bias", _VP), ("workspace", _VP), ("workspace_bytes", _U64)]


class CMlp(ctypes.Structure):
    _fields_ = [("struct_size", _U32), ("type", _I32), ("act", _I32), ("reserved", _I32), ("rows", _I64),
                ("width", _I64), ("hidden", _I64), ("x", _VP), ("x_stride", _I64), ("w_gate", _VP),
                ("w_gate_stride", _I64), ("w_up", _VP), ("w_up_stride", _I64), ("h", _VP), ("h_stride", _I64),
                ("dh", _VP), ("dh_stride", _I64), ("dx", _VP), ("dx_stride", _I64), ("dw_gate", _VP),
                ("dw_gate_stride", _I64), ("dw_up", _VP), ("dw_up_stride", _I64), ("workspace", _VP),
                ("workspace_bytes", _U64)]


_NONE = (None, 0, 0)


def _current_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# (the same handle without a Stream object: 0.1 instead of 2 us a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _current_stream)


class _Op:
    """One operator's C entries."""

    def __init__(self, name: str):
        L = load_library()
        self.forward, self.backward = getattr(L, f"dgen_hip_{name}"), getattr(L, f"dgen_hip_{name}_backward")
        self.workspace = getattr(L, f"dgen_hip_{name}_workspace")
        self.error = L.dgen_hip_last_error

    def __call__(self, desc, device: torch.device, backward: bool, scratch: bool) -> None:
        ref, index = ctypes.byref(desc), device.index
        if scratch:
            need = _U64(0)
            self._check(self.workspace(index, ref, int(backward), ctypes.byref(need)))
            if need.value:
                ws = torch.empty(need.value, dtype=torch.uint8, device=device)
                desc.workspace, desc.workspace_bytes = ws.data_ptr(), need.value
        fn = self.backward if backward else self.forward
        self._check(fn(index, ref, _raw_stream(index)))

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


def _is(t, shape, dtype, device) -> bool:
    try:
        return t.dtype is dtype and t.shape == shape and t.device == device
    except AttributeError:  # not a tensor
        return False


def _seq(t, name: str, shape, dtype, device):
    """(address, batch stride, time stride) of a [batch][time][channel] tensor."""
    if not _is(t, shape, dtype, device):
        raise _wrong(name, t, f"{tuple(shape)} {dtype} on {device}")
    sb, st, sc = t.stride()
    if sc != 1 and shape[2] != 1:
        raise ValueError(f"{name}: the last axis must be contiguous")
    return t.data_ptr(), sb, st


def _dense(t, name: str, shape, dtype, device):
    """Address of a contiguous tensor (None stays None)."""
    if t is None:
        return None
    if not _is(t, shape, dtype, device):
        raise _wrong(name, t, f"{tuple(shape)} {dtype} on {device}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")
    return t.data_ptr()


def _rows(t, name: str, shape, dtype, device):
    """(address, row stride) of a tensor whose leading axes are rows."""
    if not _is(t, shape, dtype, device):
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
    xp = _rows(x, "x", shape, x.dtype, dev)
    w = _dense(weight, "weight", shape[-1:], torch.float32, dev)
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    yp = _rows(out, "out", shape, x.dtype, dev)
    rp = sp = (None, 0)
    st = ty
    if residual is not None:
        st = _type(residual, "residual")
        rp = _rows(residual, "residual", shape, residual.dtype, dev)
        if sum_out is None:
            sum_out = torch.empty_like(residual, memory_format=torch.contiguous_format)
        sp = _rows(sum_out, "sum_out", shape, residual.dtype, dev)
    elif sum_out is not None:
        raise ValueError("sum_out: only with a residual")
    d = CNorm(ctypes.sizeof(CNorm), ty, st, float(eps), _count(shape), shape[-1], w, *xp, *rp, *yp, *sp)
    _op("rms_norm")(d, dev, False, False)
    return out if residual is None else (out, sum_out)


def rms_norm_backward(dy, s, weight, ds=None, eps: float = 1e-5, out=None):
    """(dx, dweight) from the gradient of y and the stored sum ``s`` (x itself
    where there was no residual).  dx, in the sum's type, is the gradient of x
    and of the residual alike; ``ds``, the gradient that reaches the stored sum
    from elsewhere, is added to it."""
    ty, st, shape, dev = _type(dy, "dy"), _type(s, "s"), s.shape, s.device
    if s.dim() < 2:
        raise _wrong("s", s, "rows ([..., width])")
    if out is None:
        out = torch.empty_like(s, memory_format=torch.contiguous_format)
    dw = torch.empty(shape[-1], dtype=torch.float32, device=dev)
    d = CNorm(struct_size=ctypes.sizeof(CNorm), x_type=ty, s_type=st, eps=float(eps), rows=_count(shape),
              width=shape[-1], weight=_dense(weight, "weight", shape[-1:], torch.float32, dev), dweight=dw.data_ptr())
    if d.weight is None:
        raise ValueError("weight: missing")
    d.dy, d.dy_stride = _rows(dy, "dy", shape, dy.dtype, dev)
    d.s, d.s_stride = _rows(s, "s", shape, s.dtype, dev)
    d.dx, d.dx_stride = _rows(out, "out", shape, s.dtype, dev)
    if ds is not None:
        d.ds, d.ds_stride = _rows(ds, "ds", shape, s.dtype, dev)
    _op("rms_norm")(d, dev, True, True)
    return out, dw


# -------------------------------------------------------------- convolution
def _conv_parts(x, weight, bias, state, lengths):
    ty = _type(x, "x")
    if x.dim() != 3:
        raise _wrong("x", x, "[batch][time][channel]")
    B, T, D = shape = x.shape
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise _wrong("weight", weight, "[channel][width]")
    W, dev = weight.shape[1], x.device
    f32 = torch.float32
    head = (ty, (B, T, D), _dense(weight, "weight", (D, W), f32, dev), _dense(bias, "bias", (D,), f32, dev),
            _dense(lengths, "lengths", (B,), torch.int32, dev), _seq(x, "x", shape, x.dtype, dev),
            _dense(state, "state", (B, W - 1, D), x.dtype, dev))
    return W, dev, head


def causal_conv(x, weight, bias=None, silu: bool = True, state=None, state_out=None, lengths=None, out=None):
    """y[t] = silu(bias + sum_i weight[:, i] x[t - W + 1 + i]) per channel of
    x [batch][time][D], weight [D][W] (W up to 8).  The frames before the
    first are ``state`` ([batch][W-1][D], x's type, oldest first) or 0;
    ``state_out`` receives the last W-1 frames of each sequence."""
    W, dev, (ty, (B, T, D), w, b, n, xs, st) = _conv_parts(x, weight, bias, state, lengths)
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    d = CConv(ctypes.sizeof(CConv), ty, 1 if silu else 0, W, B, T, D, w, b, n, xs,
              _seq(out, "out", x.shape, x.dtype, dev), st,
              _dense(state_out, "state_out", (B, W - 1, D), x.dtype, dev))
    _op("causal_conv")(d, dev, False, False)
    return out


def causal_conv_backward(dy, x, weight, bias=None, silu: bool = True, state=None, lengths=None, out=None):
    """(dx, dweight, dbias) of ``causal_conv`` (dbias None without a bias);
    the state counts as given."""
    W, dev, (ty, (B, T, D), w, b, n, xs, st) = _conv_parts(x, weight, bias, state, lengths)
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    dw = torch.empty((D, W), dtype=torch.float32, device=dev)
    db = None if bias is None else torch.empty(D, dtype=torch.float32, device=dev)
    d = CConv(ctypes.sizeof(CConv), ty, 1 if silu else 0, W, B, T, D, w, b, n, xs, _NONE, st, None,
              _seq(dy, "dy", x.shape, x.dtype, dev), _seq(out, "out", x.shape, x.dtype, dev), dw.data_ptr(),
              None if db is None else db.data_ptr())
    _op("causal_conv")(d, dev, True, True)
    return out, dw, db


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


def _scan_desc(x, dt, A, B, C, D, z, dt_bias, state, lengths):
    ty = _type(x, "x")
    if x.dim() != 3:
        raise _wrong("x", x, "[batch][time][channel]")
    if not isinstance(A, torch.Tensor) or A.dim() != 2:
        raise _wrong("A", A, "[channel][state]")
    shape, dev, f32, et = x.shape, x.device, torch.float32, x.dtype
    n, T, ch = shape
    N = A.shape[1]
    bc = torch.Size((n, T, N))
    return CScan(ctypes.sizeof(CScan), ty, n, T, ch, N, _dense(A, "A", (ch, N), f32, dev),
                 _dense(D, "D", (ch,), f32, dev), _dense(dt_bias, "dt_bias", (ch,), f32, dev),
                 _dense(lengths, "lengths", (n,), torch.int32, dev), _dense(state, "state", (n, ch, N), f32, dev), None,
                 _seq(x, "x", shape, et, dev), _seq(dt, "dt", shape, et, dev),
                 _NONE if z is None else _seq(z, "z", shape, et, dev), _seq(B, "B", bc, et, dev),
                 _seq(C, "C", bc, et, dev))


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, state=None, state_out=None, lengths=None, out=None):
    """The selective scan over x [batch][time][channels]: with step =
    softplus(dt + dt_bias), h[t] = exp(step A) h[t-1] + step x[t] B[t] per
    channel ([channels][N] states, N up to 64), y[t] = (C[t].h[t] + D x[t])
    silu(z[t]).  B and C are [batch][time][N]; A, D, dt_bias and the states
    ([batch][channels][N]) are float32; D, z and dt_bias may be left out.
    Results of a sequence can differ in rounding with the number of sequences
    and channels in the call, which decide how time is cut."""
    d = _scan_desc(x, dt, A, B, C, D, z, dt_bias, state, lengths)
    dev = x.device
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    d.y = _seq(out, "out", x.shape, x.dtype, dev)
    d.state_out = _dense(state_out, "state_out", (d.batch, d.D, d.N), torch.float32, dev)
    # (a call of few frames is one launch without scratch)
    _op("selective_scan")(d, dev, False, d.T > 32)
    return out


def selective_scan_backward(dy, x, dt, A, B, C, D=None, z=None, dt_bias=None, state=None, lengths=None) -> ScanGrads:
    """Gradients of ``selective_scan``; the state counts as given."""
    d = _scan_desc(x, dt, A, B, C, D, z, dt_bias, state, lengths)
    dev, et, f32 = x.device, x.dtype, torch.float32
    d.dy = _seq(dy, "dy", x.shape, et, dev)

    def like(shape, dtype, given=True):
        return torch.empty(shape, dtype=dtype, device=dev) if given else None

    bc = (d.batch, d.T, d.N)
    g = ScanGrads(like(x.shape, et), like(x.shape, et), like((d.D, d.N), f32), like(bc, et), like(bc, et),
                  like((d.D,), f32, D is not None), like(x.shape, et, z is not None),
                  like((d.D,), f32, dt_bias is not None))
    for name in ("dx", "ddt", "dB", "dC", "dz"):
        t = getattr(g, name)
        if t is not None:
            setattr(d, name, (t.data_ptr(), t.stride(0), t.stride(1)))
    d.dA = g.dA.data_ptr()
    d.dskip = None if g.dD is None else g.dD.data_ptr()
    d.ddt_bias = None if g.ddt_bias is None else g.ddt_bias.data_ptr()
    _op("selective_scan")(d, dev, True, True)
    return g


# ------------------------------------------------------ gated feed-forward
def _mlp_desc(x, w_gate, w_up, activation):
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
    return CMlp(ctypes.sizeof(CMlp), ty, act, 0, _count(shape), ws[0], ws[1], *_rows(x, "x", shape, x.dtype, dev),
                *_rows(w_gate, "w_gate", ws, x.dtype, dev), *_rows(w_up, "w_up", ws, x.dtype, dev))


def gated_mlp(x, w_gate, w_up, activation: str = "silu", out=None):
    """act(x w_gate) * (x w_up) for x [..., width] and weights
    [width][hidden] of x's type; act is "silu" or "gelu" (tanh form).  Products
    of bfloat16 are accumulated in float32; float32 operands are multiplied as
    accurately as in float32."""
    d = _mlp_desc(x, w_gate, w_up, activation)
    shape = (*x.shape[:-1], d.hidden)
    if out is None:
        out = torch.empty(shape, dtype=x.dtype, device=x.device)
    d.h, d.h_stride = _rows(out, "out", shape, x.dtype, x.device)
    # (few rows take no scratch)
    _op("gated_mlp")(d, x.device, False, d.rows > 16)
    return out


def gated_mlp_backward(dh, x, w_gate, w_up, activation: str = "silu"):
    """(dx, dw_gate, dw_up) of ``gated_mlp``; the projections are formed
    again, so nothing is kept between the passes."""
    d = _mlp_desc(x, w_gate, w_up, activation)
    dev = x.device
    d.dh, d.dh_stride = _rows(dh, "dh", (*x.shape[:-1], d.hidden), x.dtype, dev)
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
    dg, du = (torch.empty(w_gate.shape, dtype=x.dtype, device=dev) for _ in range(2))
    d.dx, d.dx_stride = dx.data_ptr(), d.width
    d.dw_gate, d.dw_gate_stride = dg.data_ptr(), d.hidden
    d.dw_up, d.dw_up_stride = du.data_ptr(), d.hidden
    _op("gated_mlp")(d, dev, True, True)
    return dx, dg, du
