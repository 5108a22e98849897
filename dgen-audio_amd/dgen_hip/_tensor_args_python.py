"""What sequence.py takes from the native module ``_tensor_args``
(csrc/tensor_args.cpp), for hosts where that was not built."""
from __future__ import annotations

import torch


def _turned_down(t, *_):
    """Leaves the test of an argument to sequence.py's own."""
    return None


dense = rows = sequence = _turned_down


def _extent(t: torch.Tensor, pitch: int = 0) -> int:
    """Bytes from the first element to past the last, along the axes whose
    steps are no multiples of ``pitch`` bytes (0: along all)."""
    k = t.itemsize
    return k + sum((n - 1) * s * k for n, s in zip(t.shape, t.stride()) if pitch == 0 or s * k % pitch)


def _overlap(a: torch.Tensor, b: torch.Tensor) -> int:
    """0: the tensors share no memory, 1: they are the same view, 2: otherwise,
    or it cannot be told."""
    if a.numel() == 0 or b.numel() == 0:
        return 0
    x, y = a.data_ptr(), b.data_ptr()
    if x + _extent(a) <= y or y + _extent(b) <= x:
        return 0
    if x == y and a.dtype == b.dtype and a.shape == b.shape and all(
            n == 1 or p == q for n, p, q in zip(a.shape, a.stride(), b.stride())):
        return 1
    for t in (a, b):
        for n, s in zip(t.shape, t.stride()):
            pitch = s * t.itemsize
            # modulo the step of some axis each takes a range of the bytes
            if n > 1 and pitch and _extent(a, pitch) <= (y - x) % pitch <= pitch - _extent(b, pitch):
                return 0
    return 2


def covers(may: int, t: torch.Tensor, *others) -> bool:
    """Whether writing ``t`` changes what is read or written of the others; the
    first ``may`` of them may be ``t`` itself, element by element."""
    return any(o is not None and _overlap(t, o) > (i < may) for i, o in enumerate(others))
