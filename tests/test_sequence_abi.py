"""The sequence operators' C entries on a host without a GPU: descriptors are
checked before any device is touched, scratch sizes come from the sizes alone,
and the binding's packed descriptors have the sizes of the header's structs."""
import ctypes
import os
import subprocess

import pytest

from dgen_hip import runtime as R

sequence = pytest.importorskip("dgen_hip.sequence")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID = -1
AT = 1 << 20  # an address that is never followed: nothing here reaches a device


def call(op, desc, entry="", tail=(0, 0)):
    L = R.load_library()
    return getattr(L, f"dgen_hip_{op}{entry}")(0, desc + sequence._WORKSPACE.pack(*tail), None)


def workspace(op, desc, backward):
    n = ctypes.c_uint64(7)
    rc = getattr(R.load_library(), f"dgen_hip_{op}_workspace")(0, desc + sequence._NO_WORKSPACE, backward, ctypes.byref(n))
    return rc, n.value


def message():
    return R.load_library().dgen_hip_last_error().decode()


def test_descriptor_sizes_are_the_headers(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "dgen_hip.h"\nint main(void) { printf("%zu %zu %zu %zu\\n", '
                   "sizeof(dgen_hip_norm), sizeof(dgen_hip_conv), sizeof(dgen_hip_scan), sizeof(dgen_hip_mlp)); }\n")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True)
    sizes = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert sizes == [sequence._NORM_SIZE, sequence._CONV_SIZE, sequence._SCAN_SIZE, sequence._MLP_SIZE]


def norm(size=None, x_type=0, s_type=0, eps=1e-5, rows=4, width=8, weight=AT, x=(AT, 8), residual=(0, 0), y=(AT, 8), s=(0, 0),
         back=(0,) * 7):
    return sequence._NORM.pack(sequence._NORM_SIZE if size is None else size, x_type, s_type, eps, rows, width, weight,
                               *x, *residual, *y, *s, *back)


def conv(type=0, width=4, batch=2, T=5, D=8, weight=AT, x=(AT, 40, 8), y=(AT, 40, 8), state=0, state_out=0):
    return sequence._CONV.pack(sequence._CONV_SIZE, type, 1, width, batch, T, D, weight, 0, 0, *x, *y, state, state_out,
                               *(0,) * 8)


def scan(type=0, batch=2, T=5, D=8, N=4, A=AT, x=(AT, 40, 8), y=(AT, 40, 8), grads=(0,) * 21):
    return sequence._SCAN.pack(sequence._SCAN_SIZE, type, batch, T, D, N, A, 0, 0, 0, 0, 0, *x, AT, 40, 8, 0, 0, 0, AT, 20,
                               4, AT, 20, 4, *y, *grads)


def mlp(type=0, act=0, rows=20, width=8, hidden=16, x=(AT, 8), wg=(AT, 16), h=(AT, 16), back=(0,) * 8):
    return sequence._MLP.pack(sequence._MLP_SIZE, type, act, 0, rows, width, hidden, *x, *wg, AT, 16, *h, *back)


@pytest.mark.parametrize("op,desc,says", [
    ("rms_norm", norm(size=8), "struct_size"),
    ("rms_norm", norm(x_type=2), "types"),
    ("rms_norm", norm(width=0), "width"),
    ("rms_norm", norm(width=32769), "width"),
    ("rms_norm", norm(eps=float("nan")), "eps"),
    ("rms_norm", norm(weight=0), "weight"),
    ("rms_norm", norm(residual=(AT, 8)), "come together"),
    ("rms_norm", norm(y=(AT, 7)), "overlap"),
    ("rms_norm", norm(x=(AT, -8)), "negative"),
    ("causal_conv", conv(type=7), "type"),
    ("causal_conv", conv(width=9), "width"),
    ("causal_conv", conv(T=0), "T 0"),
    ("causal_conv", conv(batch=70000), "batch"),
    ("causal_conv", conv(weight=0), "weight"),
    ("causal_conv", conv(y=(AT, 39, 8)), "overlapping"),
    ("causal_conv", conv(x=(AT, 40, -8)), "negative"),
    ("causal_conv", conv(width=1, state=AT), "no state"),
    ("selective_scan", scan(N=65), "N 65"),
    ("selective_scan", scan(N=0), "N 0"),
    ("selective_scan", scan(A=0), "null A"),
    ("selective_scan", scan(T=1 << 25), "T"),
    ("selective_scan", scan(x=(AT, 40, 1 << 27)), "stride"),
    ("selective_scan", scan(y=(AT, 0, 8)), "overlapping"),
    ("selective_scan", scan(T=200, x=(AT, 1600, 8), y=(AT, 1600, 8)), "workspace"),
    ("gated_mlp", mlp(act=2), "activation"),
    ("gated_mlp", mlp(hidden=0), "hidden"),
    ("gated_mlp", mlp(wg=(0, 16)), "w_gate"),
    ("gated_mlp", mlp(h=(AT, 15)), "overlapping"),
    ("gated_mlp", mlp(x=(0, 8)), "null x"),
], ids=lambda v: v if isinstance(v, str) else "descriptor")
def test_refusals(op, desc, says):
    assert call(op, desc) == INVALID
    assert says in message(), message()


def test_backward_refusals_and_scratch():
    assert call("rms_norm", norm(back=(AT, 8, 0, 0, AT, 8, 0), s=(AT, 8)), "_backward") == INVALID and "dweight" in message()
    full = norm(back=(AT, 8, 0, 0, AT, 8, AT), s=(AT, 8))
    rc, n = workspace("rms_norm", full, 1)
    assert rc == 0 and n > 0 and n % 256 == 0
    assert call("rms_norm", full, "_backward", (AT, n - 256)) == INVALID and "workspace" in message()
    # a descriptor without its gradients' places is refused by the size query too
    assert workspace("selective_scan", scan(), 1)[0] == INVALID
    assert workspace("selective_scan", scan(), 0) == (0, 0)
    rc, n = workspace("selective_scan", scan(T=2000, D=8, x=(AT, 16000, 8), y=(AT, 16000, 8)), 0)
    assert rc == 0 and n > 0
    assert workspace("gated_mlp", mlp(), 0) == (0, 0)
    assert R.load_library().dgen_hip_gated_mlp(0, None, None) == INVALID
