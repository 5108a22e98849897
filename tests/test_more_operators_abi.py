"""C entries of the delta rule, the norms around a block and the optimiser's
step on a host without a GPU: descriptors are checked before any device is
touched, scratch sizes come from the sizes alone, and the binding's packed
descriptors have the sizes of the header's structs."""
import ctypes
import os
import struct
import subprocess

import pytest

from dgen_hip import runtime as R

sequence = pytest.importorskip("dgen_hip.sequence")
from dgen_hip import optim  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID = -1
AT = 1 << 20  # an address that is never followed: nothing here reaches a device


def call(op, desc, entry="", tail=(0, 0)):
    L = R.load_library()
    return getattr(L, f"dgen_hip_{op}{entry}")(0, desc + sequence._WORKSPACE.pack(*tail), None)


def workspace(op, desc, *backward):
    n = ctypes.c_uint64(7)
    rc = getattr(R.load_library(), f"dgen_hip_{op}_workspace")(0, desc + sequence._NO_WORKSPACE, *backward, ctypes.byref(n))
    return rc, n.value


def message():
    return R.load_library().dgen_hip_last_error().decode()


def test_descriptor_sizes_are_the_headers(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "dgen_hip.h"\nint main(void) { printf("%zu %zu %zu %zu\\n", '
                   "sizeof(dgen_hip_delta), sizeof(dgen_hip_block_norms), sizeof(dgen_hip_adamw), sizeof(dgen_hip_adamw_tensor)); }\n")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True)
    sizes = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert sizes == [sequence._DELTA_SIZE, sequence._BLOCK_SIZE, optim._ADAMW_SIZE, 9 * 8]


def delta(size=None, type=0, batch=2, T=5, G=2, H=4, K=8, V=6, scale=1.0, q=(AT, 80, 16, 8), v=(AT, 120, 24, 6), g=(AT, 20, 4),
          y=(AT, 12000, 24, 6), back=(0,) * 22):
    return sequence._DELTA.pack(sequence._DELTA_SIZE if size is None else size, type, 1, scale, batch, T, G, H, K, V, 0, 0, 0, *q,
                                AT, 80, 16, 8, *v, *g, AT, 20, 4, *y, *back)


BACK = (AT, 120, 24, 6, AT, 80, 16, 8, AT, 80, 16, 8, AT, 120, 24, 6, AT, 20, 4, AT, 20, 4)


def block(size=None, x_type=0, s_type=0, act=1, rows=6, width=8, each=1, eps=1e-5, post=AT, pre=AT, scale=0, x=(AT, 8),
          residual=(AT, 8), gate=(0, 0), y=(AT, 8), s=(AT, 8), back=(0,) * 13):
    return sequence._BLOCK.pack(sequence._BLOCK_SIZE if size is None else size, x_type, s_type, act, rows, width, each, eps, post, pre,
                                scale, *x, *residual, *gate, *y, *s, *back)


BLOCK_BACK = (AT, 8, 0, 0, AT, 8, AT, 8, 0, 0, AT, AT, 0)


@pytest.mark.parametrize("op,desc,says", [
    ("gated_delta_rule", delta(size=8), "struct_size"),
    ("gated_delta_rule", delta(type=2), "type"),
    ("gated_delta_rule", delta(batch=-1), "batch"),
    ("gated_delta_rule", delta(T=0), "T 0"),
    ("gated_delta_rule", delta(T=(1 << 24) + 1), "T"),
    ("gated_delta_rule", delta(G=3), "key heads"),
    ("gated_delta_rule", delta(G=0), "key heads"),
    ("gated_delta_rule", delta(K=129), "K 129"),
    ("gated_delta_rule", delta(K=0), "K 0"),
    ("gated_delta_rule", delta(V=1025), "V 1025"),
    ("gated_delta_rule", delta(scale=float("inf")), "scale"),
    ("gated_delta_rule", delta(batch=1 << 22), "too many"),
    ("gated_delta_rule", delta(q=(0, 80, 16, 8)), "null"),
    ("gated_delta_rule", delta(v=(AT, 120, -24, 6)), "negative"),
    ("gated_delta_rule", delta(g=(0, 20, 4)), "g or beta"),
    ("gated_delta_rule", delta(y=(AT, 120, 24, 5)), "overlapping"),
    ("gated_delta_rule", delta(y=(AT, 119, 24, 6)), "overlapping"),
    ("gated_delta_rule", delta(T=100), "workspace"),
    ("block_norm", block(size=8), "struct_size"),
    ("block_norm", block(x_type=2), "types"),
    ("block_norm", block(act=2), "act"),
    ("block_norm", block(width=0), "width"),
    ("block_norm", block(width=8193), "width"),
    ("block_norm", block(rows=-1), "rows"),
    ("block_norm", block(rows=1 << 31), "rows"),
    ("block_norm", block(each=4), "gate_rows"),
    ("block_norm", block(each=0), "gate_rows"),
    ("block_norm", block(eps=float("nan")), "eps"),
    ("block_norm", block(pre=0), "post or pre"),
    ("block_norm", block(residual=(0, 8)), "null"),
    ("block_norm", block(x=(AT, -8)), "negative"),
    ("block_norm", block(s=(AT, 7)), "overlap"),
], ids=lambda v: v if isinstance(v, str) else "descriptor")
def test_refusals(op, desc, says):
    assert call(op, desc) == INVALID
    assert says in message(), message()


def test_delta_backward_refusals_and_scratch():
    full = delta(back=BACK)
    rc, n = workspace("gated_delta_rule", full, 1)
    assert rc == 0 and n > 0 and n % 256 == 0
    assert call("gated_delta_rule", full, "_backward", (AT, n - 256)) == INVALID and "workspace" in message()
    for at, wrong, says in ((0, 0, "dy"), (4, 0, "dq"), (8, 0, "dk"), (7, 7, "overlapping"), (12, 0, "dv"), (16, 0, "dg"), (19, 0, "dbeta"),
                            (18, 3, "overlapping")):
        back = list(BACK)
        back[at] = wrong
        assert call("gated_delta_rule", delta(back=back), "_backward", (AT, n)) == INVALID and says in message(), message()
    # a few frames take no scratch forward; no sequences take none at all
    assert workspace("gated_delta_rule", delta(T=16), 0) == (0, 0)
    assert workspace("gated_delta_rule", delta(batch=0, T=500), 1)[0] == INVALID  # (the gradients' places are missing)
    assert workspace("gated_delta_rule", delta(batch=0, T=500, back=BACK), 1) == (0, 0)
    # a long call's scratch grows past 32 bits
    big = delta(batch=8, T=1 << 18, G=4, H=4, K=128, V=128, q=(AT, 1 << 27, 512, 128), v=(AT, 1 << 27, 512, 128),
                g=(AT, 1 << 20, 4), back=(AT, 1 << 27, 512, 128) * 4 + (AT, 1 << 20, 4) * 2)
    rc, n = workspace("gated_delta_rule", big, 1)
    assert rc == 0 and n > 1 << 34


def test_block_backward_refusals_and_scratch():
    full = block(back=BLOCK_BACK)
    rc, n = workspace("block_norm", full, 1)
    assert rc == 0 and n > 0 and n % 256 == 0
    assert workspace("block_norm", block(), 0) == (0, 0)
    assert call("block_norm", full, "_backward", (AT, n - 256)) == INVALID and "workspace" in message()
    for at, wrong, says in ((0, 0, "dy"), (4, 0, "dx"), (6, 0, "dresidual"), (7, 7, "overlap"), (10, 0, "dpost"), (12, AT, "dscale")):
        back = list(BLOCK_BACK)
        back[at] = wrong
        assert call("block_norm", block(back=back), "_backward", (AT, n)) == INVALID and says in message(), message()
    assert call("block_norm", block(gate=(AT, 8), back=BLOCK_BACK), "_backward", (AT, n)) == INVALID and "dgate" in message()


def adamw(rows=((AT, AT * 2, AT * 3, AT * 4, AT, AT * 3, AT * 4, 0, 10),), size=None, type=0, count=None, lr=1e-3, beta1=0.9, beta2=0.99,
          eps=1e-8, decay=0.1, bound=0.0, step=1, at=0, norm=0):
    host = ctypes.create_string_buffer(b"".join(struct.pack("@8Qq", *r) for r in rows) or b"\0")
    adamw.kept = host
    return optim._ADAMW.pack(optim._ADAMW_SIZE if size is None else size, type, len(rows) if count is None else count,
                             ctypes.addressof(host), lr, beta1, beta2, eps, decay, bound, step, at, norm)


ONE = (AT, AT * 2, AT * 3, AT * 4, AT, AT * 3, AT * 4, 0, 10)
TWO = (AT * 5, AT * 6, AT * 7, AT * 8, AT * 5, AT * 7, AT * 8, 0, 10)


@pytest.mark.parametrize("kw,says", [
    (dict(size=8), "struct_size"), (dict(type=2), "type"), (dict(count=-1), "count"), (dict(lr=-1.0), "lr"),
    (dict(lr=float("nan")), "lr"), (dict(beta1=1.0), "betas"), (dict(beta2=-0.1), "betas"), (dict(eps=-1.0), "eps"),
    (dict(decay=float("inf")), "weight_decay"), (dict(bound=-1.0), "max_norm"), (dict(step=0), "step"),
    (dict(bound=1.0), "norm"), (dict(bound=1.0, norm=AT * 20), "workspace"),
    (dict(rows=[(*ONE[:8], -1)]), "elements"), (dict(rows=[(*ONE[:8], 1 << 35)]), "elements"),
    (dict(rows=[(0, *ONE[1:])]), "null"), (dict(rows=[(*ONE[:6], 0, *ONE[7:])]), "null"),
    # results over other tensors, over gradients, over one another, beside their own place
    (dict(rows=[ONE, (*TWO[:4], AT, *TWO[5:])]), "shares memory"), (dict(rows=[ONE, (*TWO[:7], AT * 2 + 8, 10)]), "shares memory"),
    (dict(rows=[(*ONE[:5], AT, *ONE[6:])]), "shares memory"), (dict(rows=[(*ONE[:4], AT + 4, *ONE[5:])]), "shares memory"),
    (dict(rows=[ONE, (AT * 5, AT + 36, *TWO[2:])]), "shares memory"), (dict(rows=[(*ONE[:7], AT + 39, 10)]), "shares memory"),
    (dict(rows=[ONE], bound=1.0, norm=AT * 2 + 36), "shares memory"), (dict(rows=[ONE], at=AT + 32), "shares memory"),
])
def test_adamw_refusals(kw, says):
    assert call("adamw_step", adamw(**kw)) == INVALID
    assert says in message(), message()


def test_adamw_scratch():
    assert workspace("adamw", adamw()) == (0, 0)
    # (a gradient may be read twice, and an empty tensor has no address)
    shared = [ONE, (*TWO[:1], AT * 2, *TWO[2:]), (0,) * 9]
    rc, n = workspace("adamw", adamw(shared, bound=1.0, norm=AT * 20))
    assert rc == 0 and n > 0 and n % 256 == 0
    assert call("adamw_step", adamw(shared, bound=1.0, norm=AT * 20), tail=(AT, n - 256)) == INVALID and "workspace" in message()
