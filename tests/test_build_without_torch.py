"""The library on a host without PyTorch's headers: it builds to the end with
hipcc alone, and the Python package does without the native module."""
import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")  # (what is tested is that the rest does without its headers)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "dgen-audio_amd", "csrc")


def commands(*args):
    return subprocess.run(["make", "-n", "-B", "-C", CSRC, *args], capture_output=True, text=True, check=True).stdout


def test_the_library_builds_without_pytorch():
    without = commands("PYTHON=false")
    assert "libdgen_hip.so" in without and "-lhiprtc" in without
    assert "tensor_args" not in without
    assert "tensor_args.cpp" in commands(f"PYTHON={sys.executable}")


def test_the_package_does_without_the_native_module(tmp_path):
    """In another process, where importing the module fails."""
    code = (
        "import sys; sys.modules['dgen_hip._tensor_args'] = None\n"
        "import torch\n"
        "from dgen_hip import sequence as Q\n"
        "assert Q.covers.__module__ == 'dgen_hip._tensor_args_python'\n"
        "x = torch.zeros(2, 8)\n"
        "try: Q.rms_norm(x, x[0])\n"
        "except ValueError as e: print('refused:', e)\n")
    env = dict(os.environ, PYTHONPATH=os.path.join(ROOT, "dgen-audio_amd"))
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, env=env)
    assert out.returncode == 0 and out.stdout.startswith("refused: x:"), out.stderr


def test_overlaps_in_python_as_in_native_code():
    from test_tensor_covers import views

    from dgen_hip import _tensor_args as native
    from dgen_hip import _tensor_args_python as plain

    t = torch.zeros(4, 6, 10)
    for a in views(t):
        for b in views(t) + [None]:
            for may in (0, 1):
                assert plain.covers(may, a, b) is native.covers(may, a, b)


@pytest.mark.gpu
def test_calls_without_the_native_module(gpu, monkeypatch):
    """The same results, state in place and results over operands included."""
    from dgen_hip import _tensor_args_python as plain
    from dgen_hip import sequence as Q

    g = torch.Generator().manual_seed(1)
    x, w, state = (torch.randn(*s, generator=g).cuda() for s in ((2, 40, 16), (16, 4), (2, 3, 16)))
    A, Bm = -torch.rand(16, 8, generator=g).cuda(), torch.randn(2, 40, 8, generator=g).cuda()
    h = torch.zeros(2, 16, 8, device="cuda")

    def calls():
        s, c, k = x.clone(), state.clone(), h.clone()
        y, _ = Q.rms_norm(x, w[:, 0].contiguous(), residual=s, sum_out=s)
        u = Q.causal_conv(y, w, state=c, state_out=c, out=y)
        o = Q.selective_scan(u, x, A, Bm, Bm, state=k, state_out=k)
        m = Q.gated_mlp(o, w, w)
        grads = Q.gated_mlp_backward(m, o, w, w)
        return [s, c, k, y, o, m, *grads, *Q.rms_norm_backward(o, x, w[:, 0].contiguous())]

    want = calls()
    for name in ("covers", "dense", "rows", "sequence"):
        monkeypatch.setattr(Q, name, getattr(plain, name))
    for a, b in zip(want, calls()):
        assert torch.equal(a, b)
