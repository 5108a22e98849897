"""The sequence operators pass PyTorch's streams and memory to the library:
both have to use one HIP runtime, or the operators refuse to run."""
import os
import subprocess
import sys

import pytest

pytest.importorskip("torch")
PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dgen-audio_amd")


def run(code):
    env = dict(os.environ, PYTHONPATH=PACKAGE)
    return subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, env=env)


@pytest.mark.parametrize("op", ["rms_norm", "gated_mlp"])
def test_the_library_before_torch_is_refused(op):
    """Another process; nothing of it reaches a device."""
    done = run("import dgen_hip; dgen_hip.load_library()\n"
               "from dgen_hip import sequence as Q\n"
               "n = len(Q._hip_runtimes())\n"
               f"try: Q._op({op!r})\n"
               "except dgen_hip.HIPError as e: print(n, 'refused:', e)\n"
               "else: print(n, 'taken')\n")
    assert done.returncode == 0, done.stderr
    # (one runtime where PyTorch's and the library's are the same file)
    assert done.stdout.startswith("1 taken") or done.stdout.startswith("2 refused: two HIP runtimes"), done.stdout


@pytest.mark.parametrize("first", ["import torch", "from dgen_hip import sequence"])
def test_torch_first_is_one_runtime(first):
    done = run(f"{first}\nimport dgen_hip; dgen_hip.load_library()\n"
               "from dgen_hip import sequence as Q\n"
               "Q._op('causal_conv'); print(len(Q._hip_runtimes()))\n")
    assert done.returncode == 0 and done.stdout.strip() == "1", (done.stdout, done.stderr)
