"""The sequence operators pass PyTorch's streams and memory to the library:
both have to use one HIP runtime, or the operators refuse to run."""
import os
import subprocess
import sys

import pytest

pytest.importorskip("torch")
PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dgen-audio_amd")


# prints how many HIP runtimes the process has loaded
LOADED = "print(len({l.split()[-1] for l in open('/proc/self/maps') if '/libamdhip64.so' in l}))\n"


def run(code):
    env = dict(os.environ, PYTHONPATH=PACKAGE)
    return subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, env=env)


@pytest.mark.parametrize("op", ["rms_norm", "gated_mlp"])
def test_the_library_before_torch_is_refused(op):
    """Another process; nothing of it reaches a device."""
    done = run("import dgen_hip; dgen_hip.load_library()\n"
               "from dgen_hip import sequence as Q\n"
               f"try: Q._op({op!r})\n"
               "except dgen_hip.HIPError as e: print('refused:', e)\n"
               "else: print('taken')\n" + LOADED)
    assert done.returncode == 0, done.stderr
    said, runtimes = done.stdout.splitlines()
    # (one runtime where PyTorch's and the library's are the same file)
    assert said.startswith("refused: two HIP runtimes") if runtimes == "2" else said == "taken", done.stdout


@pytest.mark.parametrize("first", ["import torch", "from dgen_hip import sequence"])
def test_torch_first_is_one_runtime(first):
    done = run(f"{first}\nimport dgen_hip; dgen_hip.load_library()\n"
               "from dgen_hip import sequence as Q\n"
               "Q._op('causal_conv')\n" + LOADED)
    assert done.returncode == 0 and done.stdout.strip() == "1", (done.stdout, done.stderr)
