"""The bound on the gradients' norm (dgen_hip.optim) with gradients whose squares
32 bits do not hold, and second moments of such, against the formula in 64 bits with test_gpu_adamw's
tolerances.  Needs a GPU."""
import pytest

torch = pytest.importorskip("torch")

from dgen_hip import optim  # noqa: E402
from test_gpu_adamw import ARGS, check, formula, tensors  # noqa: E402
from test_gpu_sequence import F64, close  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-35, 1e-25, 1e-20, 1e17, 1e25, 1e37])
@pytest.mark.parametrize("one", [False, True])
def test_gradients_of_any_finite_size(gpu, grad, size, one):
    """All of that size, or one of them among ordinary ones: the step is the one
    of the gradients scaled to the bound."""
    p, g, m, v = tensors(8, [(40,), (5000,), (3, 7)], grad=grad)
    for t in g if not one else g[:1]:
        t[:] = (t.double() * (size * 100)).to(grad)  # (the tensors' own are of 1e-2)
    assert all(torch.isfinite(t).all() for t in g)
    want = formula(p, g, m, v, 3, max_norm=0.5, **ARGS)
    norm = optim.adamw(p, g, m, v, 3, max_norm=0.5, **ARGS)
    check((p, m, v), want)
    if want[3] > torch.finfo(torch.float32).max:  # (5000 of 1e37: 1e37 sqrt(5000) = 7.07e38, past 3.40e38)
        assert torch.isinf(norm)
    else:
        close(norm, want[3].cpu(), 70, "norm")
    assert norm > 0 and any((t != 0).any() for t in m)


def test_a_norm_past_the_largest_number(gpu):
    """It is reported as infinity, and the step is still the scaled gradients'."""
    p, g, m, v = tensors(9, [(5000,), (60,)])
    for t in g:
        t[:] = t.sign() * 3e38
    want = formula(p, g, m, v, 3, max_norm=0.5, **ARGS)
    norm = optim.adamw(p, g, m, v, 3, max_norm=0.5, **ARGS)
    check((p, m, v), want)
    assert torch.isinf(norm) and want[3].to(F64) > torch.finfo(torch.float32).max


@pytest.mark.parametrize("step", [1, 50])
def test_second_moments_near_the_largest_number(gpu, step):
    """(1 - beta2) g^2 is within 32 bits where g^2 is not."""
    p, g, m, v = tensors(10, [(300,), (4100,)])
    for t in g:
        t[:] = t.sign() * 3e19
    want = formula(p, g, m, v, step, **ARGS)
    assert all(torch.isfinite(t.float()).all() for t in want[2]) and 3e19 ** 2 > torch.finfo(torch.float32).max
    optim.adamw(p, g, m, v, step, **ARGS)
    check((p, m, v), want)
