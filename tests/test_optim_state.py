"""What the framework's optimiser keeps: its count of steps, and the rounded
copies of the parameters.  Refusals on any host; the rest needs a GPU."""
import pytest

torch = pytest.importorskip("torch")

from dgen_hip import optim  # noqa: E402


def test_a_refused_step_does_not_count_on_the_host():
    """(Parameters that are not on a GPU are refused.)"""
    own = optim.AdamW([torch.ones(4)])
    for _ in range(3):
        with pytest.raises(ValueError):
            own.step([torch.ones(4)])
    assert int(own.count) == 0


@pytest.mark.gpu
def test_a_refused_step_does_not_count(gpu):
    """The steps around it are those of an optimiser that never saw it."""
    shapes = [(5, 3), (4100,)]
    a, b = ([torch.linspace(-1, 1, s[0] * (s[1] if len(s) > 1 else 1), device="cuda").view(s) for s in shapes] for _ in range(2))
    one, two = optim.AdamW(a, lr=0.1, max_norm=1.0), optim.AdamW(b, lr=0.1, max_norm=1.0)
    grads = [torch.full(s, 0.5, device="cuda") for s in shapes]
    for k in range(3):
        for wrong in (grads[:1], [grads[0].t(), grads[1]], [grads[0].bfloat16(), grads[1]], [grads[0], b[1]], [grads[0], None]):
            with pytest.raises(ValueError):
                two.step(wrong)
        one.step(grads), two.step(grads)
        assert int(one.count) == int(two.count) == k + 1
    for x, y in zip((*one.params, *one.exp_avg, *one.exp_avg_sq), (*two.params, *two.exp_avg, *two.exp_avg_sq)):
        assert torch.equal(x, y)


def test_copies_are_the_rounded_parameters_from_the_start():
    """They are what a pass before the first step reads."""
    p = [torch.linspace(-1, 1, 12).view(3, 4).requires_grad_(), torch.full((), 0.1), torch.zeros(0, 2)]
    copies = [torch.full(t.shape, 9.0, dtype=torch.bfloat16) for t in p]
    copies[1] = None
    optim.AdamW(p, copies=copies)
    assert torch.equal(copies[0], p[0].detach().bfloat16()) and copies[2].shape == (0, 2)


def test_copies_that_do_not_fit_are_refused_and_left():
    p = [torch.ones(3, 4), torch.ones(5)]
    for wrong in ([torch.zeros(3, 4), None], [torch.zeros(4, dtype=torch.bfloat16), None], [None], [None, None, None], [3, None]):
        with pytest.raises(ValueError):
            optim.AdamW(p, copies=wrong)
        assert all(not isinstance(t, torch.Tensor) or not t.any() for t in wrong)
