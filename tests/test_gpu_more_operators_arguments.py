"""Arguments of the delta rule, the norms around a block and the optimiser's
step that are no numbers, lists or tensors: ValueError, whatever they are.  Needs
a GPU (nothing is launched)."""
import pytest

torch = pytest.importorskip("torch")

from dgen_hip import optim  # noqa: E402
from dgen_hip import sequence as Q  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("wrong", [dict(betas=(0.9,)), dict(betas=(0.9, 0.99, 0.9)), dict(betas=0.9), dict(betas=None), dict(betas=("a", 0.9)),
                                   dict(lr=None), dict(lr="x"), dict(eps=[1e-8]), dict(weight_decay="x"), dict(max_norm="x"),
                                   dict(step=1.5), dict(step=-1), dict(step=0), dict(step=1 << 63), dict(step="1"), dict(step=None),
                                   dict(step=float("nan")), dict(step=float("inf")),
                                   dict(out=5), dict(out=()), dict(params=3), dict(grads=3), dict(copies=3), dict(grads=None)], ids=str)
def test_optimiser(gpu, wrong):
    p, g, m, v = ([torch.ones(4, device="cuda")] for _ in range(4))
    ok = dict(params=p, grads=g, exp_avg=m, exp_avg_sq=v, step=1)
    with pytest.raises(ValueError):
        optim.adamw(**{**ok, **wrong})
    assert all(torch.equal(t[0], torch.ones_like(t[0])) for t in (p, g, m, v))


def test_counts_that_are_whole(gpu):
    import numpy as np
    results = []
    for step in (3, 3.0, np.int64(3), torch.tensor(3)[None].numpy()[0]):
        p, m, v = ([torch.ones(4, device="cuda")] for _ in range(3))
        optim.adamw(p, [torch.full((4,), 0.3, device="cuda")], m, v, step)
        results.append(p[0])
    assert all(torch.equal(t, results[0]) for t in results)


@pytest.mark.parametrize("wrong", [dict(eps="x"), dict(eps=None), dict(post_weight=None), dict(pre_weight=None), dict(gate=3),
                                   dict(residual_scale=3)], ids=str)
def test_block_norm(gpu, wrong):
    x, w = torch.zeros(3, 8, device="cuda"), torch.ones(8, device="cuda")
    with pytest.raises(ValueError):
        Q.block_norm(**{**dict(x=x, post_weight=w, residual=x, pre_weight=w), **wrong})
    with pytest.raises(ValueError):
        Q.block_norm_backward(**{**dict(dy=x, x=x, residual=x, s=x, post_weight=w, pre_weight=w), **wrong})


@pytest.mark.parametrize("wrong", [dict(scale="x"), dict(scale=[1.0]), dict(scale=1e39), dict(k=None), dict(beta=2.0), dict(lengths=3)], ids=str)
def test_delta_rule(gpu, wrong):
    q, g = torch.zeros(1, 20, 1, 8, device="cuda"), torch.zeros(1, 20, 1, device="cuda")
    ok = dict(q=q, k=q, v=q, g=g, beta=g)
    with pytest.raises(ValueError):
        Q.gated_delta_rule(**{**ok, **wrong})
    with pytest.raises(ValueError):
        Q.gated_delta_rule_backward(q, **{**ok, **wrong})
