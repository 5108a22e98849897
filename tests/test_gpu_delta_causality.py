"""The gated delta rule with values that are not finite: no frame's result depends
on a later frame's operands, and no gradient that a frame's operands do not reach
depends on them, bit for bit, however the call is cut.  Needs a GPU."""
import pytest

torch = pytest.importorskip("torch")

from dgen_hip import sequence as Q  # noqa: E402
from test_gpu_delta_rule import INPUTS, data, on_gpu  # noqa: E402
from test_gpu_sequence import TYPES  # noqa: E402

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")

# (batch, frames, heads, K, V): a few frames, one chunk, several, two blocks of values, segments
SIZES = [(1, 10, 2, 16, 8), (2, 64, 2, 24, 20), (1, 200, 1, 128, 48), (1, 150, 2, 33, 40), (1, 600, 1, 32, 20), (1, 900, 1, 64, 33)]


def spots(T):
    return sorted({0, 1, T // 2, min(T - 1, 15), min(T - 1, 17), T - 1})


def equal(a, b):
    return torch.equal(a, b) and torch.isfinite(a).all()


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("B,T,H,K,V", SIZES)
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_results_do_not_depend_on_later_frames(gpu, ty, B, T, H, K, V, bad):
    x, _, s, _ = data(B, T, H, H, K, V, ty, slow=True)
    a = on_gpu(x, s=s)
    after = torch.empty_like(a["state"])
    y = Q.gated_delta_rule(**a, state_out=after)
    left = after.clone()
    for at in spots(T):
        for name in INPUTS:
            if name == "g" and bad == -INF:
                continue  # (that one is a gate that forgets)
            b = {k: t.clone() for k, t in a.items()}
            where = (0, at, 0) + ((3,) if name in "qkv" else ())
            b[name][where] = bad
            z = Q.gated_delta_rule(**b, state_out=after)
            where = (name, at)
            assert equal(z[:, :at], y[:, :at]), where
            assert equal(z[:, :, 1:], y[:, :, 1:]) and equal(z[1:], y[1:]), where
            assert equal(after[1:], left[1:]) and equal(after[:, 1:], left[:, 1:]), where
            if name == "v":  # one value's column; the others know nothing of it
                assert not torch.isfinite(z[0, at:, 0, 3]).any(), where
                z[0, at:, 0, 3] = y[0, at:, 0, 3]
                assert equal(z, y), where
                assert not torch.isfinite(after[0, 0, :, 3]).any(), where
                after[0, 0, :, 3] = left[0, 0, :, 3]
                assert equal(after, left), where
            elif name == "q":  # one frame's result
                assert not torch.isfinite(z[0, at, 0]).any(), where
                z[0, at, 0] = y[0, at, 0]
                assert equal(z, y) and equal(after, left), where
            else:
                assert not torch.isfinite(z[0, at:, 0]).any(), where


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("B,T,H,K,V", SIZES)
@pytest.mark.parametrize("bad", [NAN, INF])
def test_gradients_that_a_value_does_not_reach(gpu, ty, B, T, H, K, V, bad):
    """A value's are those of the frames before it (and of all values); a result's
    gradient's are those of the frames after it (and of all queries but its own)."""
    x, _, s, d = data(B, T, H, H, K, V, ty, slow=True)
    a, dy = on_gpu(x, s=s), d.normal(B, T, H, V, type=ty).cuda()
    r = Q.gated_delta_rule_backward(dy, **a)
    for at in spots(T):
        b = {k: t.clone() for k, t in a.items()}
        b["v"][0, at, 0, 3] = bad
        z = Q.gated_delta_rule_backward(dy, **b)
        assert equal(z.dv, r.dv), at
        for k, one, two in zip(INPUTS, z, r):
            assert equal(one[:, :at], two[:, :at]) and equal(one[1:], two[1:]) and equal(one[:, :, 1:], two[:, :, 1:]), (k, at)
        e = dy.clone()
        e[0, at, 0, 3] = bad
        z = Q.gated_delta_rule_backward(e, **a)
        for k, one, two in zip(INPUTS, z, r):
            assert equal(one[:, at + 1:], two[:, at + 1:]) and equal(one[1:], two[1:]) and equal(one[:, :, 1:], two[:, :, 1:]), (k, at)
        z.dq[0, at, 0] = r.dq[0, at, 0]
        assert equal(z.dq, r.dq), at
