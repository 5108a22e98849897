"""Long calls of the selective scan, whose time is cut into chunks (few of them
join their states by themselves, many in a launch of their own), and sequences
without frames."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from dgen_hip import sequence as Q  # noqa: E402
from test_gpu_sequence import F64, close, ref_call, scan_data, scan_gpu, scan_ops, spoil, wide  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    if not torch.cuda.is_available():
        pytest.fail("no GPU")
    return torch.device("cuda")


def ends(T):
    return [T, 0, 1, T // 2, 64, T - 1]


@pytest.mark.parametrize("T", [65, 512, 1024, 1056, 1800])
@pytest.mark.parametrize("N", [3, 16, 40])
def test_forward_with_its_state_in_place(gpu, T, N):
    B, D = 6, 70
    v, _, d = scan_data(B, T, D, N, torch.float32, True, True, True, seed=5)
    v["dt_bias"] = d.uniform(D, lo=-7.0, hi=-4.0)  # long memories
    lengths = ends(T)
    want, left = ref_call(wide(v), lengths)
    g = scan_gpu(v, lengths, True)
    so = torch.empty(B, D, N, device="cuda")
    y = Q.selective_scan(**g, state_out=so)
    close(y, want, scan_ops(T, N), "y")
    close(so, left, scan_ops(T, N), "state")
    for _ in range(3):
        state = g["state"].clone()
        assert torch.equal(Q.selective_scan(**{**g, "state": state}, state_out=state), y)
        assert torch.equal(state, so)


@pytest.mark.parametrize("T", [512, 1056])
@pytest.mark.parametrize("N", [3, 16, 40])
def test_backward(gpu, T, N):
    B, D = 6, 10
    v, _, d = scan_data(B, T, D, N, torch.float32, True, True, True, seed=6)
    v["dt_bias"] = d.uniform(D, lo=-7.0, hi=-4.0)
    lengths = ends(T)
    dy = d.normal(B, T, D)
    names = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")
    w = wide(v, names)
    grads = torch.autograd.grad((ref_call(w, lengths)[0] * dy.to(F64)).sum(), [w[k] for k in names])
    got = Q.selective_scan_backward(spoil(dy, lengths).cuda(), **scan_gpu(v, lengths, True))
    for k, want in zip(names, grads):
        close(getattr(got, "d" + k), want, 4 * scan_ops(T, N) + 8 * (B * T) ** 0.5, "d" + k)


def test_convolution_gradients_take_nothing_of_an_empty_sequence(gpu):
    """A voice without frames, its state whatever an unused slot holds."""
    B, T, D, W = 3, 9, 12, 4
    g = torch.Generator().manual_seed(1)
    x, dy = (torch.randn(B, T, D, generator=g).cuda() for _ in range(2))
    w, b, state = torch.randn(D, W, generator=g).cuda(), torch.randn(D, generator=g).cuda(), torch.randn(B, W - 1, D, generator=g)
    spoiled = state.clone()
    spoiled[1] = float("nan")
    lengths = torch.tensor([T, 0, 5], dtype=torch.int32, device="cuda")
    want = Q.causal_conv_backward(dy, x, w, b, state=state.cuda(), lengths=lengths)
    got = Q.causal_conv_backward(dy, x, w, b, state=spoiled.cuda(), lengths=lengths)
    for a, c in zip(got, want):
        assert torch.isfinite(a).all() and torch.equal(a, c)
