"""Sequence operators on tensors of more than 2^31 elements: the last rows and
frames are those of a call on them alone.  Needs a GPU (up to 20 GB of it)."""
import pytest

torch = pytest.importorskip("torch")

from dgen_hip import sequence as Q  # noqa: E402

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def pattern(*shape, seed=0):
    """bfloat16 values of about unit size, without a second large tensor: a
    random run of odd length, repeated."""
    n = 1
    for s in shape:
        n *= s
    run = torch.randn(65521, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(BF16)
    return run.repeat(-(-n // len(run)))[:n].view(shape)


@pytest.fixture(autouse=True)
def memory_back():
    yield
    torch.cuda.empty_cache()


def test_norm(gpu):
    rows, n = (1 << 20) + 5, 2100
    x, w = pattern(rows, n), torch.rand(n, device="cuda") + 0.5
    assert x.numel() > 1 << 31
    y = Q.rms_norm(x, w)
    assert torch.equal(y[-70:], Q.rms_norm(x[-70:], w)) and torch.equal(y[:70], Q.rms_norm(x[:70], w))
    dx, _ = Q.rms_norm_backward(x, x, w, out=y)
    assert torch.equal(dx[-70:], Q.rms_norm_backward(x[-70:], x[-70:], w)[0])


def test_convolution(gpu):
    T, D, W = (1 << 20) + 77, 2052, 4
    x, w = pattern(1, T, D), torch.rand(D, W, device="cuda") - 0.5
    assert x.numel() > 1 << 31
    left = torch.empty(1, W - 1, D, dtype=BF16, device="cuda")
    y = Q.causal_conv(x, w, state_out=left)
    assert torch.equal(y[:, -50:], Q.causal_conv(x[:, -50:], w, state=x[:, -50 - W + 1:-50].contiguous()))
    assert torch.equal(left, x[:, -W + 1:])
    dx, dw, _ = Q.causal_conv_backward(x, x, w, silu=False, out=y)
    # dx[t] = sum_i w[i] dy[t + W - 1 - i], dy = x here
    tail = x[0, -40:].double()
    ahead = torch.cat([tail, torch.zeros(W - 1, D, dtype=torch.float64, device="cuda")])
    want = sum(ahead[W - 1 - i:W - 1 - i + 40] * w[:, i].double() for i in range(W))
    assert ((dx[0, -40:].double() - want).abs() <= 2.0 ** -8 * 1.01 * want.abs() + 1e-5).all()
    assert torch.isfinite(dw).all()


def test_scan(gpu):
    """The last frames from the state before them; in 32 bits of a state of
    unit size that forgets within a thousand frames."""
    T, D, N = (1 << 20) + 77, 2052, 4
    x, dt, Bm, Cm = pattern(1, T, D), pattern(1, T, D, seed=1), pattern(1, T, N, seed=2), pattern(1, T, N, seed=3)
    A = -(torch.rand(D, N, device="cuda") + 0.5)
    h, mid = torch.empty(1, D, N, device="cuda"), torch.empty(1, D, N, device="cuda")
    y = Q.selective_scan(x, dt, A, Bm, Cm, state_out=h)
    cut = T - 45
    near = slice(cut - 1000, cut)
    Q.selective_scan(x[:, near], dt[:, near], A, Bm[:, near], Cm[:, near], state_out=mid)
    last = slice(cut, T)
    part = Q.selective_scan(x[:, last], dt[:, last], A, Bm[:, last], Cm[:, last], state=mid, state_out=mid)
    assert (mid - h).abs().max() <= 1e-4
    want = part.float()
    assert ((y[:, last].float() - want).abs() <= 2.0 ** -7 * want.abs() + 1e-3).all()


@pytest.mark.parametrize("hidden", [2080, 2077])
def test_gated_block(gpu, hidden):
    """Past 2^31 in the result, and (its rows and columns exchanged) in the operand."""
    rows, width = (1 << 20) + 40, 64
    for n, f in ((width, hidden), (hidden, width)):
        x, a, b = pattern(rows, n), pattern(n, f, seed=1) * 0.125, pattern(n, f, seed=2) * 0.125
        assert rows * max(n, f) > 1 << 31
        h = Q.gated_mlp(x, a, b)
        for part in (slice(0, 200), slice(rows - 200, rows)):
            t = x[part].double()
            g, u = t @ a.double(), t @ b.double()
            want = g * torch.sigmoid(g) * u
            size = (t.abs() @ a.double().abs()) * u.abs() * 1.2 + g.abs() * (t.abs() @ b.double().abs())
            bound = (n + 32) * 2.0 ** -24 * (size + want.abs()) + 2.0 ** -8 * 1.01 * want.abs() + 1e-30
            assert ((h[part].double() - want).abs() <= bound).all()
        del x, h
