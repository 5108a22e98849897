"""Sequence operators on infinities and very large values: where the formula's
result is a number or an infinity, so is the operator's.  Needs a GPU."""
import pytest

torch = pytest.importorskip("torch")

from dgen_hip import sequence as Q  # noqa: E402

pytestmark = pytest.mark.gpu
F64 = torch.float64
INF = float("inf")


def alike(got, want, what, rtol=1e-5, atol=1e-6):
    """Infinities and NaN in the same places, numbers within rtol and atol."""
    want = want.to(torch.float32)
    ok = torch.isclose(got.detach().cpu().float(), want.cpu(), rtol=rtol, atol=atol, equal_nan=True)
    assert ok.all(), f"{what}: {got.cpu()[~ok][:4].tolist()} for {want.cpu()[~ok][:4].tolist()}"


@pytest.mark.parametrize("T,at", [(20, 19), (20, 7), (20, 8), (41, 31), (13, 12)])
@pytest.mark.parametrize("ty", [torch.float32, torch.bfloat16])
def test_weight_gradients_of_a_convolution_with_an_infinite_frame(gpu, T, at, ty):
    """Frames past a tile's or a sequence's end add nothing to its sums, not
    even 0 times what lies before them."""
    B, D, W = 2, 6, 4
    g = torch.Generator().manual_seed(T + at)
    x, dy = (torch.rand(B, T, D, generator=g).add(0.5).to(ty) for _ in range(2))
    w = torch.rand(D, W, generator=g) + 0.5
    x[0, at, 2] = INF
    x[1, 2, 3] = INF
    n = [T, 3]
    dw = torch.zeros(D, W, dtype=F64)
    for b in range(B):
        row = torch.cat([torch.zeros(W - 1, D, dtype=F64), x[b, :n[b]].to(F64)])
        for t in range(n[b]):
            dw += (dy[b, t].to(F64) * row[t:t + W]).T
    lengths = torch.tensor(n, dtype=torch.int32, device="cuda")
    _, got, _ = Q.causal_conv_backward(dy.cuda(), x.cuda(), w.cuda(), silu=False, lengths=lengths)
    assert torch.isinf(dw).any() and not torch.isnan(dw).any()
    alike(got, dw, "dweight")
