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
