"""The sizes that the sequence operators take and refuse, by the scratch query
(no device), and calls near them."""
import pytest

from test_sequence_abi import AT, scan, sequence, workspace


def scan_of(batch, T, D, N):
    return scan(batch=batch, T=T, D=D, N=N, x=(AT, T * D, D), y=(AT, T * D, D))


@pytest.mark.parametrize("batch,T,D,N", [(2048, 1, 1024, 16), (4096, 1, 1024, 64), (100000, 1, 1024, 16), (1 << 20, 1, 64, 16),
                                         (8192, 200, 512, 16)])
def test_scans_of_many_voices_are_taken(batch, T, D, N):
    """A call that does not cut time into chunks needs no launch to join them."""
    assert workspace("selective_scan", scan_of(batch, T, D, N), 0) == (0, 0)


@pytest.mark.parametrize("batch,T,D,N", [(1, 1 << 24, 64, 64), (1, 1 << 24, 1, 1), (159, 1 << 20, 64, 64)])
def test_scans_in_chunks(batch, T, D, N):
    rc, n = workspace("selective_scan", scan_of(batch, T, D, N), 0)
    assert rc == 0 and n > 0


@pytest.mark.parametrize("batch,T,D,N", [(1 << 20, 1, 1024, 16), ((1 << 20) + 1, 1, 1, 1), (2, 1 << 25, 8, 4)])
def test_scans_past_a_launch_are_refused(batch, T, D, N):
    assert workspace("selective_scan", scan_of(batch, T, D, N), 0)[0] == -1


@pytest.mark.gpu
def test_one_frame_of_many_voices(gpu):
    """As the halves of the voices, bit for bit."""
    torch = pytest.importorskip("torch")
    g = torch.Generator(device="cuda").manual_seed(1)
    B, D, N = 2100, 1024, 16
    x, dt, z = (torch.randn(B, 1, D, generator=g, device="cuda") for _ in range(3))
    Bm, Cm = (torch.randn(B, 1, N, generator=g, device="cuda") for _ in range(2))
    A, h = -torch.rand(D, N, generator=g, device="cuda"), torch.randn(B, D, N, generator=g, device="cuda")
    after, parts = torch.empty_like(h), torch.empty_like(h)
    y = sequence.selective_scan(x, dt, A, Bm, Cm, z=z, state=h, state_out=after)
    for s in (slice(0, 1050), slice(1050, B)):
        part = sequence.selective_scan(x[s], dt[s], A, Bm[s], Cm[s], z=z[s], state=h[s], state_out=parts[s])
        assert torch.equal(part, y[s])
    assert torch.equal(after, parts)
    step = torch.nn.functional.softplus(dt[-1, 0].double())
    last = torch.exp(step[:, None] * A) * h[-1] + (step * x[-1, 0])[:, None] * Bm[-1]
    assert (after[-1] - last).abs().max() < 1e-5
