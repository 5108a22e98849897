"""The sizes that the sequence operators take and refuse, by the scratch query
(no device), and calls near them."""
import pytest

from test_sequence_abi import AT, message, scan, sequence, workspace


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


@pytest.mark.parametrize("T,taken", [(1, True), (2, False)])
def test_the_stride_of_a_single_frame_says_nothing(T, taken):
    """One frame out of a time-major recording of many voices."""
    d = scan(batch=4, T=T, D=8, x=(AT, 8, 1 << 27), y=(AT, 40, 8))
    assert (workspace("selective_scan", d, 0) == (0, 0)) is taken


def mlp_of(rows, width, hidden, type, backward, x=AT):
    grads = (AT, hidden, AT, width, AT, hidden, AT, hidden) if backward else (0,) * 8
    return sequence._MLP.pack(sequence._MLP_SIZE, type, 0, 0, rows, width, hidden, x, width, AT, hidden, AT, hidden,
                              *((0, 0) if backward else (AT, hidden)), *grads)


@pytest.mark.parametrize("rows,width,hidden,type,backward,x,taken", [
    (300, 1 << 16, (1 << 17) - 32, 1, 1, AT, True),    # weight gradients joined by just under 2^32 threads
    (300, 1 << 16, 1 << 17, 1, 1, AT, False),
    (1 << 21, 1 << 13, 1 << 13, 1, 0, AT + 2, True),   # x packed by 2^31 threads
    (1 << 22, 1 << 13, 64, 1, 0, AT + 2, False),
    (1 << 22, 1 << 13, 64, 1, 0, AT, True),            # (aligned: not packed)
    (64, 64, 128, 0, 1, AT, True),
])
def test_gated_blocks_past_a_launch_are_refused(rows, width, hidden, type, backward, x, taken):
    rc, _ = workspace("gated_mlp", mlp_of(rows, width, hidden, type, backward, x), backward)
    assert (rc == 0) is taken
    assert taken or "too large" in message()


@pytest.mark.parametrize("type", [0, 1])
def test_calls_that_the_binding_gives_no_scratch_need_none(type):
    """sequence.py asks for no scratch for scans of up to 32 frames and gated
    blocks of up to 16 rows and 8192 columns."""
    for T in (1, 2, 31, 32):
        for batch in (1, 3, 64, 5000):
            for D in (1, 64, 65, 1024):
                for N in (1, 16, 17, 64):
                    d = scan(type=type, batch=batch, T=T, D=D, N=N, x=(AT, T * D, D), y=(AT, T * D, D))
                    assert workspace("selective_scan", d, 0) == (0, 0), (batch, T, D, N)
    for rows in (1, 2, 8, 9, 15, 16):
        for width in (1, 33, 512, 4096):
            for hidden in (1, 16, 1408, 4096, 4097, 8191, 8192):
                for x in (AT, AT + 4):
                    assert workspace("gated_mlp", mlp_of(rows, width, hidden, type, 0, x), 0) == (0, 0), (rows, width, hidden)


@pytest.mark.gpu
def test_a_single_frame_with_a_far_stride(gpu):
    torch = pytest.importorskip("torch")
    g = torch.Generator().manual_seed(2)
    B, D, N = 3, 40, 8
    x, dt, Bm, Cm = (torch.randn(B, n, generator=g).cuda() for n in (D, D, N, N))
    A = -torch.rand(D, N, generator=g).cuda()
    far = [t.as_strided((B, 1, t.shape[1]), (t.shape[1], 1 << 40, 1)) for t in (x, dt, Bm, Cm)]
    assert torch.equal(sequence.selective_scan(far[0], far[1], A, far[2], far[3]),
                       sequence.selective_scan(x[:, None], dt[:, None], A, Bm[:, None], Cm[:, None]))
    got = sequence.selective_scan_backward(far[0], far[0], far[1], A, far[2], far[3])
    want = sequence.selective_scan_backward(x[:, None], x[:, None], dt[:, None], A, Bm[:, None], Cm[:, None])
    for a, b in zip(got, want):
        assert a is b is None or torch.equal(a, b)


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
