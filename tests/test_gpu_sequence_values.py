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


@pytest.mark.parametrize("N", [1, 3, 5, 12, 16, 33])
@pytest.mark.parametrize("T", [9, 100, 1100])
@pytest.mark.parametrize("which", ["x", "dt"])
def test_scan_with_an_infinite_value(gpu, N, T, which):
    """An infinite input, or step, makes its channel infinite from that frame
    on, whatever the number of states."""
    B, D, at = 2, 5, T // 2 + 1
    g = torch.Generator().manual_seed(N + T)
    x, Bm, Cm = (torch.rand(B, T, n, generator=g) + 0.5 for n in (D, N, N))
    dt, A = torch.randn(B, T, D, generator=g) - 2.0, -(torch.rand(D, N, generator=g) + 0.1)
    (x if which == "x" else dt)[1, at, 3] = INF
    h, ys = torch.zeros(B, D, N, dtype=F64), []
    step = torch.nn.functional.softplus(dt.to(F64), threshold=1e9)
    for t in range(T):
        u = (step[:, t] * x[:, t].to(F64))[..., None] * Bm[:, t, None].to(F64)
        h = torch.exp(step[:, t, :, None] * A.to(F64)) * h + u
        ys.append((h * Cm[:, t, None].to(F64)).sum(-1))
    want = torch.stack(ys, 1)
    assert torch.isinf(want[1, at:, 3]).all() and not torch.isnan(want).any()
    after = torch.empty(B, D, N, device="cuda")
    y = Q.selective_scan(x.cuda(), dt.cuda(), A.cuda(), Bm.cuda(), Cm.cuda(), state_out=after)
    alike(y, want, "y", rtol=1e-4)
    alike(after, h, "state", rtol=1e-4)


@pytest.mark.parametrize("N", [3, 12, 16])
def test_scan_gradients_beside_an_infinite_channel(gpu, N):
    """The last channel's states are infinite from the middle on: its gradients
    and the shared ones are infinite as the formula's, the other channels' are
    numbers."""
    B, T, D, at = 1, 48, 5, 20
    g = torch.Generator().manual_seed(N)
    x, Bm, Cm, dy = (torch.rand(B, T, n, generator=g) + 0.5 for n in (D, N, N, D))
    dt, A = torch.randn(B, T, D, generator=g) - 2.0, -(torch.rand(D, N, generator=g) + 0.1)
    x[0, at, D - 1] = INF
    got = Q.selective_scan_backward(dy.cuda(), x.cuda(), dt.cuda(), A.cuda(), Bm.cuda(), Cm.cuda())
    # dC[t] = sum over channels of h[t] dy[t]
    dC = got.dC[0].cpu()
    assert torch.isfinite(dC[:at]).all() and (dC[at:] == INF).all()
    assert torch.isfinite(got.dx[..., :D - 1]).all() and torch.isfinite(got.ddt[..., :D - 1]).all()
    assert torch.isfinite(got.dx).all() and torch.isfinite(got.dA[:D - 1]).all()


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("ty", [torch.float32, torch.bfloat16])
def test_slopes_of_the_activations_far_out(gpu, act, ty):
    """There the slope is 0 or 1 (powers of the argument in GELU's overflow)."""
    x = torch.tensor([[-1e14], [-1e8], [-1e7], [1e7], [1e8], [1e14]], dtype=ty).repeat(30, 1)
    wg, wu = torch.full((1, 5), 1e6, dtype=ty), torch.full((1, 5), 1e-14, dtype=ty)
    dh = torch.ones(len(x), 5, dtype=ty)
    dx, dwg, dwu = Q.gated_mlp_backward(dh.cuda(), x.cuda(), wg.cuda(), wu.cuda(), activation=act)
    a, b, c = x.to(F64), wg.to(F64), wu.to(F64)
    on = (a > 0).to(F64)
    dg, du = a @ c * on, a @ b * on
    rtol = 2.0 ** -6 if ty == torch.bfloat16 else 1e-5  # bfloat16: three roundings of 2^-8
    alike(dx, dg @ b.T + du @ c.T, "dx", rtol, 0.0)
    alike(dwg, a.T @ dg, "dw_gate", rtol, 0.0)
    alike(dwu, a.T @ du, "dw_up", rtol, 0.0)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("rows", [3, 150])
@pytest.mark.parametrize("ty", [torch.float32, torch.bfloat16])
def test_a_value_that_is_none_stays_so(gpu, act, rows, ty):
    """NaN in a row reaches that row's results and gradients and the weights'
    gradients, and no other row."""
    g = torch.Generator().manual_seed(rows)
    x, wg, wu = (torch.randn(*s, generator=g).to(ty) for s in ((rows, 20), (20, 30), (20, 30)))
    dh = torch.randn(rows, 30, generator=g).to(ty)
    x[1, 4] = float("nan")
    h = Q.gated_mlp(x.cuda(), wg.cuda(), wu.cuda(), activation=act).isnan().cpu()
    grads = Q.gated_mlp_backward(dh.cuda(), x.cuda(), wg.cuda(), wu.cuda(), activation=act)
    dx, dwg, dwu = (t.isnan().cpu() for t in grads)
    for t in (h, dx):
        assert t[1].all() and not t[0].any() and not t[2:].any()
    assert dwg.all() and dwu.all()


def form(x, wg, wu):
    """Projections in 64 bits rounded to 32 (a sum that overflows there is an
    infinity), and the activation and its slope."""
    g, u = ((x.to(F64) @ w.to(F64)).float().to(F64) for w in (wg, wu))
    p = torch.sigmoid(g)
    return g, u, (g * p).float().to(F64), p * (1 + g * (1 - p))


# rows of the kernel for a few, of the tiles; a reduction in one and in several pieces
@pytest.mark.parametrize("rows,width,hidden", [(3, 40, 70), (200, 40, 70), (300, 65, 1000), (2000, 96, 1408)])
@pytest.mark.parametrize("value", [INF, -INF, 3.4e38, -3.4e38])
@pytest.mark.parametrize("where", ["x", "w"])
def test_gated_block_of_32_bits_with_a_value_past_bfloat16(gpu, rows, width, hidden, value, where):
    """The products take their operands in bfloat16 parts, whose largest is
    3.39e38: what lies above, and an infinity, gives what it gives in 32 bits,
    however many rows there are.  Numbers are within the bound of sums of
    `width` products in 32 bits, passed on by the activation and the product."""
    g = torch.Generator().manual_seed(rows)
    x, wg, wu = (torch.randn(*s, generator=g) * 0.1 for s in ((rows, width), (width, hidden), (width, hidden)))
    if where == "x":
        x[2, 7] = value
    else:
        wu[7, 3] = value
    _, u, f, _ = form(x, wg, wu)
    want = f * u
    of_gate, of_up = (x.abs().to(F64) @ w.abs().to(F64) for w in (wg, wu))
    bound = (width + 32) * 2.0 ** -24 * (of_gate * u.abs() * 1.2 + f.abs() * of_up + want.abs()) + 1e-30
    got = Q.gated_mlp(x.cuda(), wg.cuda(), wu.cuda()).cpu()
    same = (got == want.float()) | (got.isnan() & want.isnan())
    ok = same | (torch.isfinite(got) & torch.isfinite(want) & ((got.to(F64) - want).abs() <= bound))
    assert torch.isinf(want.float()).any() or abs(value) < INF
    assert ok.all(), (got[~ok][:4], want[~ok][:4])


@pytest.mark.parametrize("rows,width,hidden", [(3, 40, 70), (200, 40, 70), (300, 65, 1000), (2000, 96, 1408)])
@pytest.mark.parametrize("value", [INF, 3.4e38])
def test_gradients_of_the_gated_block_of_32_bits_with_a_value_past_bfloat16(gpu, rows, width, hidden, value):
    g = torch.Generator().manual_seed(rows + 1)
    x, wg, wu = (torch.rand(*s, generator=g) * 0.1 + 0.01 for s in ((rows, width), (width, hidden), (width, hidden)))
    dh = torch.rand(rows, hidden, generator=g) + 0.1
    dh[1, 5] = value
    dx, dwg, dwu = Q.gated_mlp_backward(dh.cuda(), x.cuda(), wg.cuda(), wu.cuda())
    _, u, f, slope = form(x, wg, wu)
    dg, du = (dh.to(F64) * u * slope).float().to(F64), (dh.to(F64) * f).float().to(F64)
    # (everything is positive: no infinity meets its opposite, and a sum of K
    # products is within about K 2^-24 of itself, 2000 at most here)
    alike(dx, dg @ wg.to(F64).T + du @ wu.to(F64).T, "dx", 1.2e-4)
    alike(dwg, x.to(F64).T @ dg, "dw_gate", 1.2e-4)
    alike(dwu, x.to(F64).T @ du, "dw_up", 1.2e-4)


def test_norm_of_small_rows_without_eps(gpu):
    """A mean square below the smallest normal number, 2^-126."""
    w = torch.ones(8, device="cuda")
    for e in (0, -60, -62, -64, -66):
        x = torch.full((3, 8), 2.0 ** e, device="cuda")
        y = Q.rms_norm(x, w, eps=0.0)
        assert ((y - 1).abs() <= 1e-6).all(), (e, y[0, 0].item())
        dx, dw = Q.rms_norm_backward(torch.ones_like(x), x, w, eps=0.0)
        assert torch.isfinite(dx).all() and ((dw - 3).abs() <= 1e-5).all()
