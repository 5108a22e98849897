"""Sequence operators where their kernels take other shapes: the convolution's
tiles of 8 to 64 frames, the scan's chunks by the hundred, results in views,
operands that repeat or lie time-major.  Against 64 bits, with the tolerances
of test_gpu_sequence.  Needs a GPU."""
import pytest

torch = pytest.importorskip("torch")

from dgen_hip import sequence as Q  # noqa: E402
from test_gpu_sequence import EPS16, EPS32, F64, TYPES, Data, close, name_of, ref_call, scan_data, scan_gpu, scan_ops, spoil, wide  # noqa: E402

pytestmark = pytest.mark.gpu


# -------------------------------------------------------------- convolution
def conv_tile(B, T, D, backward):
    """Frames of a tile, as k_conv.hip takes them."""
    tile, groups = 64 if backward else 32, -(-D // 4)
    while tile > 8 and B * groups * -(-T // tile) < 131072:
        tile //= 2
    return tile


def within(got, want, tol, what):
    """On the GPU: |got - want| <= tol, element by element, without NaN."""
    err = (got.to(F64) - want).abs()
    assert bool((err <= tol).all()), f"{what}: off by {err.max().item():.3e}"


@pytest.mark.parametrize("B,T,D,forward,backward", [(4, 2500, 1000, 16, 16), (8, 2499, 1001, 32, 32), (32, 1030, 1024, 32, 64)])
@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("silu", [True, False])
def test_convolution_tiles(gpu, B, T, D, forward, backward, ty, silu):
    assert (conv_tile(B, T, D, False), conv_tile(B, T, D, True)) == (forward, backward)
    W, dev = 4, "cuda"
    g = torch.Generator(device=dev).manual_seed(B + T)
    x, dy = (torch.randn(B, T, D, generator=g, device=dev).to(ty) for _ in range(2))
    w, b = (torch.rand(D, W, generator=g, device=dev) * 2 - 1, torch.rand(D, generator=g, device=dev) - 0.5)
    state = torch.randn(B, W - 1, D, generator=g, device=dev).to(ty)
    n = torch.randint(T // 2, T + 1, (B,), generator=g, device=dev, dtype=torch.int32)
    n[0], n[1] = T, backward * 4 + 1
    ok = (torch.arange(T, device=dev)[None] < n[:, None])[..., None]
    xs = torch.cat([state.to(F64), torch.where(ok, x.to(F64), 0.0)], 1)
    u = b.to(F64) + sum(xs[:, i:i + T] * w[:, i].to(F64) for i in range(W))
    p = torch.sigmoid(u)
    want = torch.where(ok, u * p if silu else u, 0.0)
    bad = torch.where(ok, x.float(), float("nan")).to(ty)
    after = torch.empty_like(state)
    y = Q.causal_conv(bad, w, b, silu=silu, state=state, state_out=after, lengths=n)
    # W products and sums and the activation's operations, of the largest value; bfloat16 results round once more
    tol = 4 * (W + 10) * EPS32 * want.abs().max()
    within(y, want, tol + (EPS16 * 1.01 * want.abs() if ty == torch.bfloat16 else 0.0), f"y {name_of(ty)}")
    at = (n.long()[:, None] + torch.arange(W - 1, device=dev))[..., None].expand(B, W - 1, D)
    assert torch.equal(after.to(F64), xs.gather(1, at))
    du = torch.where(ok, dy.to(F64) * (p * (1 + u * (1 - p)) if silu else 1.0), 0.0)
    del u, p, want, y
    ahead = torch.cat([du, torch.zeros(B, W - 1, D, dtype=F64, device=dev)], 1)
    gx = torch.where(ok, sum(ahead[:, W - 1 - i:W - 1 - i + T] * w[:, i].to(F64) for i in range(W)), 0.0)
    gw = torch.stack([(xs[:, i:i + T] * du).sum((0, 1)) for i in range(W)], 1)
    gb = du.sum((0, 1))
    dx, dw, db = Q.causal_conv_backward(torch.where(ok, dy.float(), float("nan")).to(ty), bad, w, b, silu=silu, state=state,
                                        lengths=n)
    tol = 8 * (W + 16) * EPS32 * gx.abs().max()
    within(dx, gx, tol + (EPS16 * 1.01 * gx.abs() if ty == torch.bfloat16 else 0.0), f"dx {name_of(ty)}")
    sums = 64 + 8 * (B * T) ** 0.5
    within(dw, gw, sums * EPS32 * gw.abs().max(), "dweight")
    within(db, gb, sums * EPS32 * gb.abs().max(), "dbias")


# --------------------------------------------------------------------- scan
@pytest.mark.parametrize("B,T,ends", [(1, 2100, [2063]), (1, 8300, [8300]), (2, 8300, [8299, 4111]), (1, 16390, [16333])])
@pytest.mark.parametrize("ty", TYPES)
def test_scan_of_many_chunks(gpu, B, T, ends, ty):
    """66 to 260 chunks of 32 frames, 257 of 64."""
    D, N = 6, 16
    v, _, d = scan_data(B, T, D, N, ty, True, True, True, seed=7)
    v["dt_bias"] = d.uniform(D, lo=-7.0, hi=-4.0)  # long memories
    want, left = ref_call(wide(v), ends)
    g = scan_gpu(v, [min(T - 1, n) for n in ends] if max(ends) < T else [T - 1] * B, False)
    g["lengths"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
    so = torch.empty(B, D, N, device="cuda")
    y = Q.selective_scan(**g, state_out=so)
    close(y, want, scan_ops(T, N), f"y {name_of(ty)}")
    close(so, left, scan_ops(T, N), "state")
    state = g["state"].clone()
    assert torch.equal(Q.selective_scan(**{**g, "state": state}, state_out=state), y) and torch.equal(state, so)


@pytest.mark.parametrize("T,end", [(2100, 2063), (8300, 8290)])
@pytest.mark.parametrize("ty", TYPES)
def test_scan_gradients_of_many_chunks(gpu, T, end, ty):
    D, N = 6, 16
    v, _, d = scan_data(1, T, D, N, ty, True, True, True, seed=8)
    v["dt_bias"] = d.uniform(D, lo=-7.0, hi=-4.0)
    dy = d.normal(1, T, D, type=ty)
    names = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")
    w = wide(v, names)
    grads = torch.autograd.grad((ref_call(w, [end])[0] * dy.to(F64)).sum(), [w[k] for k in names])
    g = scan_gpu(v, [end], True)
    got = Q.selective_scan_backward(spoil(dy, [end]).cuda(), **g)
    for k, want in zip(names, grads):
        typed = name_of(ty) if k in ("x", "dt", "B", "C", "z") else ""
        close(getattr(got, "d" + k), want, 4 * scan_ops(T, N) + 8 * T ** 0.5, f"d{k} {typed}")


# ------------------------------------------------------- views and layouts
def within_wider(shape, ty, wide_by=5):
    """A view for a result and the tensor around it, NaN all over."""
    full = torch.full((*shape[:-1], shape[-1] + wide_by), float("nan"), dtype=ty, device="cuda")
    return full[..., 2:2 + shape[-1]], full


def untouched(full, width):
    return torch.isnan(full[..., :2]).all() and torch.isnan(full[..., 2 + width:]).all()


def time_major(t):
    return t.transpose(0, 1).contiguous().transpose(0, 1)


@pytest.mark.parametrize("ty", TYPES)
def test_results_in_views(gpu, ty):
    d = Data(11)
    x, r, w = d.normal(37, 50, type=ty).cuda(), d.normal(37, 50).cuda(), d.uniform(50).cuda()
    (out, full), (so, sfull) = within_wider((37, 50), ty), within_wider((37, 50), torch.float32)
    y, s = Q.rms_norm(x, w, residual=r)
    Q.rms_norm(x, w, residual=r, out=out, sum_out=so)
    assert torch.equal(out, y) and torch.equal(so, s) and untouched(full, 50) and untouched(sfull, 50)
    dx, _ = Q.rms_norm_backward(x, r, w)
    out, full = within_wider((37, 50), torch.float32)
    Q.rms_norm_backward(x, r, w, out=out)
    assert torch.equal(out, dx) and untouched(full, 50)
    for B, T, D in ((3, 70, 33), (2, 9, 3)):
        x, dy, w = d.normal(B, T, D, type=ty).cuda(), d.normal(B, T, D, type=ty).cuda(), d.uniform(D, 4).cuda()
        out, full = within_wider((B, T, D), ty)
        assert torch.equal(Q.causal_conv(x, w, out=out), Q.causal_conv(x, w)) and untouched(full, D)
        out, full = within_wider((B, T, D), ty)
        assert torch.equal(Q.causal_conv_backward(dy, x, w, out=out)[0], Q.causal_conv_backward(dy, x, w)[0])
        assert untouched(full, D)
        for T2 in (T, 200):  # one piece, and chunks
            v, lengths, _ = scan_data(B, T2, D, 16, ty, False, False, True)
            g = scan_gpu(v, lengths, False)
            out, full = within_wider((B, T2, D), ty)
            assert torch.equal(Q.selective_scan(**g, out=out), Q.selective_scan(**g)) and untouched(full, D)
            tm = torch.full((T2, B, D), float("nan"), dtype=ty, device="cuda").transpose(0, 1)
            assert torch.equal(Q.selective_scan(**g, out=tm), Q.selective_scan(**g))
    for rows, width, hidden in ((5, 40, 70), (150, 40, 70), (2400, 64, 1920)):
        x, a, b = d.normal(rows, width, type=ty).cuda(), d.normal(width, hidden, type=ty).cuda(), d.normal(width, hidden, type=ty).cuda()
        out, full = within_wider((rows, hidden), ty)
        assert torch.equal(Q.gated_mlp(x, a, b, out=out), Q.gated_mlp(x, a, b)) and untouched(full, hidden)


@pytest.mark.parametrize("ty", TYPES)
def test_operands_that_repeat_or_lie_time_major(gpu, ty):
    """As the same values in contiguous tensors, bit for bit."""
    d = Data(12)
    one = d.normal(1, 50, type=ty).cuda()
    x, w = one.expand(37, 50), d.uniform(50).cuda()
    r = d.normal(37, 50).cuda()
    for a, b in zip(Q.rms_norm(x, w, residual=r), Q.rms_norm(x.contiguous(), w, residual=r)):
        assert torch.equal(a, b)
    for a, b in zip(Q.rms_norm_backward(x, r, w, ds=r[:1].expand(37, 50)),
                    Q.rms_norm_backward(x.contiguous(), r, w, ds=r[:1].expand(37, 50).contiguous())):
        assert torch.equal(a, b)
    B, T, D, N = 3, 70, 33, 12
    taps = d.uniform(D, 4).cuda()
    for make in (time_major, lambda t: t[:1].expand(B, T, D), lambda t: t[:, :1].expand(B, T, D)):
        x, dy = make(d.normal(B, T, D, type=ty).cuda()), make(d.normal(B, T, D, type=ty).cuda())
        xc, dyc = x.contiguous(), dy.contiguous()
        assert torch.equal(Q.causal_conv(x, taps), Q.causal_conv(xc, taps))
        for a, b in zip(Q.causal_conv_backward(dy, x, taps)[:2], Q.causal_conv_backward(dyc, xc, taps)[:2]):
            assert torch.equal(a, b)
    for T2 in (20, T, 1100):  # one piece, chunks that join themselves, chunks with a carry
        v, lengths, _ = scan_data(B, T2, D, N, ty, False, True, True)
        g = scan_gpu(v, lengths, False)
        dy = d.normal(B, T2, D, type=ty).cuda()
        for make in (time_major, lambda t: t[:1].expand(B, *t.shape[1:]), lambda t: t[:, :1].expand(B, T2, t.shape[2])):
            h = {k: make(t) if k in ("x", "dt", "z", "B", "C") else t for k, t in g.items()}
            c = {k: None if t is None else t.contiguous() for k, t in h.items()}
            assert torch.equal(Q.selective_scan(**h), Q.selective_scan(**c))
            for a, b in zip(Q.selective_scan_backward(make(dy), **h), Q.selective_scan_backward(make(dy).contiguous(), **c)):
                assert torch.equal(a, b)
    for rows, width, hidden in ((5, 40, 70), (150, 40, 70)):
        x = d.normal(1, width, type=ty).cuda().expand(rows, width)
        a, b = d.normal(1, hidden, type=ty).cuda().expand(width, hidden), d.normal(width, hidden, type=ty).cuda()
        dh = d.normal(1, hidden, type=ty).cuda().expand(rows, hidden)
        assert torch.equal(Q.gated_mlp(x, a, b), Q.gated_mlp(x.contiguous(), a.contiguous(), b))
        for p, q in zip(Q.gated_mlp_backward(dh, x, a, b),
                        Q.gated_mlp_backward(dh.contiguous(), x.contiguous(), a.contiguous(), b)):
            assert torch.equal(p, q)
