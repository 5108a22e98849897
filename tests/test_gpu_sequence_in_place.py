"""Sequence operators whose results lie over their operands: the results of
calls with places of their own, bit for bit, nothing else touched.  Needs a
GPU."""
import pytest

torch = pytest.importorskip("torch")

from dgen_hip import sequence as Q  # noqa: E402
from test_gpu_sequence import TYPES, Data, scan_data, scan_gpu  # noqa: E402

pytestmark = pytest.mark.gpu


def shifted(t, by):
    """A copy of t in a buffer, and the view `by` elements further on in it."""
    flat = torch.empty(t.numel() + by, dtype=t.dtype, device="cuda")
    a = flat[:t.numel()].view(t.shape)
    a.copy_(t)
    return a, flat[by:].view(t.shape)


@pytest.mark.parametrize("ty", TYPES)
def test_norm(gpu, ty):
    d = Data(1)
    for rows, n in ((5, 7), (300, 512), (40, 2500), (3, 9000)):
        x, r, w = d.normal(rows, n, type=ty).cuda(), d.normal(rows, n, type=ty, scale=2.0).cuda(), d.uniform(n).cuda()
        y, s = Q.rms_norm(x, w, residual=r)
        for out, sums in ((0, 1), (1, 0), (0, None), (None, 0), (1, None), (None, 1)):
            ins = [x.clone(), r.clone()]
            places = [None if i is None else ins[i] for i in (out, sums)]
            got = Q.rms_norm(ins[0], w, residual=ins[1], out=places[0], sum_out=places[1])
            for g, want, place in zip(got, (y, s), places):
                assert torch.equal(g, want) and (place is None or g is place)
        for by in (1, n, n + 3):
            a, over = shifted(x, by)
            assert torch.equal(Q.rms_norm(a, w, residual=r, out=over)[0], y) and torch.equal(over, y)
            a, over = shifted(r, by)
            assert torch.equal(Q.rms_norm(x, w, residual=a, sum_out=over)[1], s) and torch.equal(over, s)
        dy, ds = d.normal(rows, n, type=ty).cuda(), d.normal(rows, n, type=ty).cuda()
        dx, dw = Q.rms_norm_backward(dy, s, w, ds=ds)
        for k in range(3):
            ins = [dy.clone(), s.clone(), ds.clone()]
            got = Q.rms_norm_backward(ins[0], ins[1], w, ds=ins[2], out=ins[k])
            assert got[0] is ins[k] and torch.equal(got[0], dx) and torch.equal(got[1], dw)
        a, over = shifted(s, n + 1)
        got = Q.rms_norm_backward(dy, a, w, ds=ds, out=over)
        assert torch.equal(over, dx) and torch.equal(got[1], dw)


@pytest.mark.parametrize("B,T,D", [(3, 1, 40), (2, 50, 33), (4, 300, 700), (1, 3, 6)])
@pytest.mark.parametrize("ty", TYPES)
def test_convolution(gpu, B, T, D, ty):
    d, W = Data(2), 4
    x, dy = d.normal(B, T, D, type=ty).cuda(), d.normal(B, T, D, type=ty).cuda()
    w, b = d.uniform(D, W).cuda(), d.uniform(D).cuda()
    state = d.normal(B, W - 1, D, type=ty).cuda()
    left = torch.empty_like(state)
    y = Q.causal_conv(x, w, b, state=state, state_out=left)
    a = x.clone()
    assert Q.causal_conv(a, w, b, state=state, out=a) is a and torch.equal(a, y)
    for by in (1, D, T * D):
        a, over = shifted(x, by)
        Q.causal_conv(a, w, b, state=state, out=over)
        assert torch.equal(over, y)
        a, over = shifted(state, by)
        Q.causal_conv(x, w, b, state=a, state_out=over)
        assert torch.equal(over, left)
    dx, dw, db = Q.causal_conv_backward(dy, x, w, b, state=state)
    for k in range(2):
        ins = [dy.clone(), x.clone()]
        got = Q.causal_conv_backward(ins[0], ins[1], w, b, state=state, out=ins[k])
        assert got[0] is ins[k]
        for p, q in zip(got, (dx, dw, db)):
            assert torch.equal(p, q)
    # the halves of one tensor are apart
    xz = torch.cat([x, torch.zeros_like(x)], -1)
    assert torch.equal(Q.causal_conv(xz[..., :D], w, b, state=state, out=xz[..., D:]), y)
    assert torch.equal(xz[..., :D], x)


@pytest.mark.parametrize("B,T,D,N", [(3, 1, 40, 16), (2, 70, 33, 12), (2, 1200, 70, 16), (2, 40, 16, 16)])
@pytest.mark.parametrize("ty", TYPES)
def test_scan(gpu, B, T, D, N, ty):
    v, lengths, _ = scan_data(B, T, D, N, ty, False, True, True)
    g = scan_gpu(v, lengths, False)
    left = torch.empty_like(g["state"])
    y = Q.selective_scan(**g, state_out=left)
    for k in ("x", "dt", "z") + (("B", "C") if D == N else ()):
        h = {**g, k: g[k].clone()}
        after = torch.empty_like(left)
        assert Q.selective_scan(**h, out=h[k], state_out=after) is h[k]
        assert torch.equal(h[k], y) and torch.equal(after, left)
        a, over = shifted(g[k], D + 1)
        if a.shape == y.shape:
            Q.selective_scan(**{**g, k: a}, out=over)
            assert torch.equal(over, y)
    a, over = shifted(g["state"], N)
    Q.selective_scan(**{**g, "state": a}, state_out=over)
    assert torch.equal(over, left)


@pytest.mark.parametrize("rows,n", [(3, 64), (200, 64), (4200, 1024)])
@pytest.mark.parametrize("ty", TYPES)
def test_gated_block(gpu, rows, n, ty):
    d = Data(3)
    x, a, b = d.normal(rows, n, type=ty).cuda(), d.normal(n, n, type=ty).cuda(), d.normal(n, n, type=ty).cuda()
    h = Q.gated_mlp(x, a, b)
    c = x.clone()
    assert Q.gated_mlp(c, a, b, out=c) is c and torch.equal(c, h)
    c, over = shifted(x, n + 8)
    Q.gated_mlp(c, a, b, out=over)
    assert torch.equal(over, h)


def test_two_results_in_one_place_are_refused(gpu):
    x, w = torch.zeros(4, 6, 8, device="cuda"), torch.zeros(8, 4, device="cuda")
    with pytest.raises(ValueError):
        Q.rms_norm(x, w[:, 0].contiguous(), residual=x, out=x, sum_out=x)
    out = torch.zeros(4, 6, 8, device="cuda")
    with pytest.raises(ValueError):
        Q.causal_conv(x, w, out=out, state_out=out.view(-1)[:96].view(4, 3, 8))
    with pytest.raises(ValueError):
        Q.selective_scan(x, x, w, x[..., :4], x[..., :4], out=out, state_out=out.view(-1)[:128].view(4, 8, 4))
