"""The norms around a block (dgen_hip.sequence.block_norm) against their
definition in 64 bits, forward and backward, with each kind of gate.  Needs a GPU.

Tolerances, in roundings of fp32 (2^-24) relative to the largest magnitude on
the way: a sum of n squares is at most 40 additions a thread and 10 levels over
threads deep, and both norms chain two of those; sums over rows grow as the
square root of their number.  bfloat16 results are rounded once more."""
import pytest

torch = pytest.importorskip("torch")

from dgen_hip import sequence as Q  # noqa: E402
from test_gpu_sequence import F64, TYPES, Data, close, gpu_view, name_of  # noqa: E402

pytestmark = pytest.mark.gpu
EPS = 1e-5


def block(x, post, r, pre, gate, act, scale):
    n = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * post
    if gate is not None:
        n = (torch.sigmoid(gate) if act == "sigmoid" else gate) * n
    s = n + (r if scale is None else scale * r)
    return s / torch.sqrt(s.square().mean(-1, keepdim=True) + EPS) * pre, s


SIZES = [(1, 1, 1), (2, 3, 7), (3, 5, 64), (1, 2, 129), (40, 2, 130), (2, 30, 512), (3, 4, 513), (2, 9, 1023), (1, 3, 2049), (2, 2, 4500),
         (1, 1, 8192), (2, 1500, 33), (700, 3, 20), (1, 5000, 16)]


@pytest.mark.parametrize("B,T,n", SIZES)
@pytest.mark.parametrize("xt,st", [(0, 0), (1, 0), (1, 1), (0, 1)])
@pytest.mark.parametrize("gate,act,scale", [("rows", "sigmoid", True), ("clips", "sigmoid", False), ("clips", "none", True), (None, "none", False)])
def test_both_ways(gpu, B, T, n, xt, st, gate, act, scale):
    xt, st = TYPES[xt], TYPES[st]
    d = Data(B + 3 * T + 5 * n)
    x, r = d.normal(B, T, n, type=xt), d.normal(B, T, n, type=st, scale=2.0)
    post, pre = d.uniform(n, lo=0.5, hi=1.5), d.uniform(n, lo=0.5, hi=1.5)
    z = None if gate is None else d.normal(B, T if gate == "rows" else 1, n, type=xt)
    w = d.uniform(n, lo=0.8, hi=1.2) if scale else None

    def up(t, grad=False):
        return None if t is None else t.to(F64).requires_grad_(grad)

    def there(t):
        return None if t is None else t.cuda()

    def view(t, wide, lead):  # columns of a wider tensor, as rows
        if t is None:
            return None
        return gpu_view(t.reshape(-1, n), wide, lead)

    extra = dict(gate_activation=act, residual_scale=there(w), eps=EPS)
    y, s = Q.block_norm(x.cuda(), post.cuda(), r.cuda(), pre.cuda(), gate=there(z), **extra)
    wy, ws = block(up(x), up(post), up(r), up(pre), up(z), act, up(w))
    close(y, wy, 150, f"y {name_of(xt)}")
    close(s, ws, 80, f"s {name_of(st)}")
    assert y.dtype == xt and s.dtype == st
    if gate != "clips":  # views of rows
        y2, s2 = Q.block_norm(view(x, 3, 1), post.cuda(), view(r, 5, 2), pre.cuda(), gate=view(z, 2, 1), **extra)
        assert torch.equal(y2, y.view(-1, n)) and torch.equal(s2, s.view(-1, n))
    # backward, from the stored sum
    dy, ds = d.normal(B, T, n, type=xt), d.normal(B, T, n, type=st)
    stored = ws.to(st)
    ins = [up(t, True) for t in (x, post, r, pre)]
    z64, w64 = up(z, True), up(w, True)
    _, sum64 = block(*ins, z64, act, w64)
    # (the gradient passes the rounding of the stored sum as it is)
    through = sum64 + (stored.to(F64) - sum64).detach()
    out = through / torch.sqrt(through.square().mean(-1, keepdim=True) + EPS) * ins[3]
    leaves = [t for t in (*ins, z64, w64) if t is not None]
    grads = dict(zip([k for k, t in zip(("x", "post", "r", "pre", "z", "w"), (*ins, z64, w64)) if t is not None],
                     torch.autograd.grad((out * dy.to(F64)).sum() + (through * ds.to(F64)).sum(), leaves)))
    got = Q.block_norm_backward(dy.cuda(), x.cuda(), r.cuda() if scale else None, stored.cuda(), post.cuda(), pre.cuda(), gate=there(z),
                                ds=ds.cuda(), **extra)
    # (the terms of dx and of the sum's gradient cancel, entirely where n = 1)
    rs = torch.rsqrt(stored.to(F64).square().mean(-1, keepdim=True) + EPS)
    da = ((dy.to(F64) * pre.to(F64)).abs() * rs).max().item() * 2 + ds.to(F64).abs().max().item()
    rx = torch.rsqrt(x.to(F64).square().mean(-1, keepdim=True) + EPS).max().item()
    most = 1.0 if z is None else max(1.0, z.to(F64).abs().max().item()) if act == "none" else 1.0
    close(got.dresidual, grads["r"], 200, f"dresidual {name_of(st)}", 1.2 * da)
    close(got.dx, grads["x"], 400, f"dx {name_of(xt)}", 2 * 1.5 * da * rx * most)
    over = 64 + 8 * (B * T) ** 0.5
    norm = (x.to(F64).abs().max() * rx).item() + 1.0
    close(got.dpre, grads["pre"], 150 + over, "dpre", max(1.0, grads["pre"].abs().max().item()))
    close(got.dpost, grads["post"], 300 + over, "dpost", max(da * most * min(norm, n ** 0.5), grads["post"].abs().max().item()))
    assert (got.dgate is None) == (z is None) and (got.dresidual_scale is None) == (w is None)
    if z is not None:
        assert got.dgate.shape == z.shape
        close(got.dgate, grads["z"], 300 + (0 if gate == "rows" else 8 * T ** 0.5 + 64), f"dgate {name_of(xt)}",
              max(1.5 * da * min(norm, n ** 0.5), grads["z"].abs().max().item()))
    if w is not None:
        close(got.dresidual_scale, grads["w"], 200 + over, "dscale",
              max(da * r.to(F64).abs().max().item(), grads["w"].abs().max().item()))


def test_gradients_against_differences(gpu):
    B, T, n = 2, 5, 40
    d = Data(3)
    a = dict(x=d.normal(B, T, n).cuda(), post_weight=d.uniform(n, lo=0.5, hi=1.5).cuda(), residual=d.normal(B, T, n).cuda(),
             pre_weight=d.uniform(n, lo=0.5, hi=1.5).cuda(), gate=d.normal(B, 1, n).cuda(),
             residual_scale=d.uniform(n, lo=0.8, hi=1.2).cuda())
    dy, ds = d.normal(B, T, n).cuda(), d.normal(B, T, n).cuda()
    got = Q.block_norm_backward(dy, s=Q.block_norm(**a)[1], ds=ds, **a)
    for k, g in zip(("x", "residual", "gate", "post_weight", "pre_weight", "residual_scale"), got):
        u = d.normal(*a[k].shape).cuda()
        u /= u.norm()
        e = 1e-2
        (y1, s1), (y0, s0) = (Q.block_norm(**{**a, k: a[k] + sign * e * u}) for sign in (1, -1))
        num = (((y1 - y0).double() * dy).sum() + ((s1 - s0).double() * ds).sum()) / (2 * e)
        ana = (g.double() * u).sum()
        assert abs(num - ana) <= 2e-3 * max(1.0, abs(ana.item())), (k, num.item(), ana.item())


def test_gates_far_out(gpu):
    """A closed gate lets nothing through, an open one everything, and their
    gradients end at 0 without a NaN."""
    n = 16
    x, r, w = torch.ones(1, n, device="cuda"), torch.full((1, n), 2.0, device="cuda"), torch.ones(n, device="cuda")
    for z, f in ((-1e30, 0.0), (float("-inf"), 0.0), (-200.0, 0.0), (200.0, 1.0), (float("inf"), 1.0), (0.0, 0.5)):
        gate = torch.full((1, n), z, device="cuda")
        s = Q.block_norm(x, w, r, w, gate=gate, eps=1e-30)[1]
        assert torch.allclose(s, r + f * x, atol=1e-6)
        d = Q.block_norm_backward(x, x, r, s, w, w, gate=gate, ds=r, eps=1e-30)
        assert all(torch.isfinite(t).all() for t in d if t is not None)
        assert torch.allclose(d.dgate, torch.full_like(x, 2.0 * f * (1 - f)), atol=1e-5)


def test_rows_of_zeros_and_no_rows(gpu):
    f = dict(device="cuda")
    w = torch.ones(40, **f)
    y, s = Q.block_norm(torch.zeros(3, 40, **f), w, torch.zeros(3, 40, **f), w)
    assert torch.equal(y, torch.zeros_like(y)) and torch.equal(s, y)
    e = torch.zeros(0, 40, **f)
    y, s = Q.block_norm(e, w, e, w, gate=e, residual_scale=w)
    assert y.shape == s.shape == (0, 40)
    g = Q.block_norm_backward(e, e, e, e, w, w, gate=e, residual_scale=w)
    zero = torch.zeros(40, **f)
    assert g.dx.shape == (0, 40) and all(torch.equal(t, zero) for t in (g.dpost, g.dpre, g.dresidual_scale))
    # rows whose squares are below fp32: without an eps such a row's norm cannot be told, which is refused; the least eps
    # stands far above what is lost
    t = torch.full((2, 40), 1e-25, **f)
    with pytest.raises(ValueError, match="eps"):
        Q.block_norm(t, w, torch.zeros(2, 40, **f), w, eps=0.0)
    y, s = Q.block_norm(t, w, torch.zeros(2, 40, **f), w, eps=1e-30)
    assert torch.allclose(s, torch.full_like(s, 1e-10), rtol=1e-5, atol=0.0)
    assert torch.allclose(y, torch.full_like(s, 1e-10 / (1e-20 + 1e-30) ** 0.5), rtol=1e-5, atol=0.0)


@pytest.mark.parametrize("ty", TYPES)
def test_results_over_operands(gpu, ty):
    d = Data(5)
    for rows, n in ((5, 7), (300, 512), (40, 2500)):
        x, r, z, w = d.normal(rows, n, type=ty).cuda(), d.normal(rows, n, type=ty).cuda(), d.normal(rows, n, type=ty).cuda(), \
            d.uniform(n).cuda()
        y, s = Q.block_norm(x, w, r, w, gate=z, residual_scale=w)
        for k in range(3):
            for m in range(3):
                if k == m:
                    continue
                ins = [t.clone() for t in (x, r, z)]
                got = Q.block_norm(ins[0], w, ins[1], w, gate=ins[2], residual_scale=w, out=ins[k], sum_out=ins[m])
                assert got[0] is ins[k] and got[1] is ins[m] and torch.equal(got[0], y) and torch.equal(got[1], s)
        flat = torch.cat([x.flatten(), x.flatten()[:3]])
        a, over = flat[:-3].view(rows, n), flat[3:].view(rows, n)
        assert torch.equal(Q.block_norm(a, w, r, w, gate=z, residual_scale=w, out=over)[0], y)
        with pytest.raises(ValueError, match="share memory"):
            Q.block_norm(x, w, r, w, out=x, sum_out=x)


def test_repeat_capture_and_streams(gpu):
    d = Data(7)
    B, T, n = 5, 300, 200
    x, r, z, w = d.normal(B, T, n).cuda(), d.normal(B, T, n).cuda(), d.normal(B, 1, n).cuda(), d.uniform(n).cuda()

    def both():
        y, s = Q.block_norm(x, w, r, w, gate=z, residual_scale=w)
        return (y, s, *Q.block_norm_backward(y, x, r, s, w, w, gate=z, residual_scale=w, ds=s))

    first = both()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = both()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = both()
    for k in range(4):
        x.copy_(d.normal(B, T, n))
        want = both()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, want))


def test_refusals(gpu):
    f = dict(device="cuda")
    x, w = torch.zeros(2, 3, 8, **f), torch.ones(8, **f)
    ok = dict(x=x, post_weight=w, residual=x, pre_weight=w)
    Q.block_norm(**ok)
    wide = torch.zeros(2, 8193, **f)
    for wrong in (dict(x=x.cpu()), dict(x=x.half()), dict(residual=x[:, :2]), dict(residual=None), dict(post_weight=w[:7]),
                  dict(pre_weight=w.bfloat16()), dict(gate=x.bfloat16()), dict(gate=x[:1, :1]), dict(gate=w), dict(gate=x[:, :2]),
                  dict(gate=x, gate_activation="silu"), dict(residual_scale=w[:7]), dict(eps=-1.0), dict(eps=0.0), dict(eps=float("nan")),
                  dict(out=x[:, :1].expand(2, 3, 8)), dict(sum_out=x.bfloat16()),
                  dict(x=wide, residual=wide, post_weight=wide[0], pre_weight=wide[0]), dict(x=w, residual=w)):
        with pytest.raises(ValueError):
            Q.block_norm(**{**ok, **wrong})
    with pytest.raises(ValueError):
        Q.block_norm_backward(x, x, None, x, w, w, residual_scale=w)  # the residual is needed
    with pytest.raises(ValueError):
        Q.block_norm_backward(x, x, None, x, w, w, ds=x.bfloat16())
