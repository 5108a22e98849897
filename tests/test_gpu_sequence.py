"""Sequence operators (dgen_hip.sequence) against their definitions in 64 bits
on the CPU: norm with the residual's addition, causal convolution, selective
scan; forward, backward (against the definition's gradient by torch's
autograd in 64 bits, and against differences), single frames, streaming in
pieces, sequences of unequal length, views, and refusals.

Tolerances.  eps = 2^-24 is the relative rounding error of one fp32 operation.
A result formed by k operations in sequence, none of which cancels more than
its operands' magnitudes, is off by at most about k eps times the largest
magnitude on its way; the bounds below count those operations and take the
largest magnitude of the result's tensor times a small factor for the
cancellation in sums of signed terms.  bfloat16 results are rounded once more,
by at most 2^-8 of their own magnitude (eight significand bits).  Needs a GPU."""
import pytest
import torch

from dgen_hip import sequence as Q

pytestmark = pytest.mark.gpu

EPS32, EPS16 = 2.0 ** -24, 2.0 ** -8
F64 = torch.float64
TYPES = [torch.float32, torch.bfloat16]


def close(got, want, ops, what="", scale=None):
    """got (rounded to its type) against want in 64 bits, `ops` fp32
    operations deep; `scale`: the largest magnitude on the way, where the
    result's own terms cancel (else the result's largest)."""
    got, want = got.detach().cpu().to(F64), want.detach()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), what
    if not want.numel():
        return
    tol = ops * EPS32 * (want.abs().max().item() if scale is None else scale) + 1e-30
    bound = tol + (EPS16 * want.abs() * 1.01 if got_is_16(what) else 0.0)
    err = (got - want).abs()
    worst = (err - bound).max().item()
    assert worst <= 0, f"{what}: off by {err.max().item():.3e}, scale {want.abs().max().item():.3e}"


def got_is_16(what):
    return "bf16" in what


def name_of(t):
    return "bf16" if t == torch.bfloat16 else "fp32"


class Data:
    def __init__(self, seed):
        self.g = torch.Generator().manual_seed(seed)

    def normal(self, *shape, type=torch.float32, scale=1.0):
        """On the CPU in `type`."""
        return (torch.randn(*shape, generator=self.g, dtype=F64) * scale).to(type)

    def uniform(self, *shape, lo=0.0, hi=1.0):
        return (torch.rand(*shape, generator=self.g, dtype=F64) * (hi - lo) + lo).float()


def gpu_view(t, wide=0, lead=0):
    """On the GPU, as the columns [lead, lead + n) of a tensor `wide` columns
    wider, filled with NaN elsewhere."""
    if not wide:
        return t.cuda()
    full = torch.full((*t.shape[:-1], t.shape[-1] + wide), float("nan"), dtype=t.dtype, device="cuda")
    v = full[..., lead:lead + t.shape[-1]]
    v.copy_(t)
    return v


# -------------------------------------------------------------------- norm
def norm_ref(x, r, w, eps):
    s = x + r
    return s * torch.rsqrt(s.square().mean(-1, keepdim=True) + eps) * w, s


@pytest.mark.parametrize("rows,n", [(1, 1), (3, 7), (5, 64), (2, 129), (33, 130), (4, 512), (7, 1023), (3, 2049), (2, 5000),
                                    (2, 8193), (1, 32768)])
@pytest.mark.parametrize("xt,st", [(0, 0), (1, 0), (1, 1), (0, 1)])
def test_norm(gpu, rows, n, xt, st):
    xt, st = TYPES[xt], TYPES[st]
    d = Data(rows * 7 + n)
    x, r, w = d.normal(rows, n, type=xt), d.normal(rows, n, type=st, scale=2.0), d.uniform(n, lo=0.5, hi=1.5)
    y, s = Q.rms_norm(gpu_view(x, 3, 1), w.cuda(), residual=gpu_view(r, 5, 2), eps=1e-5)
    wy, ws = norm_ref(x.to(F64), r.to(F64), w.to(F64), 1e-5)
    # a sum of n squares in at most 40 additions a thread and 10 levels over threads
    close(y, wy, 64, f"y {name_of(xt)}")
    close(s, ws, 2, f"s {name_of(st)}")
    assert y.dtype == xt and s.dtype == st
    plain = Q.rms_norm(x.cuda(), w.cuda(), eps=1e-3)
    close(plain, norm_ref(x.to(F64), 0.0, w.to(F64), 1e-3)[0], 64, f"plain {name_of(xt)}")
    # the sum may replace the residual
    rr = r.cuda()
    y2, s2 = Q.rms_norm(x.cuda(), w.cuda(), residual=rr, eps=1e-5, sum_out=rr)
    assert s2.data_ptr() == rr.data_ptr() and torch.equal(s2, s) and torch.equal(y2, y)


@pytest.mark.parametrize("rows,n", [(1, 1), (3, 7), (5, 64), (6000, 33), (33, 130), (1030, 512), (70, 1023), (3, 2049), (20, 5000),
                                    (2, 8193), (1, 32768), (600, 8200)])
@pytest.mark.parametrize("xt,st", [(0, 0), (1, 0), (1, 1)])
def test_norm_backward(gpu, rows, n, xt, st):
    xt, st = TYPES[xt], TYPES[st]
    d = Data(rows * 5 + n)
    dy, s = d.normal(rows, n, type=xt), d.normal(rows, n, type=st, scale=2.0)
    ds, w = d.normal(rows, n, type=st), d.uniform(n, lo=0.5, hi=1.5)
    s64, w64 = s.to(F64).requires_grad_(), w.to(F64).requires_grad_()
    y = norm_ref(s64, 0.0, w64, 1e-5)[0]
    gs, gw = torch.autograd.grad((y * dy.to(F64)).sum(), (s64, w64))
    dx, dw = Q.rms_norm_backward(gpu_view(dy, 2, 1), gpu_view(s, 2, 1), w.cuda(), ds=gpu_view(ds, 1, 1), eps=1e-5)
    # dx = r (v - n mean(v n)): the two terms cancel (entirely, where n = 1)
    terms = (dy.to(F64) * w64.detach() * torch.rsqrt(s.to(F64).square().mean(-1, keepdim=True) + 1e-5)).abs().max().item()
    close(dx, gs + ds.to(F64), 100, f"dx {name_of(st)}", max(terms, ds.to(F64).abs().max().item()))
    # rows terms in a sum that grows as their square root
    close(dw, gw, 64 + 8 * rows ** 0.5, "dweight")
    dx2, _ = Q.rms_norm_backward(dy.cuda(), s.cuda(), w.cuda(), eps=1e-5)
    close(dx2, gs, 100, f"dx alone {name_of(st)}", terms)
    buf = ds.cuda()
    dx3, _ = Q.rms_norm_backward(dy.cuda(), s.cuda(), w.cuda(), ds=buf, eps=1e-5, out=buf)
    assert torch.equal(dx3, dx)


def test_norm_rows_of_zeros_and_empty(gpu):
    w = torch.ones(40, device="cuda")
    assert torch.equal(Q.rms_norm(torch.zeros(3, 40, device="cuda"), w), torch.zeros(3, 40, device="cuda"))
    assert Q.rms_norm(torch.zeros(0, 40, device="cuda"), w).shape == (0, 40)
    dx, dw = Q.rms_norm_backward(torch.zeros(0, 40, device="cuda"), torch.zeros(0, 40, device="cuda"), w)
    assert dx.shape == (0, 40) and torch.equal(dw, torch.zeros(40, device="cuda"))
    y = Q.rms_norm(torch.ones(2, 3, 40, device="cuda"), w, eps=0.0)
    assert y.shape == (2, 3, 40) and torch.allclose(y, torch.ones_like(y), atol=2e-7)


# -------------------------------------------------------------- convolution
def conv_ref(x, w, b, silu, state, lengths):
    """Definition in 64 bits: (y, state after)."""
    B, T, D = x.shape
    W = w.shape[1]
    ys, left = [], []
    for i in range(B):
        n = max(0, min(T, lengths[i]))
        row = torch.cat([state[i], x[i, :n]])
        u = sum((row[k:k + n] * w[:, k] for k in range(W)), torch.zeros(n, D, dtype=F64)) + b
        y = u * torch.sigmoid(u) if silu else u
        ys.append(torch.cat([y, torch.zeros(T - n, D, dtype=F64)]))
        left.append(row[n:])
    return torch.stack(ys), torch.stack(left)


def spoil(t, lengths):
    """NaN in the frames past each sequence's end."""
    t = t.clone()
    for i, n in enumerate(lengths):
        t[i, max(0, n):] = float("nan")
    return t


CONVS = [(1, 1, 1, 4), (2, 1, 33, 2), (3, 5, 6, 3), (2, 17, 64, 4), (4, 33, 130, 4), (1, 300, 7, 8), (2, 70, 257, 5), (1, 9, 4, 1)]


@pytest.mark.parametrize("B,T,D,W", CONVS)
@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("silu,ragged,state", [(True, True, True), (False, False, True), (True, False, False)])
def test_conv(gpu, B, T, D, W, ty, silu, ragged, state):
    d = Data(B * 31 + T + D)
    x, w, b = d.normal(B, T, D, type=ty), d.uniform(D, W, lo=-1, hi=1), d.uniform(D, lo=-1, hi=1)
    lengths = [[T, 0, T + 5, -3, max(0, T - 1), T // 2][(i + T) % 6] for i in range(B)] if ragged else [T] * B
    st = d.normal(B, W - 1, D, type=ty) if state and W > 1 else None
    st64 = torch.zeros(B, W - 1, D, dtype=F64) if st is None else st.to(F64)
    dev_len = torch.tensor(lengths, dtype=torch.int32, device="cuda") if ragged else None
    want, left = conv_ref(x.to(F64), w.to(F64), b.to(F64), silu, st64, lengths)
    args = dict(silu=silu, lengths=dev_len)
    xv = gpu_view(spoil(x, lengths), 3, 2)
    so = torch.full((B, W - 1, D), float("nan"), dtype=ty, device="cuda") if W > 1 else None
    y = Q.causal_conv(xv, w.cuda(), b.cuda(), state=None if st is None else st.cuda(), state_out=so, **args)
    # W products and sums, the activation's ten operations
    close(y, want, 4 * (W + 10), f"y {name_of(ty)}")
    if W > 1:
        assert torch.equal(so.cpu().to(F64), left)
    if st is not None:
        inplace = st.cuda()
        y2 = Q.causal_conv(xv, w.cuda(), b.cuda(), state=inplace, state_out=inplace, **args)
        assert torch.equal(y2, y) and torch.equal(inplace, so)
    # gradients
    x64, w64, b64 = (t.to(F64).requires_grad_() for t in (x, w, b))
    dy = d.normal(B, T, D, type=ty)
    out, _ = conv_ref(x64, w64, b64, silu, st64, lengths)
    gx, gw, gb = torch.autograd.grad((out * dy.to(F64)).sum(), (x64, w64, b64), allow_unused=True)
    dx, dw, db = Q.causal_conv_backward(gpu_view(spoil(dy, lengths), 1), xv, w.cuda(), b.cuda(),
                                        state=None if st is None else st.cuda(), **args)
    zero = torch.zeros(1, dtype=F64)
    close(dx, zero.expand(B, T, D) if gx is None else gx, 8 * (W + 16), f"dx {name_of(ty)}")
    close(dw, gw, 64 + 8 * (B * T) ** 0.5, "dweight")
    close(db, gb, 64 + 8 * (B * T) ** 0.5, "dbias")
    nodx, nodw, none = Q.causal_conv_backward(dy.cuda(), x.cuda(), w.cuda(), silu=silu)
    assert none is None and torch.isfinite(nodx).all() and torch.isfinite(nodw).all()


@pytest.mark.parametrize("ty", TYPES)
def test_conv_in_pieces_is_the_whole(gpu, ty):
    """Any split into calls gives the same samples: every output is formed in
    the same order from the same values."""
    d = Data(9)
    B, T, D, W = 3, 61, 70, 4
    x, w, b = d.normal(B, T, D, type=ty).cuda(), d.uniform(D, W, lo=-1, hi=1).cuda(), d.uniform(D).cuda()
    whole = Q.causal_conv(x, w, b)
    state = torch.zeros(B, W - 1, D, dtype=ty, device="cuda")
    got, t = [], 0
    for n in (1, 1, 2, 30, 3, 1, 23):
        got.append(Q.causal_conv(x[:, t:t + n], w, b, state=state, state_out=state))
        t += n
    assert t == T and torch.equal(torch.cat(got, 1), whole)


# --------------------------------------------------------------------- scan
def scan_ref(x, dt, A, Bm, Cm, D, z, bias, state, lengths):
    """Definition in 64 bits, frame by frame: (y, state after)."""
    n, T, ch = x.shape
    live = torch.tensor([[t < max(0, L) for t in range(T)] for L in lengths])
    step = torch.where(live[..., None], torch.nn.functional.softplus(dt + bias, threshold=1e9), torch.zeros(1, dtype=F64))
    h, ys = state, []
    for t in range(T):
        h = torch.exp(step[:, t, :, None] * A) * h + (step[:, t] * x[:, t])[..., None] * Bm[:, t, None, :]
        y = (h * Cm[:, t, None, :]).sum(-1) + D * x[:, t]
        g = z[:, t] * torch.sigmoid(z[:, t]) if z is not None else 1.0
        ys.append(torch.where(live[:, t, None], y * g, torch.zeros(1, dtype=F64)))
    return torch.stack(ys, 1), h


def scan_data(B, T, D, N, ty, ragged, state, full, seed=0):
    d = Data(B * 131 + T * 7 + D + N + seed)
    lengths = [[T, 0, T + 5, -3, max(0, T - 1), T // 2 + 1][(i + T) % 6] for i in range(B)] if ragged else [T] * B
    v = dict(x=d.normal(B, T, D, type=ty), dt=d.normal(B, T, D, type=ty, scale=0.7), B=d.normal(B, T, N, type=ty),
             C=d.normal(B, T, N, type=ty), A=-d.uniform(D, N, lo=0.01, hi=N))
    v["z"] = d.normal(B, T, D, type=ty) if full else None
    v["D"] = d.uniform(D, lo=0.5, hi=1.5) if full else None
    v["dt_bias"] = d.uniform(D, lo=-6.0, hi=-1.0) if full else None
    v["state"] = d.normal(B, D, N) if state else None
    return v, lengths, d


SCANS = [(1, 1, 1, 1), (3, 1, 70, 16), (2, 3, 5, 4), (2, 33, 64, 16), (3, 65, 65, 7), (2, 130, 20, 16), (1, 200, 130, 12),
         (1, 97, 17, 33), (2, 40, 9, 64), (1, 300, 3, 16), (6, 20, 33, 24)]


def scan_gpu(v, lengths, ragged, pad=0):
    g = {k: (None if t is None else t.cuda()) for k, t in v.items()}
    for k in ("x", "dt", "z", "B", "C"):
        if v[k] is not None:
            g[k] = gpu_view(spoil(v[k], lengths) if ragged else v[k], pad, pad // 2)
    g["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda") if ragged else None
    return g


def wide(v, grad=()):
    zeros = torch.zeros(v["A"].shape[0], dtype=F64)
    out = {k: None if t is None else t.to(F64) for k, t in v.items()}
    for k in ("D", "dt_bias"):
        out[k] = zeros if out[k] is None else out[k]
    if out["state"] is None:
        B, _, D = v["x"].shape
        out["state"] = torch.zeros(B, D, v["A"].shape[1], dtype=F64)
    for k in grad:
        if out[k] is not None:
            out[k] = out[k].clone().requires_grad_()
    return out


def ref_call(w, lengths):
    return scan_ref(w["x"], w["dt"], w["A"], w["B"], w["C"], w["D"], w["z"], w["dt_bias"], w["state"], lengths)


def scan_ops(T, N):
    """A state is T steps of four operations deep (its decays keep what came
    before from growing); sums over N states, the step's and gate's functions."""
    return 4 * T + 2 * N + 64


@pytest.mark.parametrize("B,T,D,N", SCANS)
@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("ragged,state,full", [(True, True, True), (False, False, True), (False, True, False)])
def test_scan(gpu, B, T, D, N, ty, ragged, state, full):
    v, lengths, _ = scan_data(B, T, D, N, ty, ragged, state, full)
    want, left = ref_call(wide(v), lengths)
    g = scan_gpu(v, lengths, ragged, pad=6)
    so = torch.full((B, D, N), float("nan"), device="cuda")
    y = Q.selective_scan(**g, state_out=so)
    close(y, want, scan_ops(T, N), f"y {name_of(ty)}")
    close(so, left, scan_ops(T, N), "state")
    if state:
        g["state"] = g["state"].clone()
        y2 = Q.selective_scan(**g, state_out=g["state"])
        assert torch.equal(y2, y) and torch.equal(g["state"], so)


@pytest.mark.parametrize("B,T,D,N", SCANS)
@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("ragged,state,full", [(True, True, True), (False, False, True), (False, True, False)])
def test_scan_backward(gpu, B, T, D, N, ty, ragged, state, full):
    v, lengths, d = scan_data(B, T, D, N, ty, ragged, state, full)
    dy = d.normal(B, T, D, type=ty)
    names = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")
    w = wide(v, names)
    out, _ = ref_call(w, lengths)
    live = [k for k in names if w[k] is not None]
    grads = dict(zip(live, torch.autograd.grad((out * dy.to(F64)).sum(), [w[k] for k in live], allow_unused=True)))
    g = scan_gpu(v, lengths, ragged, pad=6)
    got = Q.selective_scan_backward(gpu_view(spoil(dy, lengths) if ragged else dy, 2), **g)
    for k in names:
        t = getattr(got, "d" + k)
        if v[k] is None:
            assert t is None
            continue
        want = grads[k] if grads[k] is not None else torch.zeros(t.shape, dtype=F64)
        typed = name_of(ty) if k in ("x", "dt", "B", "C", "z") else ""
        # forward states and adjoint, then sums over channels (B, C) or frames
        ops = 4 * scan_ops(T, N) + (8 * (B * T) ** 0.5 if k in ("A", "D", "dt_bias") else 2 * D)
        close(t, want, ops, f"d{k} {typed}")


def test_scan_gradient_against_differences(gpu):
    """The gradient along a random direction of every input against central
    differences of the forward pass (fp32 on the GPU): the difference of two
    outputs of size 1 over 2e-2 is good to about 1e-5 of them, and the third
    derivative leaves 1e-4."""
    v, lengths, d = scan_data(2, 40, 33, 16, torch.float32, False, True, True, seed=3)
    dy = d.normal(2, 40, 33)
    g = scan_gpu(v, lengths, False)
    got = Q.selective_scan_backward(dy.cuda(), **g)
    for k in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias"):
        u = d.normal(*v[k].shape).cuda()
        u /= u.norm()
        e = 1e-2
        hi, lo = (Q.selective_scan(**{**g, k: (g[k] + s * e * u).contiguous()}).double() for s in (1, -1))
        num = ((hi - lo) * dy.cuda().double()).sum() / (2 * e)
        ana = (getattr(got, "d" + k).double() * u.double()).sum()
        assert abs(num - ana) <= 2e-3 * max(1.0, abs(ana.item())), (k, num.item(), ana.item())


@pytest.mark.parametrize("B,T,D,N", [(1, 4000, 10, 16), (2, 1537, 70, 8), (330, 40, 20, 16)])
def test_scan_long(gpu, B, T, D, N):
    """Time cut into chunks, and many sequences that are not."""
    v, lengths, d = scan_data(B, T, D, N, torch.float32, True, True, True)
    v["dt_bias"] = d.uniform(D, lo=-7.0, hi=-4.0)  # long memories
    want, left = ref_call(wide(v), lengths)
    g = scan_gpu(v, lengths, True)
    so = torch.empty(B, D, N, device="cuda")
    y = Q.selective_scan(**g, state_out=so)
    close(y, want, scan_ops(T, N), "y")
    close(so, left, scan_ops(T, N), "state")


def test_scan_backward_long(gpu):
    B, T, D, N = 2, 700, 12, 16
    v, lengths, d = scan_data(B, T, D, N, torch.float32, True, True, True)
    lengths = [700, 333]
    v["dt_bias"] = d.uniform(D, lo=-7.0, hi=-4.0)
    dy = d.normal(B, T, D)
    names = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")
    w = wide(v, names)
    grads = torch.autograd.grad((ref_call(w, lengths)[0] * dy.to(F64)).sum(), [w[k] for k in names])
    got = Q.selective_scan_backward(spoil(dy, lengths).cuda(), **scan_gpu(v, lengths, True))
    for k, want in zip(names, grads):
        close(getattr(got, "d" + k), want, 4 * scan_ops(T, N) + 8 * (B * T) ** 0.5, "d" + k)


@pytest.mark.parametrize("ty", TYPES)
def test_scan_in_pieces(gpu, ty):
    """A prompt, then single frames, carry the state: as the whole clip."""
    B, T, D, N = 3, 90, 40, 16
    v, lengths, _ = scan_data(B, T, D, N, ty, False, True, True)
    g = scan_gpu(v, lengths, False)
    g.pop("lengths")
    want, left = ref_call(wide(v), lengths)
    state, t, got = g["state"].clone(), 0, []
    for n in (70, 1, 1, 1, 5, 1, 11):
        part = {k: a[:, t:t + n] if k in ("x", "dt", "z", "B", "C") else a for k, a in g.items()}
        got.append(Q.selective_scan(**{**part, "state": state}, state_out=state))
        t += n
    assert t == T
    close(torch.cat(got, 1), want, scan_ops(T, N), f"y {name_of(ty)}")
    close(state, left, scan_ops(T, N), "state")


def test_scan_calls_repeat_bit_for_bit(gpu):
    """No sum depends on the order in which workgroups run."""
    v, lengths, d = scan_data(2, 300, 100, 16, torch.bfloat16, True, True, True)
    g, dy = scan_gpu(v, lengths, True), d.normal(2, 300, 100, type=torch.bfloat16).cuda()
    first, again = (Q.selective_scan_backward(dy, **g) for _ in range(2))
    for a, b in zip(first, again):
        assert torch.equal(a, b)
    assert torch.equal(Q.selective_scan(**g), Q.selective_scan(**g))


def test_other_streams(gpu):
    """Work goes to torch's current stream."""
    v, lengths, _ = scan_data(2, 100, 33, 16, torch.float32, False, False, True)
    g = scan_gpu(v, lengths, False)
    want = Q.selective_scan(**g)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        x = g["x"].clone()  # on the side stream
        got = Q.selective_scan(**{**g, "x": x})
    side.synchronize()
    assert torch.equal(got, want)


def test_refusals(gpu):
    f = dict(device="cuda")
    x, w = torch.zeros(2, 5, 8, **f), torch.zeros(8, 4, **f)
    with pytest.raises(ValueError):
        Q.rms_norm(torch.zeros(2, 8), torch.zeros(8))  # host tensors
    with pytest.raises(ValueError):
        Q.rms_norm(torch.zeros(2, 8, dtype=torch.float16, **f), torch.zeros(8, **f))
    with pytest.raises(ValueError):
        Q.rms_norm(torch.zeros(2, 8, **f), torch.zeros(7, **f))
    with pytest.raises(ValueError):
        Q.rms_norm(torch.zeros(2, 32769, **f), torch.zeros(32769, **f))
    with pytest.raises(ValueError):
        Q.rms_norm(torch.zeros(2, 8, **f), torch.zeros(8, **f), eps=-1.0)
    with pytest.raises(ValueError):
        Q.rms_norm(torch.zeros(8, 2, **f).t(), torch.zeros(8, **f))  # strided last axis
    with pytest.raises(ValueError):
        Q.rms_norm(torch.zeros(2, 8, **f), torch.zeros(8, **f), out=torch.zeros(1, 8, **f).expand(2, 8))
    with pytest.raises(ValueError):
        Q.causal_conv(x, torch.zeros(8, 9, **f))  # window
    with pytest.raises(ValueError):
        Q.causal_conv(x, w, state=torch.zeros(2, 4, 8, **f))
    with pytest.raises(ValueError):
        Q.causal_conv(x, w, lengths=torch.zeros(2, dtype=torch.int64, **f))
    with pytest.raises(ValueError):
        Q.causal_conv(x, w, out=torch.zeros(1, 5, 8, **f).expand(2, 5, 8))
    A, bc = torch.zeros(8, 4, **f), torch.zeros(2, 5, 4, **f)
    with pytest.raises(ValueError):
        Q.selective_scan(x, x, torch.zeros(8, 65, **f), torch.zeros(2, 5, 65, **f), torch.zeros(2, 5, 65, **f))
    with pytest.raises(ValueError):
        Q.selective_scan(x, x.bfloat16(), A, bc, bc)
    with pytest.raises(ValueError):
        Q.selective_scan(x, x, A, bc, bc[:, :4])
    with pytest.raises(ValueError):
        Q.selective_scan(x, x, A, bc, bc, state=torch.zeros(2, 8, 4, dtype=torch.bfloat16, **f))
    with pytest.raises(ValueError):
        Q.selective_scan(x[:, :0], x[:, :0], A, bc[:, :0], bc[:, :0])  # no frames
    assert Q.selective_scan(x[:0], x[:0], A, bc[:0], bc[:0]).shape == (0, 5, 8)
