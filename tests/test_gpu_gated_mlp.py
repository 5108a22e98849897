"""The gated feed-forward block (dgen_hip.sequence.gated_mlp) against its
definition in 64 bits: forward for single rows to many, backward against
autograd in 64 bits and against differences, odd sizes, views, refusals.

Tolerances.  A sum of K products accumulated in fp32 is off by at most about
K 2^-24 times the sum of the products' magnitudes (the split products of fp32
operands are exact to 2^-24 of theirs too), and passes on with the derivative
of what follows; a bfloat16 result is rounded by 2^-8 of itself.  The backward
pass stores dg and du in the operands' type: in bfloat16 each term of the sums
over them is off by another 2^-8 of itself.  Needs a GPU."""
import math

import pytest
import torch

from dgen_hip import sequence as Q

pytestmark = pytest.mark.gpu

EPS32, EPS16 = 2.0 ** -24, 2.0 ** -8
F64 = torch.float64
TYPES = [torch.float32, torch.bfloat16]


def act64(name, v):
    """Activation and derivative."""
    if name == "silu":
        p = torch.sigmoid(v)
        return v * p, p * (1 + v * (1 - p))
    t = torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
    return (0.5 * v * (1 + t),
            0.5 * (1 + t) + 0.5 * v * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * v * v))


def within(got, want, bound, what):
    err = (got.detach().cpu().to(F64) - want.cpu()).abs()
    assert torch.isfinite(err).all(), what
    bad = (err - bound.cpu()).max().item() if err.numel() else 0
    assert bad <= 0, f"{what}: off by {err.max().item():.3e}"


def make(rows, width, hidden, ty, seed=0):
    g = torch.Generator().manual_seed(seed + rows * 7 + width * 3 + hidden)

    def normal(*s, scale=1.0):
        return (torch.randn(*s, generator=g, dtype=F64) * scale).to(ty)

    return (normal(rows, width), normal(width, hidden, scale=width ** -0.5), normal(width, hidden, scale=width ** -0.5),
            normal(rows, hidden))


def view(t, wide=3, lead=1):
    full = torch.full((t.shape[0], t.shape[1] + wide), float("nan"), dtype=t.dtype, device="cuda")
    full[:, lead:lead + t.shape[1]] = t.cuda()
    return full[:, lead:lead + t.shape[1]]


SIZES = [(1, 1, 1), (1, 33, 65), (3, 512, 130), (8, 70, 64), (9, 100, 31), (16, 1030, 200), (17, 40, 7), (64, 64, 64),
         (65, 129, 127), (130, 200, 333), (300, 65, 1000), (1000, 96, 520)]


def check_forward(rows, width, hidden, ty, act, out=None):
    x, wg, wu, _ = make(rows, width, hidden, ty)
    h = Q.gated_mlp(view(x), view(wg, 5, 4), view(wu, 2, 1), activation=act)
    a, b, c = (t.to(F64) for t in (x, wg, wu))
    g, u = a @ b, a @ c
    f, df = act64(act, g)
    mag_g, mag_u = a.abs() @ b.abs(), a.abs() @ c.abs()
    k = (width + 32) * EPS32
    bound = k * (mag_g * u.abs() * 1.2 + f.abs() * mag_u + (f * u).abs()) + 1e-30
    if ty == torch.bfloat16:
        bound = bound + EPS16 * 1.01 * (f * u).abs()
    within(h, f * u, bound, "h")
    return x, wg, wu


@pytest.mark.parametrize("rows,width,hidden", SIZES)
@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_forward(gpu, rows, width, hidden, ty, act):
    check_forward(rows, width, hidden, ty, act)


@pytest.mark.parametrize("rows,width,hidden", [(2500, 72, 1700), (4100, 64, 1024), (300, 40, 8200), (9, 40, 16500)])
@pytest.mark.parametrize("ty", TYPES)
def test_forward_large(gpu, rows, width, hidden, ty):
    check_forward(rows, width, hidden, ty, "silu")


def check_backward(rows, width, hidden, ty, act):
    x, wg, wu, dh = make(rows, width, hidden, ty, 5)
    dx, dwg, dwu = Q.gated_mlp_backward(view(dh, 1), view(x), view(wg, 5, 4), view(wu, 2, 1), activation=act)
    a, b, c, d = (t.to(F64) for t in (x, wg, wu, dh))
    g, u = a @ b, a @ c
    f, df = act64(act, g)
    dg, du = d * u * df, d * f
    k1 = (width + 32) * EPS32
    mag_g, mag_u = a.abs() @ b.abs(), a.abs() @ c.abs()
    # errors of dg and du: of the projections (second derivatives are below
    # 1.2), and their own rounding
    own = EPS16 * 1.01 if ty == torch.bfloat16 else EPS32
    eg = k1 * d.abs() * (mag_u * df.abs() + u.abs() * mag_g * 1.2) + (own + 16 * EPS32) * dg.abs()
    eu = k1 * d.abs() * mag_g * 1.2 + (own + 16 * EPS32) * du.abs()

    def bound(e1, m1, e2, m2, terms, want):
        out = e1 @ m1.abs() + (terms + 32) * EPS32 * e2 + 1e-30
        return out + (EPS16 * 1.01 * want.abs() if ty == torch.bfloat16 else EPS32 * want.abs())

    want = dg @ b.T + du @ c.T
    within(dx, want, bound(eg, b.T, dg.abs() @ b.T.abs() + du.abs() @ c.T.abs(), None, 2 * hidden, want)
           + eu @ c.T.abs(), "dx")
    for got, dd, ee, what in ((dwg, dg, eg, "dw_gate"), (dwu, du, eu, "dw_up")):
        want = a.T @ dd
        within(got, want, bound(a.T.abs(), ee, a.T.abs() @ dd.abs(), None, rows, want), what)
    return x, wg, wu, dh, dx, dwg, dwu


@pytest.mark.parametrize("rows,width,hidden", SIZES)
@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_backward(gpu, rows, width, hidden, ty, act):
    check_backward(rows, width, hidden, ty, act)


@pytest.mark.parametrize("rows,width,hidden", [(2500, 520, 900), (3001, 1100, 300), (2085, 512, 992), (2100, 33, 1801),
                                               (8300, 70, 450), (300, 40, 8200)])
@pytest.mark.parametrize("ty", TYPES)
def test_backward_large(gpu, rows, width, hidden, ty):
    """Large tiles and row ranges; repeated calls give the same bits."""
    x, wg, wu, dh, *first = check_backward(rows, width, hidden, ty, "silu")
    again = Q.gated_mlp_backward(dh.cuda(), x.cuda(), wg.cuda(), wu.cuda())
    once = Q.gated_mlp_backward(dh.cuda(), x.cuda(), wg.cuda(), wu.cuda())
    for a, b, c in zip(first, again, once):
        assert torch.equal(a, b) and torch.equal(b, c)


@pytest.mark.parametrize("rows,width,hidden", [(4096, 64, 1024), (2100, 96, 1920), (9000, 256, 256)])
def test_aligned_operands(gpu, rows, width, hidden):
    """bfloat16 tensors that start at 16 bytes with sizes in multiples of 32,
    as training batches have them, and a number of rows that has not."""
    ty = torch.bfloat16
    x, wg, wu, dh = make(rows, width, hidden, ty, 5)
    h = Q.gated_mlp(x.cuda(), wg.cuda(), wu.cuda())
    viewed = Q.gated_mlp(view(x), view(wg), view(wu))  # the same by unaligned loads
    a, b, c = (t.to(F64) for t in (x, wg, wu))
    f, _ = act64("silu", a @ b)
    want, mag = f * (a @ c), (a.abs() @ b.abs()) * (a @ c).abs() * 1.2 + f.abs() * (a.abs() @ c.abs())
    bound = (width + 32) * EPS32 * mag + EPS16 * 1.01 * want.abs() + 1e-30
    within(h, want, bound, "h")
    within(viewed, want, bound, "h of views")
    got = Q.gated_mlp_backward(dh.cuda(), x.cuda(), wg.cuda(), wu.cuda())
    ref = Q.gated_mlp_backward(view(dh), view(x), view(wg), view(wu))
    for p, q in zip(got, ref):
        # both are within the bound of check_backward; between them, rounding
        scale = q.double().abs().max().item()
        assert (p.double() - q.double()).abs().max().item() <= 2 * EPS16 * scale


def test_gradient_against_differences(gpu):
    """Along a random direction of every input, central differences of the
    fp32 forward over 2e-2: the sums' rounding leaves about 1e-4 of the
    derivative, the third derivative less."""
    x, wg, wu, dh = (t.cuda() for t in make(40, 50, 60, torch.float32, 2))
    grads = Q.gated_mlp_backward(dh, x, wg, wu, activation="gelu")
    g = torch.Generator().manual_seed(1)
    for i, grad in enumerate(grads):
        u = torch.randn(grad.shape, generator=g).cuda()
        u /= u.norm()
        ins = [x, wg, wu]
        vals = []
        for s in (1e-2, -1e-2):
            moved = list(ins)
            moved[i] = ins[i] + s * u
            vals.append((Q.gated_mlp(*moved, activation="gelu").double() * dh.double()).sum())
        num, ana = (vals[0] - vals[1]) / 2e-2, (grad.double() * u.double()).sum()
        assert abs(num - ana) <= 2e-3 * max(1.0, abs(ana.item())), (i, num.item(), ana.item())


def test_large_arguments_of_the_activations(gpu):
    """Far out, SiLU and GELU are 0 or the argument itself, without NaN."""
    for act in ("silu", "gelu"):
        x = torch.tensor([[-1e4], [-100.0], [-30.0], [0.0], [30.0], [100.0], [1e4]], device="cuda").repeat(3, 1)
        one = torch.ones(1, 5, device="cuda")
        h = Q.gated_mlp(x, one, one, activation=act)
        want = torch.where(x > 0, x * x, torch.zeros_like(x)).expand(-1, 5)
        assert torch.allclose(h, want, rtol=1e-6, atol=1e-8)
        dx, dg, du = Q.gated_mlp_backward(torch.ones_like(h), x, one, one, activation=act)
        assert torch.isfinite(dx).all() and torch.isfinite(dg).all() and torch.isfinite(du).all()


def test_no_rows_and_leading_axes(gpu):
    w = torch.ones(6, 9, device="cuda")
    assert Q.gated_mlp(torch.zeros(0, 6, device="cuda"), w, w).shape == (0, 9)
    dx, dg, du = Q.gated_mlp_backward(torch.zeros(0, 9, device="cuda"), torch.zeros(0, 6, device="cuda"), w, w)
    assert dx.shape == (0, 6) and not dg.any() and not du.any()
    x = torch.randn(2, 3, 6, device="cuda")
    assert torch.equal(Q.gated_mlp(x, w, w).view(6, 9), Q.gated_mlp(x.view(6, 6), w, w))


def test_refusals(gpu):
    x, w = torch.zeros(4, 6, device="cuda"), torch.zeros(6, 9, device="cuda")
    for bad in (lambda: Q.gated_mlp(x, w, w, activation="relu"), lambda: Q.gated_mlp(x, w, w[:, :8]),
                lambda: Q.gated_mlp(x, w[:5], w[:5]), lambda: Q.gated_mlp(x.bfloat16(), w, w),
                lambda: Q.gated_mlp(x, w.t().contiguous().t(), w), lambda: Q.gated_mlp(x.cpu(), w.cpu(), w.cpu()),
                lambda: Q.gated_mlp(x, w, w, out=torch.zeros(1, 9, device="cuda").expand(4, 9)),
                lambda: Q.gated_mlp_backward(x, x, w, w)):
        with pytest.raises(ValueError):
            bad()
