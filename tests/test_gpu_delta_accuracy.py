"""How exact the gated delta rule's sums are where they cancel: results, and the
gradients of gates that forget.  Needs a GPU.

Results in bfloat16 are rounded once, at the end: before that they are as
accurate as float32 ones.  The operands of their tests make every product exact, and each
result the difference of two numbers below 2 that agree in their leading bits, so
that it is off by half a step of bfloat16 (2^-8 of itself) and at most four
roundings of float32 of the numbers it is the difference of (4 x 2^-24 x 2)."""
import pytest

torch = pytest.importorskip("torch")

from dgen_hip import sequence as Q  # noqa: E402
from test_gpu_delta_rule import INPUTS, data, on_gpu, ops_of  # noqa: E402
from test_gpu_sequence import EPS32, F64, TYPES, Data, spoil  # noqa: E402

pytestmark = pytest.mark.gpu

# (keys' channels, values): within a block of values, over two, and odd
WIDTHS = [(32, 32), (33, 20), (64, 48), (128, 33)]


def within(got, want, what):
    half = 2.0 ** -8 if got.dtype == torch.bfloat16 else 0.0
    err = (got.cpu().to(F64) - want).abs()
    assert (err <= half * want.abs() + 2.0 ** -21).all(), (what, (err / (half * want.abs() + 2.0 ** -21)).max().item())


def blank(T, H, K, V, ty):
    f = dict(device="cuda")
    return dict(q=torch.zeros(1, T, H, K, dtype=ty, **f), k=torch.zeros(1, T, H, K, dtype=ty, **f),
                v=torch.zeros(1, T, H, V, dtype=ty, **f), g=torch.zeros(1, T, H, **f), beta=torch.zeros(1, T, H, **f))


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("K,V", WIDTHS)
@pytest.mark.parametrize("T", [5, 20, 64, 100])
def test_what_a_query_reads_of_the_memory(gpu, ty, K, V, T):
    """Two rows of the memory that differ in their last bits, one less the
    other."""
    H = 2
    a, d = blank(T, H, K, V, ty), Data(K + T)
    state = torch.zeros(1, H, K, V)
    state[0, :, 0] = (d.uniform(H, V) * 0.99 + 1.0)
    less = torch.randint(1, 1 << 10, (H, V), generator=d.g).double() * 2.0 ** -23  # (exact in float32)
    state[0, :, 1] = (state[0, :, 0].double() - less).float()
    want = state[0, :, 0].double() - state[0, :, 1].double()
    a["q"][..., 0], a["q"][..., 1] = 1.0, -1.0
    y = Q.gated_delta_rule(**a, state=state.cuda(), scale=1.0, normalize=False)
    within(y, want[None, None].expand(1, T, H, V), "memory")


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("K,V", WIDTHS)
@pytest.mark.parametrize("T", [5, 20, 64, 100])
def test_what_a_query_reads_of_the_chunks_writes(gpu, ty, K, V, T):
    """Two frames write with keys at right angles and strengths that differ in
    their last bits; later frames read one less the other."""
    H = 2
    a, d = blank(T, H, K, V, ty), Data(K + T + 1)
    a["k"][0, 0, :, 0], a["k"][0, 1, :, 1] = 1.0, 1.0
    v = d.uniform(H, V, lo=0.5, hi=1.0).to(ty)
    a["v"][0, 0], a["v"][0, 1] = v.cuda(), v.cuda()
    one = d.uniform(H, lo=0.5, hi=0.99)
    two = (one.double() + torch.randint(1, 1 << 10, (H,), generator=d.g).double() * 2.0 ** -24).float()
    a["beta"][0, 0], a["beta"][0, 1] = one.cuda(), two.cuda()
    a["q"][0, 2:, :, 0], a["q"][0, 2:, :, 1] = -1.0, 1.0
    want = torch.zeros(1, T, H, V, dtype=F64)
    want[0, 2:] = ((two.double() - one.double())[:, None] * v.to(F64))[None]
    within(Q.gated_delta_rule(**a, scale=1.0, normalize=False), want, "writes")


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("K,V", WIDTHS)
@pytest.mark.parametrize("T", [5, 20, 64, 100])
def test_what_a_small_decay_leaves(gpu, ty, K, V, T):
    """Two equal writes, a decay of nearly 1 between them and a common one after
    them; later frames read one less the other."""
    H = 8
    a, d = blank(T, H, K, V, ty), Data(K + T + 2)
    a["k"][0, 0, :, 0], a["k"][0, 1, :, 1] = 1.0, 1.0
    a["v"][0, :2], a["beta"][0, :2] = 1.0, 1.0
    g, both = -torch.randint(1, 1 << 7, (H,), generator=d.g).float() * 2.0 ** -20, -d.uniform(H, lo=0.1, hi=0.6)
    a["g"][0, 1], a["g"][0, 2] = g.cuda(), both.cuda()
    a["q"][0, 2:, :, 0], a["q"][0, 2:, :, 1] = -1.0, 1.0
    want = torch.zeros(1, T, H, V, dtype=F64)
    want[0, 2:] = (torch.exp(both.double()) * -torch.expm1(g.double()))[None, :, None]
    within(Q.gated_delta_rule(**a, scale=1.0, normalize=False), want, "decays")

def gates_gradients(x, dy, s, lengths, scale):
    """Definition in 64 bits: the gradients of g, and the size of what each is
    the sum of, e^g |S| |D|, with the memory before the frame and the adjoint
    after its decay made of their terms' magnitudes."""
    q, k, v, g, beta = (x[n].to(F64) for n in INPUTS)
    B, T, H, V = v.shape
    share = H // q.shape[2]
    q, k = (t / torch.sqrt(t.square().sum(-1, keepdim=True) + 1e-6) for t in (q, k))
    q, k, dy = q.repeat_interleave(share, 2) * scale, k.repeat_interleave(share, 2), dy.to(F64)
    live = (torch.arange(T) < torch.tensor(lengths)[:, None]).to(F64)[..., None]
    decay, beta, dy = torch.where(live > 0, torch.exp(g), 1.0), beta * live, dy * live[..., None]
    S = torch.zeros(B, H, k.shape[-1], V, dtype=F64) if s is None else s.to(F64)
    size, kept = S.abs(), []
    for t in range(T):
        kept.append((S, size))
        S, size = decay[:, t, :, None, None] * S, decay[:, t, :, None, None] * size
        u = beta[:, t, :, None] * (v[:, t] - (k[:, t, :, None] @ S)[:, :, 0])
        S, size = S + k[:, t, :, :, None] * u[:, :, None], size + (k[:, t, :, :, None] * u[:, :, None]).abs()
    dg, most = torch.zeros(B, T, H, dtype=F64), torch.zeros(B, T, H, dtype=F64)
    D, dsize = torch.zeros_like(S), torch.zeros_like(S)
    for t in reversed(range(T)):
        reads = q[:, t, :, :, None] * dy[:, t, :, None]
        D, dsize = D + reads, dsize + reads.abs()
        dv = beta[:, t, :, None] * (k[:, t, :, None] @ D)[:, :, 0]
        back = k[:, t, :, :, None] * dv[:, :, None]
        D, dsize = D - back, dsize + back.abs()
        D, dsize = decay[:, t, :, None, None] * D, decay[:, t, :, None, None] * dsize
        dg[:, t] = (kept[t][0] * D).sum((-1, -2))
        most[:, t] = kept[t][1].square().sum((-1, -2)).sqrt() * dsize.square().sum((-1, -2)).sqrt()
    return dg * live, most * live


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("B,T,G,H,K,V", [(2, 40, 1, 2, 16, 12), (1, 64, 1, 1, 64, 64), (2, 130, 2, 4, 33, 20), (1, 200, 1, 2, 128, 40),
                                         (1, 513, 1, 3, 24, 33)])
@pytest.mark.parametrize("low", [-0.01, -5.0, -10.0, -16.0, -60.0, "any"])
def test_gradients_of_gates_that_forget(gpu, ty, B, T, G, H, K, V, low):
    """As exact as what the gate lets through, however little that is: no more
    is lost than 4 ops_of + 4 V roundings of its terms."""
    x, _, s, d = data(B, T, G, H, K, V, ty)
    x["g"] = d.uniform(B, T, H, lo=-24.0, hi=0.0) if low == "any" else torch.full((B, T, H), low)
    lengths, dy = [T, T - 3][:B], d.normal(B, T, H, V, type=ty)
    want, size = gates_gradients(x, dy, s, lengths, K ** -0.5)
    got = Q.gated_delta_rule_backward(spoil(dy, lengths).cuda(), **on_gpu(x, lengths, s, True)).dg.cpu().to(F64)
    tol = (4 * ops_of(T, K) + 4 * V) * EPS32
    err = (got - want).abs()
    assert (err <= tol * size).all(), (err / (tol * size + 1e-300)).max().item()


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("low", [-104.0, -128.0, -1e30, -float("inf")])
@pytest.mark.parametrize("T", [1, 50, 140, 600])
def test_gates_that_let_nothing_through(gpu, ty, low, T):
    """No gradient reaches them, not even a rounding's."""
    B, G, H, K, V = 2, 1, 2, 24, 20
    x, _, s, d = data(B, T, G, H, K, V, ty)
    shut = torch.rand(B, T, H, generator=d.g) < 0.3
    shut[:, T // 2] = True
    x["g"] = torch.where(shut, low, x["g"])
    r = Q.gated_delta_rule_backward(d.normal(B, T, H, V, type=ty).cuda(), **on_gpu(x, s=s))
    assert (r.dg[shut.cuda()] == 0).all() and all(torch.isfinite(t).all() for t in r)
