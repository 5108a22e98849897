"""How exact the gated delta rule's sums are where they cancel.  Needs a GPU.

Results in bfloat16 are rounded once, at the end: before that they are as
accurate as float32 ones.  The operands here make every product exact, and each
result the difference of two numbers below 2 that agree in their leading bits, so
that it is off by half a step of bfloat16 (2^-8 of itself) and at most four
roundings of float32 of the numbers it is the difference of (4 x 2^-24 x 2)."""
import pytest

torch = pytest.importorskip("torch")

from dgen_hip import sequence as Q  # noqa: E402
from test_gpu_sequence import F64, TYPES, Data  # noqa: E402

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
