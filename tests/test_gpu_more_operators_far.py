"""The delta rule, the norms around a block and the optimiser's step at their
largest: values and heads as many as they take, tensors and scratch past 2^31
elements.  Needs a GPU (and up to 60 GB of its memory)."""
import pytest

torch = pytest.importorskip("torch")

from dgen_hip import optim  # noqa: E402
from dgen_hip import sequence as Q  # noqa: E402
from test_gpu_delta_rule import INPUTS, data, on_gpu, ops_of, rule, wide  # noqa: E402
from test_gpu_sequence import F64, TYPES, Data, close, name_of, spoil  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def tidy():
    yield
    torch.cuda.empty_cache()


# as many values as there may be, or nearly; many heads; many heads that share a key; many sequences
@pytest.mark.parametrize("B,T,G,H,K,V", [(1, 70, 1, 1, 128, 1024), (1, 9, 1, 2, 128, 1000), (1, 130, 1, 1, 40, 999), (1, 20, 300, 600, 8, 4),
                                         (2, 70, 1, 48, 16, 8), (3000, 17, 1, 1, 8, 4), (2000, 3, 1, 2, 8, 4)])
@pytest.mark.parametrize("ty", TYPES)
def test_delta_rule_of_many(gpu, B, T, G, H, K, V, ty):
    """Tolerances are test_gpu_delta_rule's; of many sequences the first, one
    within and the last are looked at."""
    x, lengths, s, d = data(B, T, G, H, K, V, ty, True, True)
    a, dy = on_gpu(x, lengths, s, True), d.normal(B, T, H, V, type=ty)
    after = torch.full((B, H, K, V), float("nan"), device="cuda")
    y = Q.gated_delta_rule(**a, state_out=after)
    got = Q.gated_delta_rule_backward(spoil(dy, lengths).cuda(), **a)
    for b in sorted({0, B // 2, B - 1}):
        one = {k: v[b:b + 1] for k, v in x.items()}
        w = wide(one, True)
        out, left = rule(**w, scale=K ** -0.5, state=s[b:b + 1].to(F64), lengths=lengths[b:b + 1])
        big = max(out.abs().max().item(), left.abs().max().item(), 1.0)
        close(y[b:b + 1], out.detach(), ops_of(T, K, ty), f"y {name_of(ty)}", big)
        close(after[b:b + 1], left.detach(), ops_of(T, K), "state", max(big, 4.0))
        none = sum(0.0 * t.sum() for t in w.values())
        want = torch.autograd.grad((out * dy[b:b + 1].to(F64)).sum() + none, [w[k] for k in INPUTS])
        share = (H // G) ** 0.5  # (a shared key's gradient is a sum over its heads)
        for k, t, r in zip(INPUTS, got, want):
            half = ty if k in "qkv" else torch.float32
            short = 1.0 if k not in "qk" else share / (one[k].to(F64).norm(dim=-1).min().item() + 1e-3)
            most = max(r.abs().max().item(), V ** 0.5 * (1.0 if k in ("v", "beta") else max(1.0, short)))
            close(t[b:b + 1], r, 4 * ops_of(T, K, half) + 4 * V, f"d{k} {name_of(half)}", most)


def test_delta_rule_with_scratch_past_32_bits(gpu):
    """Forty sequences that are one: each gives the same, bit for bit."""
    B, T, H, K, V, ty = 40, 8192, 8, 128, 128, torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(1)

    def normal(*shape, type=ty):
        return torch.randn(*shape, generator=g, device="cuda").to(type).expand(B, *shape[1:])

    a = dict(q=normal(1, T, H, K), k=normal(1, T, H, K), v=normal(1, T, H, V), g=-normal(1, T, H, type=torch.float32).abs() * 0.1,
             beta=torch.sigmoid(normal(1, T, H, type=torch.float32)))
    dy, after = normal(1, T, H, V), torch.empty(B, H, K, V, device="cuda")
    y = Q.gated_delta_rule(**a, state_out=after)
    r = Q.gated_delta_rule_backward(dy, **a)
    for t in (y, after, *r):
        assert torch.isfinite(t[0]).all() and t[0].any()
        for b in range(1, B):
            assert torch.equal(t[b], t[0]), b


@pytest.mark.parametrize("gates", ["rows", "one"])
def test_block_norm_past_32_bits(gpu, gates):
    """The rows at the ends of 2.4e9 elements are those of a call of their own."""
    rows, n, ty = 290_000, 8192, torch.bfloat16
    assert rows * n > 1 << 31
    d = Data(2)
    few = 64  # (rows that differ, at both ends)
    parts = [d.normal(2 * few, n, type=ty).cuda() for _ in range(5)]

    def spread(t):
        full = torch.zeros(rows, n, dtype=ty, device="cuda")
        full[:few], full[-few:] = t[:few], t[few:]
        return full

    x, r, z, dy, ds = (spread(t) for t in parts)
    w, u, scale = (d.uniform(n, lo=0.5, hi=1.5).cuda() for _ in range(3))
    gate = z if gates == "rows" else parts[2][:1]
    small = parts[2] if gates == "rows" else parts[2][:1]
    ends = lambda t: torch.cat([t[:few], t[-few:]])  # noqa: E731
    y, s = Q.block_norm(x, w, r, u, gate=gate, residual_scale=scale)
    y2, s2 = Q.block_norm(parts[0], w, parts[1], u, gate=small, residual_scale=scale)
    assert torch.equal(ends(y), y2) and torch.equal(ends(s), s2)
    got = Q.block_norm_backward(dy, x, r, s, w, u, gate=gate, residual_scale=scale, ds=ds)
    want = Q.block_norm_backward(parts[3], parts[0], parts[1], s2, w, u, gate=small, residual_scale=scale, ds=parts[4])
    assert torch.equal(ends(got.dx), want.dx) and torch.equal(ends(got.dresidual), want.dresidual)
    if gates == "rows":
        assert torch.equal(ends(got.dgate), want.dgate)
    # sums over rows, all but these of zeros: 128 terms each, in another order (2^-24 each, of the largest sum)
    for one, two in ((got.dpost, want.dpost), (got.dpre, want.dpre), (got.dresidual_scale, want.dresidual_scale)):
        assert (one - two).abs().max() <= 256 * 2.0 ** -24 * 16 * two.abs().max()


def test_adamw_past_32_bits(gpu):
    n = (1 << 31) + 12_345
    d = Data(3)
    few = 5000
    p0, m0, g0 = d.normal(2 * few, scale=0.1).cuda(), d.normal(2 * few, scale=1e-3).cuda(), d.normal(2 * few, scale=1e-2).bfloat16().cuda()
    v0 = d.uniform(2 * few, hi=1e-4).cuda()

    def spread(t):
        full = torch.zeros(n, dtype=t.dtype, device="cuda")
        full[:few], full[-few:] = t[:few], t[few:]
        return full

    p, m, v, g = (spread(t) for t in (p0, m0, v0, g0))
    copy, copy0 = torch.empty(n, dtype=torch.bfloat16, device="cuda"), torch.empty(2 * few, dtype=torch.bfloat16, device="cuda")
    norm = optim.adamw([p], [g], [m], [v], 3, max_norm=0.5, copies=[copy])
    norm0 = optim.adamw([p0], [g0], [m0], [v0], 3, max_norm=0.5, copies=[copy0])
    assert abs(norm.item() - norm0.item()) <= 4 * 2.0 ** -24 * norm0.item()
    for one, two in ((p, p0), (m, m0), (v, v0), (copy, copy0)):
        ends = torch.cat([one[:few], one[-few:]]).double()
        # (the norms are the same to the last bits, and with them the factor and what it scales: a few roundings)
        step = 2.0 ** -7 if one is copy else 16 * 2.0 ** -24
        assert ((ends - two.double()).abs() <= step * two.double().abs() + 1e-8 * (one is p)).all()
