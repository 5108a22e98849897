"""The delta rule, the norms around a block and the optimiser's step where they
can go wrong: values that are not finite, operands far apart in memory, the
smallest scales, gates of no rows, parameters that require gradients, two graphs
captured of one program, other threads' scratch.  Needs a GPU."""
import warnings

import pytest

torch = pytest.importorskip("torch")

from dgen_hip import optim  # noqa: E402
from dgen_hip import sequence as Q  # noqa: E402
from test_gpu_delta_rule import INPUTS, data, on_gpu, rule, wide  # noqa: E402
from test_gpu_sequence import F64, TYPES, Data, close  # noqa: E402

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("T,at", [(9, 4), (200, 100), (2300, 1500)])
@pytest.mark.parametrize("bad", [NAN, INF])
def test_what_a_value_that_is_not_finite_spoils(gpu, ty, T, at, bad):
    """Other sequences, heads and values, and the frames of the chunks (of 64)
    before, are what they were, bit for bit."""
    B, H, K, V = 2, 2, 24, 20
    x, _, s, d = data(B, T, H, H, K, V, ty)
    a, dy = on_gpu(x, s=s), d.normal(B, T, H, V, type=ty).cuda()
    y, r = Q.gated_delta_rule(**a), Q.gated_delta_rule_backward(dy, **a)
    b = {k: t.clone() for k, t in a.items()}
    b["v"][1, at, 1, 3] = bad
    z, q = Q.gated_delta_rule(**b), Q.gated_delta_rule_backward(dy, **b)
    before = at if T <= 16 else at // 64 * 64
    same = torch.ones(B, T, H, V, dtype=torch.bool, device="cuda")
    same[1, before:, 1, 3] = False
    assert torch.equal(z[same], y[same]) and not torch.isfinite(z[1, at:, 1, 3]).all()
    for one, two in zip(r, q):
        assert torch.equal(one[0], two[0]) and torch.equal(one[1, :, 0], two[1, :, 0])
    b = {k: t.clone() for k, t in a.items()}
    b["k"][0, at, 0, 5] = bad
    z = Q.gated_delta_rule(**b)
    same[:] = True
    same[0, before:, 0] = False
    assert torch.equal(z[same], y[same]) and not torch.isfinite(z[0, at:, 0]).all()


@pytest.mark.parametrize("T", [12, 130])
def test_operands_far_apart(gpu, T):
    """Sequences more than 2^31 elements apart, and frames 2^23: bit for bit as
    side by side."""
    B, H, K, V, ty = 2, 2, 16, 16, torch.bfloat16
    x, _, s, d = data(B, T, H, H, K, V, ty)
    a, dy = on_gpu(x, s=s), d.normal(B, T, H, V, type=ty).cuda()
    y, r = Q.gated_delta_rule(**a), Q.gated_delta_rule_backward(dy, **a)
    step = 1 << 23
    far = torch.zeros(max((1 << 31) + 4096, T * step) + T * step + 4096, dtype=ty, device="cuda")
    for n, strides in ((0, ((1 << 31) + 64, H * V, V, 1)), (1, (H * V, step, V, 1))):
        v = far.as_strided((B, T, H, V), strides)
        v.copy_(a["v"])
        assert torch.equal(Q.gated_delta_rule(**{**a, "v": v}), y)
        for one, two in zip(r, Q.gated_delta_rule_backward(dy, **{**a, "v": v})):
            assert torch.equal(one, two)
        g = far.as_strided((B, T, H, V), strides)
        g.copy_(dy)
        for one, two in zip(r, Q.gated_delta_rule_backward(g, **a)):
            assert torch.equal(one, two)
        assert torch.equal(Q.gated_delta_rule(**a, out=v), y) and torch.equal(v, y)
    with pytest.raises(ValueError, match="2\\^23"):
        Q.gated_delta_rule(**{**a, "v": far.as_strided((B, T, H, V), (H * V, step + 1, V, 1))})


@pytest.mark.parametrize("scale", [1e-41, 1e-30, -0.5, 1e20])
def test_scales(gpu, scale):
    """A scale passes through: results are the scale's times those of 1, as far
    as fp32 holds them, and the gradients of keys and values alike."""
    B, T, H, K, V = 1, 70, 2, 16, 8
    x, _, s, d = data(B, T, H, H, K, V, torch.float32)
    a, dy = on_gpu(x, s=s), d.normal(B, T, H, V).cuda()
    one, r = Q.gated_delta_rule(**a, scale=1.0), Q.gated_delta_rule_backward(dy, **a, scale=1.0)
    for got, want in zip((Q.gated_delta_rule(**a, scale=scale), *Q.gated_delta_rule_backward(dy, **a, scale=scale)), (one, *r)):
        want = want.double() * scale
        # (2^-126: numbers below that may be taken for 0)
        assert ((got.double() - want).abs() <= 1e-4 * want.abs().max() + 300 * 2.0 ** -126).all()


def test_a_memory_of_large_numbers(gpu):
    """The products' parts keep what fp32 keeps, whatever the size."""
    B, T, H, K, V = 1, 130, 1, 32, 16
    x, _, s, _ = data(B, T, H, H, K, V, torch.bfloat16)
    a = on_gpu(x, s=s)
    y = Q.gated_delta_rule(**a).double()
    for f in (2.0 ** 60, 2.0 ** -60):
        b = {**a, "v": (a["v"].float() * f).bfloat16(), "state": a["state"] * f}
        assert torch.equal(Q.gated_delta_rule(**b).double() / f, y)


def test_gates_of_no_rows(gpu):
    f = dict(device="cuda")
    w = torch.ones(8, **f)
    x, gate = torch.zeros(3, 0, 8, **f), torch.ones(3, 1, 8, **f)
    y, s = Q.block_norm(x, w, x, w, gate=gate)
    assert y.shape == s.shape == (3, 0, 8)
    g = Q.block_norm_backward(x, x, x, s, w, w, gate=gate)
    assert torch.equal(g.dgate, torch.zeros_like(gate)) and torch.equal(g.dpre, torch.zeros_like(w))


def test_a_gate_for_all_rows(gpu):
    """One gate of a matrix's rows, as the same one for each of them."""
    d = Data(3)
    x, r, w, z = d.normal(700, 24).cuda(), d.normal(700, 24).cuda(), d.uniform(24).cuda(), d.normal(1, 24).cuda()
    y, s = Q.block_norm(x, w, r, w, gate=z)
    each = z.expand(700, 24).contiguous()
    y2, s2 = Q.block_norm(x, w, r, w, gate=each)
    assert torch.equal(y, y2) and torch.equal(s, s2)
    one, many = (Q.block_norm_backward(y, x, r, s, w, w, gate=g) for g in (z, each))
    assert one.dgate.shape == (1, 24) and torch.allclose(one.dgate, many.dgate.sum(0, keepdim=True), rtol=1e-4, atol=1e-4)
    assert torch.equal(one.dx, many.dx)


def test_norms_of_values_that_are_not_finite(gpu):
    """A row that is not finite spoils itself, and the sums over rows."""
    d = Data(4)
    x, r, w = d.normal(9, 40).cuda(), d.normal(9, 40).cuda(), d.uniform(40).cuda()
    y, s = Q.block_norm(x, w, r, w)
    for bad in (NAN, INF):
        b = x.clone()
        b[4, 7] = bad
        z, t = Q.block_norm(b, w, r, w)
        rest = torch.arange(9, device="cuda") != 4
        assert torch.equal(z[rest], y[rest]) and torch.equal(t[rest], s[rest]) and not torch.isfinite(t[4]).all()
        g, h = Q.block_norm_backward(y, b, r, s, w, w), Q.block_norm_backward(y, x, r, s, w, w)
        assert torch.equal(g.dx[rest], h.dx[rest]) and torch.equal(g.dresidual, h.dresidual)


def test_gradients_are_not_recorded(gpu):
    """Operands of the sequence operators that require a gradient bring a
    warning; an optimiser's parameters may require them."""
    x, _, s, d = data(1, 20, 1, 2, 8, 8, torch.float32)
    a = on_gpu(x, s=s)
    for k in INPUTS:
        with pytest.warns(UserWarning, match="requires a gradient"):
            Q.gated_delta_rule(**{**a, k: a[k].clone().requires_grad_()})
    w, t = torch.ones(8, device="cuda"), torch.ones(3, 8, device="cuda")
    with pytest.warns(UserWarning, match="requires a gradient"):
        Q.block_norm(t.clone().requires_grad_(), w, t, w)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        with torch.no_grad():
            Q.gated_delta_rule(**{k: t.clone().requires_grad_() for k, t in a.items()})
        p = [torch.ones(5, device="cuda", requires_grad=True)]
        m, v = [torch.zeros(5, device="cuda")], [torch.zeros(5, device="cuda")]
        optim.adamw(p, [torch.ones(5, device="cuda")], m, v, 1)
        optim.AdamW(p).step([torch.ones(5, device="cuda")])
    assert (p[0] < 1).all()


def test_two_graphs_of_one_program(gpu):
    """Each has scratch of its own: replayed in turn and side by side, both give
    what eager calls give."""
    B, T, H, K, V = 2, 150, 2, 32, 16
    d = Data(8)
    sets = []
    for k in range(2):
        x, _, s, _ = data(B, T, H, H, K, V, torch.float32, seed=k)
        sets.append((on_gpu(x, s=s), d.normal(B, T, H, V).cuda()))
    want = [Q.gated_delta_rule_backward(dy, **a) for a, dy in sets]
    torch.cuda.synchronize()
    graphs = []
    for a, dy in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = Q.gated_delta_rule_backward(dy, **a)
        graphs.append((g, r))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for (g, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for (_, r), w in zip(graphs, want):
            assert all(torch.equal(one, two) for one, two in zip(r, w))


@pytest.mark.parametrize("ty", TYPES)
def test_keys_that_are_alike_and_long_memories(gpu, ty):
    """Keys near one another, strengths near 1 and no decay: the triangular
    systems are far from the identity, and the memory stays bounded."""
    B, T, H, K, V = 1, 256, 2, 32, 16
    d = Data(11)
    base = d.normal(1, 1, H, K)
    x = dict(q=d.normal(B, T, H, K, type=ty), k=(base + 0.1 * d.normal(B, T, H, K)).to(ty), v=d.normal(B, T, H, V, type=ty),
             g=torch.zeros(B, T, H), beta=d.uniform(B, T, H, lo=0.9, hi=1.0))
    want, left = rule(**wide(x), scale=1.0, state=torch.zeros(B, H, K, V, dtype=F64), lengths=[T])
    after = torch.empty(B, H, K, V, device="cuda")
    y = Q.gated_delta_rule(**on_gpu(x), scale=1.0, state_out=after)
    big = max(left.abs().max().item(), want.abs().max().item())
    # (four chained sums of up to 64 a chunk, four chunks, 2^-24 each; bfloat16: one rounding, and 3 2^-16 of eight such sums)
    tol = 4 * 64 * 4 * 2.0 ** -24
    assert ((after.cpu().double() - left).abs() <= tol * big).all()
    assert ((y.cpu().double() - want).abs() <= (tol + (24 * 2.0 ** -16 if ty == torch.bfloat16 else 0.0)) * big
            + (2.0 ** -8 * want.abs() if ty == torch.bfloat16 else 0.0)).all()


@pytest.mark.parametrize("count", [52, 53, 200, 201, 417])
def test_as_many_tensors_as_a_launch_takes_and_more(gpu, count):
    from test_gpu_adamw import ARGS, check, formula, tensors
    p, g, m, v = tensors(count, [(1 + i % 5,) for i in range(count)])
    want = formula(p, g, m, v, 3, max_norm=1e-3, **ARGS)
    norm = optim.adamw(p, g, m, v, 3, max_norm=1e-3, **ARGS)
    check((p, m, v), want)
    close(norm, want[3].cpu(), 70, "norm")
