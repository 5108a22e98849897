"""The gated delta rule (dgen_hip.sequence) against its definition in 64 bits,
frame by frame on the CPU: forward, backward (against the definition's gradient
by torch's autograd in 64 bits, and against differences), single frames,
streaming in pieces, sequences of unequal length, shared keys, views, decays
that forget, captured graphs and streams.  Needs a GPU.

Tolerances.  eps = 2^-24 is the relative rounding error of one fp32 operation.
A chunk of 64 frames chains four sums: of K products (keys with the memory),
twice of up to 64 (the triangular system and its use) and of 64 (the writes), so
a number is off by at most about 2 (K + 192) eps times the largest magnitude on
its way; with unit keys, beta and decays of at most 1 nothing that is carried
grows, and the chunks' errors, independent roundings, add up as the square root
of their number.  Gradients chain twice as many sums, and those of g, sums over
K V products, and of beta over V.  bfloat16 results are rounded once more, by
2^-8 of their own magnitude; before that their products use the two leading
parts of fp32 factors, which leaves 3 2^-16 of the summed magnitudes (taken as
eight times the largest result)."""
import pytest

torch = pytest.importorskip("torch")

from dgen_hip import sequence as Q  # noqa: E402
from test_gpu_sequence import EPS32, F64, TYPES, Data, close, name_of, spoil  # noqa: E402

pytestmark = pytest.mark.gpu

INPUTS = ("q", "k", "v", "g", "beta")


def ops_of(T, K, ty=torch.float32):
    return 2 * (K + 192) * (1 + -(-T // 64)) ** 0.5 + (24 * 2.0 ** 8 if ty == torch.bfloat16 else 0.0)


def rule(q, k, v, g, beta, scale, state, lengths, normalize=True):
    """Definition in 64 bits: (y, state after)."""
    B, T, H, V = v.shape
    share = H // q.shape[2]
    if normalize:
        q, k = (x / torch.sqrt(x.square().sum(-1, keepdim=True) + 1e-6) for x in (q, k))
    ys, left = [], []
    for b in range(B):
        S, rows = state[b], []
        for t in range(max(0, min(T, lengths[b]))):
            kt, qt = k[b, t].repeat_interleave(share, 0), q[b, t].repeat_interleave(share, 0)
            S = torch.exp(g[b, t])[:, None, None] * S
            u = beta[b, t][:, None] * (v[b, t] - (kt[:, :, None] * S).sum(1))
            S = S + kt[:, :, None] * u[:, None]
            rows.append(scale * (qt[:, :, None] * S).sum(1))
        rows += [torch.zeros(H, V, dtype=F64)] * (T - len(rows))
        ys.append(torch.stack(rows))
        left.append(S)
    return torch.stack(ys), torch.stack(left)


def data(B, T, G, H, K, V, ty, state=True, ragged=False, seed=0, slow=False):
    d = Data(B + 3 * T + 5 * H + 7 * K + seed)
    g = -d.uniform(B, T, H, lo=0.0, hi=1.0) ** 2 * (0.02 if slow else 1.0)
    x = dict(q=d.normal(B, T, G, K, type=ty), k=d.normal(B, T, G, K, type=ty), v=d.normal(B, T, H, V, type=ty), g=g,
             beta=d.uniform(B, T, H))
    lengths = [[T, 0, T + 5, -3, max(0, T - 1), T // 2][(i + T) % 6] for i in range(B)] if ragged else [T] * B
    s = d.normal(B, H, K, V, scale=0.3) if state else None
    return x, lengths, s, d


def wide(x, grad=False):
    return {k: v.to(F64).requires_grad_(grad) for k, v in x.items()}


def start(s, B, H, K, V):
    return torch.zeros(B, H, K, V, dtype=F64) if s is None else s.to(F64)


def on_gpu(x, lengths=None, s=None, ragged=False):
    out = {k: (spoil(v, lengths) if ragged else v).cuda() for k, v in x.items()}
    if s is not None:
        out["state"] = s.cuda()
    if ragged:
        out["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    return out


SIZES = [(1, 1, 1, 1, 1, 1), (2, 1, 2, 4, 40, 33), (3, 5, 1, 3, 16, 8), (2, 16, 2, 2, 128, 64), (2, 17, 1, 2, 33, 31),
         (1, 63, 1, 1, 64, 32), (2, 64, 2, 2, 32, 96), (3, 65, 1, 2, 65, 5), (6, 130, 1, 1, 128, 20), (1, 200, 2, 6, 7, 130)]


@pytest.mark.parametrize("B,T,G,H,K,V", SIZES)
@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("ragged,state", [(True, True), (False, False)])
def test_forward(gpu, B, T, G, H, K, V, ty, ragged, state):
    x, lengths, s, _ = data(B, T, G, H, K, V, ty, state, ragged)
    want, left = rule(**wide(x), scale=K ** -0.5, state=start(s, B, H, K, V), lengths=lengths)
    a = on_gpu(x, lengths, s, ragged)
    after = torch.full((B, H, K, V), float("nan"), device="cuda")
    y = Q.gated_delta_rule(**a, state_out=after)
    big = max(want.abs().max().item(), left.abs().max().item(), 1.0)
    assert y.dtype == ty
    close(y, want, ops_of(T, K, ty), f"y {name_of(ty)}", big)
    close(after, left, ops_of(T, K), "state", max(big, 4.0))
    if s is not None:  # the state may be replaced in place
        y2 = Q.gated_delta_rule(**a, state_out=a["state"])
        assert torch.equal(y2, y) and torch.equal(a["state"], after)


@pytest.mark.parametrize("B,T,G,H,K,V", SIZES)
@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("ragged,state", [(True, True), (False, False)])
def test_backward(gpu, B, T, G, H, K, V, ty, ragged, state):
    x, lengths, s, d = data(B, T, G, H, K, V, ty, state, ragged)
    w = wide(x, True)
    out, _ = rule(**w, scale=K ** -0.5, state=start(s, B, H, K, V), lengths=lengths)
    dy = d.normal(B, T, H, V, type=ty)
    none = sum(0.0 * t.sum() for t in w.values())  # (where every sequence is empty)
    want = torch.autograd.grad((out * dy.to(F64)).sum() + none, [w[k] for k in INPUTS])
    a = on_gpu(x, lengths, s, ragged)
    got = Q.gated_delta_rule_backward((spoil(dy, lengths) if ragged else dy).cuda(), **a)
    for k, t, r in zip(INPUTS, got, want):
        half = ty if k in "qkv" else torch.float32
        assert t.dtype == half
        # the gradients of short keys cancel against their norms' (1 / |k| of what they are made of)
        short = 1.0 if k not in "qk" else 1.0 / (x[k].to(F64).norm(dim=-1).min().item() + 1e-3)
        big = max(r.abs().max().item(), V ** 0.5 * (1.0 if k in ("v", "beta") else max(1.0, short)))
        close(t, r, 4 * ops_of(T, K, half) + 4 * V, f"d{k} {name_of(half)}", big)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("B,T,G,H,K,V", [(1, 2100, 1, 2, 40, 50), (1, 4000, 1, 1, 64, 32), (2, 2500, 1, 1, 128, 40)])
def test_long(gpu, B, T, G, H, K, V, ty):
    """Time cut into segments."""
    x, lengths, s, d = data(B, T, G, H, K, V, ty, True, slow=True)
    lengths = [T - 77 * i for i in range(B)]
    want, left = rule(**wide(x), scale=K ** -0.5, state=start(s, B, H, K, V), lengths=lengths)
    a = on_gpu(x, lengths, s, True)
    after = torch.empty(B, H, K, V, device="cuda")
    y = Q.gated_delta_rule(**a, state_out=after)
    big = max(want.abs().max().item(), left.abs().max().item(), 4.0)
    close(y, want, ops_of(T, K, ty), f"y {name_of(ty)}", big)
    close(after, left, ops_of(T, K), "state", big)


def test_long_backward(gpu):
    B, T, G, H, K, V, ty = 2, 2300, 1, 2, 24, 20, torch.float32
    x, _, s, d = data(B, T, G, H, K, V, ty, True, slow=True)
    lengths = [T, 1500]
    w = wide(x, True)
    dy = d.normal(B, T, H, V)
    out, _ = rule(**w, scale=K ** -0.5, state=start(s, B, H, K, V), lengths=lengths)
    want = torch.autograd.grad((out * dy.to(F64)).sum(), [w[k] for k in INPUTS])
    got = Q.gated_delta_rule_backward(spoil(dy, lengths).cuda(), **on_gpu(x, lengths, s, True))
    for k, t, r in zip(INPUTS, got, want):
        short = 1.0 if k not in "qk" else 1.0 / (x[k].to(F64).norm(dim=-1).min().item() + 1e-3)
        close(t, r, 4 * ops_of(T, K) + 4 * V, "d" + k, max(r.abs().max().item(), V ** 0.5 * max(1.0, short)))


def test_gradients_against_differences(gpu):
    B, T, G, H, K, V = 2, 70, 2, 4, 24, 20
    x, _, s, d = data(B, T, G, H, K, V, torch.float32)
    a, dy = on_gpu(x, s=s), d.normal(B, T, H, V)
    got = Q.gated_delta_rule_backward(dy.cuda(), **a)
    for k, t in zip(INPUTS, got):
        u = d.normal(*x[k].shape).cuda()
        u /= u.norm()
        e = 1e-2
        hi, lo = (Q.gated_delta_rule(**{**a, k: a[k] + sign * e * u}).double() for sign in (1, -1))
        num = ((hi - lo) * dy.cuda().double()).sum() / (2 * e)
        ana = (t.double() * u.double()).sum()
        # (third derivatives e^2 / 6, and the results' rounding over 2 e)
        assert abs(num - ana) <= 2e-3 * max(1.0, abs(ana.item())), (k, num.item(), ana.item())


@pytest.mark.parametrize("ty", TYPES)
def test_keys_as_they_are_and_a_scale(gpu, ty):
    B, T, G, H, K, V = 2, 70, 1, 2, 16, 12
    x, _, s, d = data(B, T, G, H, K, V, ty)
    x["k"] = (x["k"].to(F64) / x["k"].to(F64).norm(dim=-1, keepdim=True) * 0.9).to(ty)
    w = wide(x, True)
    out, left = rule(**w, scale=0.7, state=s.to(F64), lengths=[T] * B, normalize=False)
    a = on_gpu(x, s=s)
    after = torch.empty_like(a["state"])
    y = Q.gated_delta_rule(**a, scale=0.7, normalize=False, state_out=after)
    close(y, out, ops_of(T, K, ty), f"y {name_of(ty)}", max(8.0, out.abs().max().item()))
    close(after, left, ops_of(T, K), "state", 4.0)
    dy = d.normal(B, T, H, V, type=ty)
    want = torch.autograd.grad((out * dy.to(F64)).sum(), [w[k] for k in INPUTS])
    got = Q.gated_delta_rule_backward(dy.cuda(), **a, scale=0.7, normalize=False)
    for k, t, r in zip(INPUTS, got, want):
        half = ty if k in "qkv" else torch.float32
        close(t, r, 4 * ops_of(T, K, half) + 4 * V, f"d{k} {name_of(half)}", max(r.abs().max().item(), 4 * V ** 0.5))
    # a few frames at a time take the other kernel
    part = Q.gated_delta_rule(**{k: (v[:, :9] if k in INPUTS else v) for k, v in a.items()}, scale=0.7, normalize=False)
    close(part, out[:, :9], ops_of(9, K, ty), f"y {name_of(ty)}", max(8.0, out.abs().max().item()))


@pytest.mark.parametrize("ty", TYPES)
def test_in_pieces(gpu, ty):
    """A prompt, then single frames, carry the state: as the whole clip."""
    B, T, G, H, K, V = 3, 180, 1, 2, 40, 24
    x, lengths, s, _ = data(B, T, G, H, K, V, ty)
    want, left = rule(**wide(x), scale=K ** -0.5, state=s.to(F64), lengths=lengths)
    a = on_gpu(x, s=s)
    state, t, got = a.pop("state"), 0, []
    for n in (130, 1, 1, 1, 5, 1, 16, 17, 8):
        got.append(Q.gated_delta_rule(**{k: v[:, t:t + n] for k, v in a.items()}, state=state, state_out=state))
        t += n
    assert t == T
    close(torch.cat(got, 1), want, ops_of(T, K, ty) * 2, f"y {name_of(ty)}", max(4.0, want.abs().max().item()))
    close(state, left, ops_of(T, K) * 2, "state", 4.0)


@pytest.mark.parametrize("T", [1, 12, 64, 150])
@pytest.mark.parametrize("low", [-float("inf"), -1e30, -500.0, -128.0, -100.0])
def test_decays_that_forget(gpu, T, low):
    """What lies before such a frame counts for nothing, and what lies after it
    is as exact as ever; no gradient is spoilt."""
    B, G, H, K, V = 2, 1, 2, 16, 8
    x, lengths, s, d = data(B, T, G, H, K, V, torch.float32)
    at = T // 2
    x["g"][:, at:at + 3] = low
    x["g"][:, T - 1] = -1e-3
    if T == 1:
        x["g"][:] = low
    w = wide(x, True)
    want, left = rule(**w, scale=K ** -0.5, state=s.to(F64), lengths=lengths)
    a = on_gpu(x, s=s)
    after = torch.empty_like(a["state"])
    y = Q.gated_delta_rule(**a, state_out=after)
    close(y, want, ops_of(T, K), "y", max(1.0, want.abs().max().item()))
    close(after, left, ops_of(T, K), "state", 4.0)
    dy = d.normal(B, T, H, V)
    grads = torch.autograd.grad((want * dy.to(F64)).sum(), [w[k] for k in INPUTS])
    got = Q.gated_delta_rule_backward(dy.cuda(), **a)
    for k, t, r in zip(INPUTS, got, grads):
        r = torch.nan_to_num(r) if k == "g" else r  # (0 times infinity in the definition's own derivative)
        short = 1.0 if k not in "qk" else 1.0 / (x[k].to(F64).norm(dim=-1).min().item() + 1e-3)
        close(t, r, 4 * ops_of(T, K) + 4 * V, "d" + k, max(r.abs().max().item(), V ** 0.5 * max(1.0, short)))


def test_one_key_again_and_again(gpu):
    """The same key in every frame, written in full: the triangular system at
    its worst, and the memory holds the last value."""
    B, T, K, V = 1, 128, 32, 16
    d = Data(4)
    k = d.normal(1, 1, 1, K).expand(B, T, 1, K).contiguous()
    v, zero = d.normal(B, T, 1, V), torch.zeros(B, T, 1)
    x = dict(q=k, k=k, v=v, g=zero, beta=torch.ones(B, T, 1))
    y = Q.gated_delta_rule(**on_gpu(x), scale=1.0)
    want, _ = rule(**wide(x), scale=1.0, state=torch.zeros(B, 1, K, V, dtype=F64), lengths=[T])
    close(y, want, ops_of(T, K), "y", 4.0)
    # (a frame reads what it wrote, short of the unit's eps)
    close(y, v.to(F64), ops_of(T, K), "y", 4.0 + 1e-6 / EPS32)


def test_writes_of_twice_the_difference(gpu):
    """beta up to 2 reflects the memory, which still does not grow."""
    B, T, G, H, K, V = 1, 200, 1, 2, 16, 8
    x, lengths, s, _ = data(B, T, G, H, K, V, torch.float32)
    x["beta"] = x["beta"] * 2
    want, left = rule(**wide(x), scale=K ** -0.5, state=s.to(F64), lengths=lengths)
    a = on_gpu(x, s=s)
    after = torch.empty_like(a["state"])
    y = Q.gated_delta_rule(**a, state_out=after)
    close(y, want, 4 * ops_of(T, K), "y", max(4.0, left.abs().max().item()))
    close(after, left, 4 * ops_of(T, K), "state", max(4.0, left.abs().max().item()))


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("T", [7, 100])
def test_views(gpu, ty, T):
    """Parts of one projection's output, time-major operands, repeated keys, a
    result in a view: as of tensors of their own, bit for bit."""
    B, G, H, K, V = 2, 2, 4, 24, 17
    d = Data(T)
    qkv = d.normal(B, T, 2 * G * K + H * V + 3, type=ty).cuda()
    q, k, v = qkv[..., :G * K].unflatten(-1, (G, K)), qkv[..., G * K:2 * G * K].unflatten(-1, (G, K)), \
        qkv[..., 2 * G * K + 1:2 * G * K + 1 + H * V].unflatten(-1, (H, V))
    gb = d.uniform(T, B, 2 * H, lo=-1.0, hi=0.0).cuda().transpose(0, 1)
    g, beta = gb[..., :H], gb[..., H:]
    plain = [t.contiguous() for t in (q, k, v, g, beta)]
    want, left = (torch.empty(B, H, K, V, device="cuda") for _ in range(2))
    y = Q.gated_delta_rule(*plain, state_out=want)
    place = torch.full((T, B, H, V + 5), 7.0, dtype=ty, device="cuda")
    out = place[..., 2:2 + V].transpose(0, 1)
    assert Q.gated_delta_rule(q, k, v, g, beta, state_out=left, out=out) is out
    assert torch.equal(out, y) and torch.equal(left, want)
    assert (place[..., :2] == 7).all() and (place[..., 2 + V:] == 7).all()
    dy = d.normal(H, T, B, V, type=ty).cuda().permute(2, 1, 0, 3)
    for a, b in zip(Q.gated_delta_rule_backward(dy, q, k, v, g, beta),
                    Q.gated_delta_rule_backward(dy.contiguous(), *plain)):
        assert torch.equal(a, b) and a.is_contiguous()
    same = q[:, :1, :1].expand(B, T, G, K)
    assert torch.equal(Q.gated_delta_rule(same, same, v, g, beta), Q.gated_delta_rule(same.contiguous(), same.contiguous(), v, g, beta))


@pytest.mark.parametrize("T", [5, 70])
def test_results_over_operands(gpu, T):
    B, H, K = 2, 2, 16
    x, _, s, _ = data(B, T, H, H, K, K, torch.float32)
    a = on_gpu(x, s=s)
    want = torch.empty_like(a["state"])
    y = Q.gated_delta_rule(**a, state_out=want)
    for name in ("v", "k", "q"):
        b = {k: t.clone() for k, t in a.items()}
        assert Q.gated_delta_rule(**b, out=b[name]) is b[name] and torch.equal(b[name], y)
    b = {k: t.clone() for k, t in a.items()}
    flat = torch.cat([b["v"].flatten(), torch.zeros(7, device="cuda")])
    b["v"], out = flat[:-7].view_as(y), flat[7:].view_as(y)
    assert torch.equal(Q.gated_delta_rule(**b, out=out), y)
    both = torch.empty(max(y.numel(), want.numel()), device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        Q.gated_delta_rule(**a, out=both[:y.numel()].view_as(y), state_out=both[:want.numel()].view_as(want))


def test_calls_repeat_bit_for_bit(gpu):
    x, lengths, s, d = data(2, 300, 1, 3, 40, 33, torch.bfloat16, True, True)
    a, dy = on_gpu(x, lengths, s, True), d.normal(2, 300, 3, 33, type=torch.bfloat16).cuda()
    for one, two in zip(*(Q.gated_delta_rule_backward(dy, **a) for _ in range(2))):
        assert torch.equal(one, two)
    assert torch.equal(Q.gated_delta_rule(**a), Q.gated_delta_rule(**a))


def test_captured(gpu):
    """A captured step and a captured backward pass, replayed with other
    values, between eager calls."""
    for T in (1, 100):
        x, _, s, d = data(2, T, 1, 2, 32, 20, torch.bfloat16)
        a, dy = on_gpu(x, s=s), d.normal(2, T, 2, 20, type=torch.bfloat16).cuda()
        state = a.pop("state")
        first = state.clone()
        Q.gated_delta_rule(**a, state=first, state_out=first)  # (loads the library)
        Q.gated_delta_rule_backward(dy, **a, state=state)
        torch.cuda.synchronize()
        graph, carried = torch.cuda.CUDAGraph(), state.clone()
        with torch.cuda.graph(graph):
            grads = Q.gated_delta_rule_backward(dy, **a, state=carried)
            y = Q.gated_delta_rule(**a, state=carried, state_out=carried)
        eager = state.clone()
        for n in range(4):
            a["v"].copy_(d.normal(2, T, 2, 20, type=torch.bfloat16))
            want_grads = Q.gated_delta_rule_backward(dy, **a, state=eager)
            want = Q.gated_delta_rule(**a, state=eager, state_out=eager)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want) and torch.equal(carried, eager)
            for one, two in zip(grads, want_grads):
                assert torch.equal(one, two)


def test_streams(gpu):
    x, _, s, d = data(2, 100, 1, 2, 32, 20, torch.float32)
    a, dy = on_gpu(x, s=s), d.normal(2, 100, 2, 20).cuda()
    want, grads = Q.gated_delta_rule(**a), Q.gated_delta_rule_backward(dy, **a)
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for side in sides:  # two calls at once
        with torch.cuda.stream(side):
            v = a["v"].clone()
            got.append((Q.gated_delta_rule(**{**a, "v": v}), Q.gated_delta_rule_backward(dy, **{**a, "v": v})))
    torch.cuda.synchronize()
    for y, r in got:
        assert torch.equal(y, want) and all(torch.equal(one, two) for one, two in zip(r, grads))


def test_no_sequences_and_no_keys_that_count(gpu):
    f = dict(device="cuda")
    for T in (3, 80):
        z = torch.zeros(0, T, 2, 8, **f)
        e = torch.zeros(0, T, 2, **f)
        assert Q.gated_delta_rule(z, z, z, e, e).shape == (0, T, 2, 8)
        assert Q.gated_delta_rule_backward(z, z, z, z, e, e).dq.shape == (0, T, 2, 8)
        # keys and queries of zeros: nothing is written or read, and no gradient is spoilt
        o, b = torch.ones(2, T, 2, 8, **f), torch.ones(2, T, 2, **f)
        zero = torch.zeros_like(o)
        assert torch.equal(Q.gated_delta_rule(zero, zero, o, -b, b), zero)
        for t in Q.gated_delta_rule_backward(o, zero, zero, o, -b, b):
            assert torch.isfinite(t).all()


def test_refusals(gpu):
    f = dict(device="cuda")
    q, v, g = torch.zeros(2, 5, 2, 8, **f), torch.zeros(2, 5, 4, 6, **f), torch.zeros(2, 5, 4, **f)
    ok = dict(q=q, k=q, v=v, g=g, beta=g)
    Q.gated_delta_rule(**ok)
    for wrong in (dict(q=q.cpu()), dict(q=q.half()), dict(k=q[..., :7]), dict(k=q[:, :4]), dict(v=v[:, :4]), dict(v=v[:, :, :3]),
                  dict(g=g.bfloat16()), dict(beta=g[..., :3]), dict(q=q.transpose(2, 3)), dict(q=q[0]), dict(v=v[0]),
                  dict(state=torch.zeros(2, 4, 8, 7, **f)), dict(state=torch.zeros(2, 4, 8, 6, dtype=torch.bfloat16, **f)),
                  dict(state_out=torch.zeros(2, 4, 6, 8, **f)), dict(lengths=torch.zeros(2, dtype=torch.int64, **f)),
                  dict(lengths=torch.zeros(3, dtype=torch.int32, **f)), dict(out=torch.zeros(1, 5, 4, 6, **f).expand(2, 5, 4, 6)),
                  dict(out=torch.zeros(2, 5, 1, 6, **f).expand(2, 5, 4, 6)), dict(scale=0.0), dict(scale=float("nan")),
                  dict(q=torch.zeros(2, 5, 2, 129, **f), k=torch.zeros(2, 5, 2, 129, **f)),
                  dict(v=torch.zeros(2, 5, 4, 1025, **f)), dict(q=q[:, :0], k=q[:, :0], v=v[:, :0], g=g[:, :0], beta=g[:, :0])):
        with pytest.raises(ValueError):
            Q.gated_delta_rule(**{**ok, **wrong})
        if "out" not in wrong and "state_out" not in wrong:
            with pytest.raises(ValueError):
                Q.gated_delta_rule_backward(torch.zeros_like(v) if "v" not in wrong else torch.zeros_like(wrong["v"]), **{**ok, **wrong})
    with pytest.raises(ValueError):
        Q.gated_delta_rule_backward(v[..., :5], **ok)
