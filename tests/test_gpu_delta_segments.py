"""How the gated delta rule cuts its calls: by segments of chunks (from 8 chunks
on, from 12 with more than 64 keys' channels, as many as the square root of the
chunks suggests or the card takes) and frame by frame (up to 16 frames),
on both sides of each rule, against the definition in
64 bits.  Needs a GPU.

Tolerances are those of test_gpu_delta_rule, twice over: with segments the memory
that enters one is a product of K numbers with the segment's map, and adds as
many roundings again, no more often than a chunk does."""
import pytest

torch = pytest.importorskip("torch")

from dgen_hip import sequence as Q  # noqa: E402
from test_gpu_delta_rule import INPUTS, data, on_gpu, ops_of, rule, start, wide  # noqa: E402
from test_gpu_sequence import F64, TYPES, close, name_of, spoil  # noqa: E402

pytestmark = pytest.mark.gpu

# (batch, frames, key heads, heads, K, V): 7, 8 and 9 chunks; 11 and 12 with wide
# keys; values over two blocks and sequences that fill the card's share; a last
# segment that is shorter, and sequences that end in the first
SIZES = [(1, 448, 1, 1, 33, 20), (1, 449, 1, 2, 33, 20), (2, 576, 1, 2, 64, 40), (1, 704, 1, 1, 65, 33),
         (2, 705, 1, 1, 128, 70), (8, 520, 2, 6, 16, 33), (24, 513, 1, 2, 8, 64), (25, 513, 1, 2, 8, 64)]


def lengths_of(B, T):
    return [[T, T - 1, 70, 0, T // 2, 64][i % 6] for i in range(B)]


@pytest.mark.parametrize("B,T,G,H,K,V", SIZES)
@pytest.mark.parametrize("ty", TYPES)
def test_segments(gpu, B, T, G, H, K, V, ty):
    x, _, s, d = data(B, T, G, H, K, V, ty, True, slow=True)
    lengths, dy = lengths_of(B, T), d.normal(B, T, H, V, type=ty)
    a = on_gpu(x, lengths, s, True)
    after = torch.full((B, H, K, V), float("nan"), device="cuda")
    y = Q.gated_delta_rule(**a, state_out=after)
    got = Q.gated_delta_rule_backward(spoil(dy, lengths).cuda(), **a)
    again = Q.gated_delta_rule_backward(spoil(dy, lengths).cuda(), **a)
    assert all(torch.equal(p, q) for p, q in zip(got, again))
    for b in range(min(B, 6)):  # (the rest are as long as these)
        one = {k: v[b:b + 1] for k, v in x.items()}
        w = wide(one, True)
        out, left = rule(**w, scale=K ** -0.5, state=s[b:b + 1].to(F64), lengths=lengths[b:b + 1])
        big = max(out.abs().max().item(), left.abs().max().item(), 4.0)
        close(y[b:b + 1], out.detach(), 2 * ops_of(T, K, ty), f"y {name_of(ty)}", big)
        close(after[b:b + 1], left.detach(), 2 * ops_of(T, K), "state", big)
        none = sum(0.0 * t.sum() for t in w.values())
        want = torch.autograd.grad((out * dy[b:b + 1].to(F64)).sum() + none, [w[k] for k in INPUTS])
        for k, t, r in zip(INPUTS, got, want):
            half = ty if k in "qkv" else torch.float32
            short = 1.0 if k not in "qk" else 1.0 / (one[k].to(F64).norm(dim=-1).min().item() + 1e-3)
            most = max(r.abs().max().item(), V ** 0.5 * (1.0 if k in ("v", "beta") else max(1.0, short)))
            close(t[b:b + 1], r, 2 * (4 * ops_of(T, K, half) + 4 * V), f"d{k} {name_of(half)}", most)


@pytest.mark.parametrize("T", [11, 12, 13, 16, 17])
@pytest.mark.parametrize("ty", TYPES)
def test_few_frames(gpu, T, ty):
    B, G, H, K, V = 3, 2, 4, 40, 36
    x, _, s, _ = data(B, T, G, H, K, V, ty)
    lengths = [T, 12, 0]
    want, left = rule(**wide(x), scale=K ** -0.5, state=start(s, B, H, K, V), lengths=lengths)
    after = torch.empty(B, H, K, V, device="cuda")
    y = Q.gated_delta_rule(**on_gpu(x, lengths, s, True), state_out=after)
    big = max(want.abs().max().item(), left.abs().max().item(), 1.0)
    close(y, want, ops_of(T, K, ty), f"y {name_of(ty)}", big)
    close(after, left, ops_of(T, K), "state", max(big, 4.0))


@pytest.mark.parametrize("ty", TYPES)
def test_segments_captured(gpu, ty):
    """A captured forward and backward pass in segments, replayed on other inputs
    with eager calls of the same between."""
    B, T, G, H, K, V = 2, 800, 1, 2, 32, 48
    x, _, s, d = data(B, T, G, H, K, V, ty, True, slow=True)
    a, dy = on_gpu(x, s=s), d.normal(B, T, H, V, type=ty).cuda()
    after = torch.empty(B, H, K, V, device="cuda")

    def run():
        return (Q.gated_delta_rule(**a, state_out=after), after, *Q.gated_delta_rule_backward(dy, **a))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for k in range(4):
        other = data(B, T, G, H, K, V, ty, True, slow=True, seed=k + 1)
        for name, t in other[0].items():
            a[name].copy_(t)
        a["state"].copy_(other[2])
        graph.replay()
        got = [t.clone() for t in out]
        for t in out:
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        want = run()
        assert all(torch.equal(p, q) for p, q in zip(got, want)), k
