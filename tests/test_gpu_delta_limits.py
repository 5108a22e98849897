"""The gated delta rule where its cuts change and at the smallest scales: the first
and the last sequences of calls that fill the card's share, wide keys on both
sides of the rule for segments, scales below the normal numbers.  Needs a GPU.

Tolerances are those of test_gpu_delta_segments."""
import pytest

torch = pytest.importorskip("torch")

from dgen_hip import sequence as Q  # noqa: E402
from test_gpu_delta_rule import INPUTS, data, on_gpu, ops_of, rule, wide  # noqa: E402
from test_gpu_sequence import F64, TYPES, Data, close, name_of, spoil  # noqa: E402

pytestmark = pytest.mark.gpu

# (batch, frames, key heads, heads, K, V): 48 and 96 blocks of values, and 100;
# with keys of more than 64 channels 40, and 42, of 12 chunks
SIZES = [(8, 520, 2, 6, 16, 33), (24, 513, 1, 2, 8, 64), (25, 513, 1, 2, 8, 64), (4, 705, 1, 2, 65, 150), (6, 705, 1, 1, 128, 224)]


@pytest.mark.parametrize("B,T,G,H,K,V", SIZES)
@pytest.mark.parametrize("ty", TYPES)
def test_the_first_and_the_last_sequences(gpu, B, T, G, H, K, V, ty):
    x, _, s, d = data(B, T, G, H, K, V, ty, True, slow=True)
    lengths, dy = [[T - i, T, T - 70][i % 3] for i in range(B)], d.normal(B, T, H, V, type=ty)
    a = on_gpu(x, lengths, s, True)
    after = torch.full((B, H, K, V), float("nan"), device="cuda")
    y = Q.gated_delta_rule(**a, state_out=after)
    got = Q.gated_delta_rule_backward(spoil(dy, lengths).cuda(), **a)
    for b in (0, B - 2, B - 1):
        one = {k: v[b:b + 1] for k, v in x.items()}
        w = wide(one, True)
        out, left = rule(**w, scale=K ** -0.5, state=s[b:b + 1].to(F64), lengths=lengths[b:b + 1])
        big = max(out.abs().max().item(), left.abs().max().item(), 4.0)
        close(y[b:b + 1], out.detach(), 2 * ops_of(T, K, ty), f"y {name_of(ty)}", big)
        close(after[b:b + 1], left.detach(), 2 * ops_of(T, K), "state", big)
        want = torch.autograd.grad((out * dy[b:b + 1].to(F64)).sum(), [w[k] for k in INPUTS])
        for k, t, r in zip(INPUTS, got, want):
            half = ty if k in "qkv" else torch.float32
            short = 1.0 if k not in "qk" else 1.0 / (one[k].to(F64).norm(dim=-1).min().item() + 1e-3)
            most = max(r.abs().max().item(), V ** 0.5 * (1.0 if k in ("v", "beta") else max(1.0, short)))
            close(t[b:b + 1], r, 2 * (4 * ops_of(T, K, half) + 4 * V), f"d{k} {name_of(half)}", most)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("T", [9, 70, 600])
def test_a_scale_below_the_normal_numbers(gpu, ty, T):
    """What it gives may be taken for 0, and is no larger than it should be: each
    of the sums' few hundred terms may be rounded to the least number, 2^-149."""
    B, H, K, V, scale = 1, 2, 16, 8, 1e-41
    x, _, s, d = data(B, T, H, H, K, V, ty)
    a, dy = on_gpu(x, s=s), d.normal(B, T, H, V, type=ty).cuda()
    one, r = Q.gated_delta_rule(**a, scale=1.0), Q.gated_delta_rule_backward(dy, **a, scale=1.0)
    for got, want in zip((Q.gated_delta_rule(**a, scale=scale), *Q.gated_delta_rule_backward(dy, **a, scale=scale)), (one, *r)):
        assert torch.isfinite(got).all()
        # (bfloat16's least number is 2^-133)
        least = 512 * 2.0 ** -149 + (2.0 ** -133 if got.dtype == torch.bfloat16 else 0.0)
        assert got.double().abs().max() <= 1.01 * scale * want.double().abs().max() + least
