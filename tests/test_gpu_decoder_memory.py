"""What a pass of the control decoder keeps for its backward pass.  Needs a GPU."""
import pytest

torch = pytest.importorskip("torch")

from dgen_hip.decoder import DecoderConfig, RecurrentDecoder  # noqa: E402

pytestmark = pytest.mark.gpu


def kept_bytes(kept):
    seen = {}

    def walk(t):
        if isinstance(t, torch.Tensor):
            s = t.untyped_storage()
            seen[s.data_ptr()] = s.nbytes()
        elif isinstance(t, (tuple, list)):
            for x in t:
                walk(x)

    walk(kept)
    return sum(seen.values())


@pytest.mark.parametrize("mixer", ["scan", "delta"])
@pytest.mark.parametrize("around", [False, True])
@pytest.mark.parametrize("blocks", [1, 3])
def test_no_more_than_the_gradients_read(gpu, mixer, around, blocks):
    """Each operator's operands once; a branch's output and the stream before it
    only where a norm, a gate and a scale stand between."""
    c = DecoderConfig(controls=9, hidden=64, inner=96, states=8, rank=6, mlp=80, blocks=blocks, dtype=torch.bfloat16, mixer=mixer,
                      around=around, heads=4, key_heads=2, key=32)
    dec, B, T = RecurrentDecoder(c), 2, 50
    _, kept = dec.forward(torch.randn(B, T, 2), keep=True)
    D, E, e = c.hidden, c.inner, 2
    stream, wide = 4 * D, (2 * D if around else D) * e  # the stream, a branch's output
    if mixer == "scan":
        mix = e * (2 * E + E + (c.rank + 2 * c.states) + E + E)
    else:
        mix = e * (2 * (2 * c.key_heads * c.key + E) + E) + 4 * (2 * c.heads + c.heads + c.heads)
    block = e * D + stream + mix + e * D + stream + e * c.mlp + (2 * wide if around else 0)
    frame = e * c.features + blocks * block + e * D + stream
    most = B * T * frame + (blocks * 4 * E * c.states if mixer == "scan" else 0)
    assert kept_bytes(kept) <= most, (kept_bytes(kept), most)
