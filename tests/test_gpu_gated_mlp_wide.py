"""The gated block's bfloat16 form for many rows at sizes where every part of it
is in use: reductions of many stages, several tiles along each axis, operands
that are copied as they lie and operands that are packed first; element by
element against 64 bits.  The rule that sends a call there is held here too, so
that a change of it cannot leave these cases to another kernel unseen."""
import pytest

torch = pytest.importorskip("torch")

import test_gpu_gated_mlp as G  # noqa: E402

# (rows, width, hidden): whole stages of 32, a tail of rows, and nothing whole
SIZES = [(2304, 544, 2048), (2085, 800, 2016), (2100, 1000, 1999)]


def tiles(n, of):
    return -(-n // of)


@pytest.mark.parametrize("rows,width,hidden", SIZES)
def test_the_sizes_belong_to_the_large_tiles(rows, width, hidden):
    assert rows > 128 and tiles(rows, 256) * tiles(2 * hidden, 256) >= 128  # k_glu.hip, large()
    # stages of a product by the width, of dx and of dW; tiles of dx and of dW
    assert min(tiles(width, 32), 2 * tiles(hidden, 32), tiles(rows, 32)) > 8
    assert tiles(width, 256) > 1 and tiles(hidden, 256) > 1 and tiles(rows, 256) > 1


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,hidden", SIZES)
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("views", [False, True], ids=["contiguous", "views"])
def test_against_64_bits(gpu, monkeypatch, rows, width, hidden, act, views):
    if not views:
        monkeypatch.setattr(G, "view", lambda t, *_: t.cuda())
    G.check_forward(rows, width, hidden, torch.bfloat16, act)
    x, wg, wu, dh, *first = G.check_backward(rows, width, hidden, torch.bfloat16, act)
    again = G.Q.gated_mlp_backward(G.view(dh, 1), G.view(x), G.view(wg, 5, 4), G.view(wu, 2, 1), activation=act)
    for a, b in zip(first, again):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_calls_repeat_bit_for_bit(gpu):
    """A training batch's size, among calls that leave other values in the
    memory that the scratch comes from."""
    g = torch.Generator(device="cuda").manual_seed(1)
    rows, width, hidden = 8000, 1024, 2816

    def normal(*s, scale=1.0):
        return (torch.randn(*s, generator=g, device="cuda") * scale).bfloat16()

    x, dh = normal(rows, width), normal(rows, hidden)
    wg, wu = normal(width, hidden, scale=width ** -0.5), normal(width, hidden, scale=width ** -0.5)
    h, first = G.Q.gated_mlp(x, wg, wu), G.Q.gated_mlp_backward(dh, x, wg, wu)
    for _ in range(6):
        del_me = torch.full((1 << 27,), float("nan"), device="cuda")
        del del_me
        assert torch.equal(G.Q.gated_mlp(x, wg, wu), h)
        for a, b in zip(first, G.Q.gated_mlp_backward(dh, x, wg, wu)):
            assert torch.equal(a, b)
