"""The recurrent control decoder trained on pieces of clips, which go on from a
state, and fitted to padded ones.  Needs a GPU."""
import pytest

torch = pytest.importorskip("torch")

from dgen_hip.decoder import fit  # noqa: E402
from test_gpu_decoder import F64, norm, small  # noqa: E402

pytestmark = pytest.mark.gpu


def wide_model(cfg, P, x, state):
    """The decoder in 64 bits, frame by frame, from a state."""
    B, T, _ = x.shape
    r, h = x @ P["in"], 0.0
    for i in range(cfg.blocks):
        p = f"{i}."
        r = r + h
        u, z = (norm(r, P[p + "norm1"]) @ P[p + "xz"]).split(cfg.inner, -1)
        before, s = state[i]
        row = torch.cat([before, u], 1)
        v = sum(row[:, k:k + T] * P[p + "conv"][:, k] for k in range(cfg.window)) + P[p + "conv_bias"]
        v = v * torch.sigmoid(v)
        low, Bm, Cm = (v @ P[p + "proj"]).split([cfg.rank, cfg.states, cfg.states], -1)
        step = torch.nn.functional.softplus(low @ P[p + "dt"] + P[p + "dt_bias"])
        A, ys = -torch.exp(P[p + "log_A"]), []
        for t in range(T):
            s = torch.exp(step[:, t, :, None] * A) * s + (step[:, t] * v[:, t])[..., None] * Bm[:, t, None]
            ys.append((s * Cm[:, t, None]).sum(-1))
        r = r + ((torch.stack(ys, 1) + P[p + "D"] * v) * z * torch.sigmoid(z)) @ P[p + "out"]
        m = norm(r, P[p + "norm2"])
        g = m @ P[p + "gate"]
        h = (g * torch.sigmoid(g) * (m @ P[p + "up"])) @ P[p + "down"]
    return norm(r + h, P["norm"]) @ P["heads"] + P["heads_bias"]


def test_gradients_of_a_piece_that_goes_on_from_a_state(gpu):
    """The state counts as given; tolerances as those of whole clips."""
    dec = small()
    g = torch.Generator().manual_seed(8)
    first, x, dZ = (torch.randn(3, n, k, generator=g) for n, k in ((19, 2), (23, 2), (23, 9)))
    state = dec.state(3)
    dec.forward(first, state=state)
    start = [(c.cpu().to(F64), s.cpu().to(F64)) for c, s in state]
    assert all(c.any() and s.any() for c, s in start)
    Z, kept = dec.forward(x, state=state, keep=True)
    moved = [(c.clone(), s.clone()) for c, s in state]
    dec.forward(first, state=state)  # the state has moved on again before the backward pass
    grads = dec.backward(dZ.cuda(), kept)
    P = {k: v.cpu().to(F64).requires_grad_() for k, v in dec.params.items()}
    want = wide_model(dec.cfg, P, x.to(F64), start)
    assert (Z.cpu().to(F64) - want).abs().max() <= 2e-4 * want.abs().max()
    (want * dZ.to(F64)).sum().backward()
    for k, p in P.items():
        err = (grads[k].cpu().to(F64) - p.grad).abs().max().item()
        assert err <= 2e-4 * p.grad.abs().max().item() + 1e-9, (k, err)
    # keeping changes neither the result nor where the state goes
    again = [(c.to(dec.cfg.dtype).cuda(), s.float().cuda()) for c, s in start]
    assert torch.equal(dec.forward(x, state=again), Z)
    for (c, s), (cm, sm) in zip(again, moved):
        assert torch.equal(c, cm) and torch.equal(s, sm)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("device", ["cpu", "cuda"])
def test_fit_takes_the_lengths_as_a_program_has_them(gpu, dtype, device):
    """On the host or the device, in 32 or 64 bits; the loss is the mean over
    the clips' own frames, whatever the padding holds."""
    losses = []
    for pad in (0, 13):
        dec = small()
        g = torch.Generator().manual_seed(10)
        x, target = torch.randn(2, 30, 2, generator=g), torch.randn(2, 30, 9, generator=g)
        x = torch.cat([x, torch.full((2, pad, 2), float("nan"))], 1)
        target = torch.cat([target, torch.full((2, pad, 9), float("nan"))], 1).cuda()
        losses.append(fit(dec, x, target, steps=4, lengths=torch.tensor([30, 11], dtype=dtype, device=device)))
    for a, b in zip(*losses):
        assert abs(a - b) <= 1e-5 * a, losses
    dec = small()
    Z = dec.forward(x[:, :30], lengths=torch.tensor([30, 11], dtype=torch.int32, device="cuda"))
    d = (Z - target[:, :30]).square()
    mean = (d[0].sum() + d[1, :11].sum()) / (41 * 9)
    assert abs(losses[0][0] - mean.item()) <= 1e-5 * mean.item()
