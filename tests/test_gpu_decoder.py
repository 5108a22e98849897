"""The recurrent control decoder (dgen_hip.decoder): its passes against the
same model in 64 bits on the CPU with torch's autograd, streaming against whole
clips, and a fit that lowers its loss.  Needs a GPU."""
import pytest
import torch

from dgen_hip.decoder import DecoderConfig, RecurrentDecoder, fit

pytestmark = pytest.mark.gpu
F64 = torch.float64


def small(dtype=torch.float32, **kw):
    return RecurrentDecoder(DecoderConfig(controls=9, hidden=40, inner=72, states=8, window=4, rank=6, mlp=50, blocks=2,
                                          dtype=dtype, **kw))


def norm(s, w):
    return s * torch.rsqrt(s.square().mean(-1, keepdim=True) + 1e-5) * w


def wide_model(cfg, P, x, lengths):
    """The decoder in 64 bits, frame by frame."""
    B, T, _ = x.shape
    live = torch.tensor([[t < n for t in range(T)] for n in lengths])[..., None]
    zero = torch.zeros(1, dtype=F64)
    r, h = x @ P["in"], 0.0
    for i in range(cfg.blocks):
        p = f"{i}."
        r = r + h
        xz = norm(r, P[p + "norm1"]) @ P[p + "xz"]
        u, z = xz.split(cfg.inner, -1)
        u = torch.where(live, u, zero)
        pad = torch.cat([torch.zeros(B, cfg.window - 1, cfg.inner, dtype=F64), u], 1)
        v = sum(pad[:, k:k + T] * P[p + "conv"][:, k] for k in range(cfg.window)) + P[p + "conv_bias"]
        v = torch.where(live, v * torch.sigmoid(v), zero)
        low, Bm, Cm = (v @ P[p + "proj"]).split([cfg.rank, cfg.states, cfg.states], -1)
        step = torch.where(live, torch.nn.functional.softplus(low @ P[p + "dt"] + P[p + "dt_bias"]), zero)
        A, s, ys = -torch.exp(P[p + "log_A"]), torch.zeros(B, cfg.inner, cfg.states, dtype=F64), []
        for t in range(T):
            s = torch.exp(step[:, t, :, None] * A) * s + (step[:, t] * v[:, t])[..., None] * Bm[:, t, None]
            ys.append((s * Cm[:, t, None]).sum(-1))
        y = (torch.stack(ys, 1) + P[p + "D"] * v) * z * torch.sigmoid(z)
        r = r + torch.where(live, y, zero) @ P[p + "out"]
        m = norm(r, P[p + "norm2"])
        g = m @ P[p + "gate"]
        h = (g * torch.sigmoid(g) * (m @ P[p + "up"])) @ P[p + "down"]
    return norm(r + h, P["norm"]) @ P["heads"] + P["heads_bias"]


@pytest.mark.parametrize("lengths", [None, [37, 0, 20]])
def test_passes_against_64_bits(gpu, lengths):
    """fp32: a few hundred operations deep through two blocks, each within a
    few 2^-24 of its largest values; 2e-4 of the largest entry leaves a factor
    of ten over 2000 of them."""
    dec = small()
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 37, 2, generator=g)
    dZ = torch.randn(3, 37, 9, generator=g)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    Z, kept = dec.forward(x, lengths=n, keep=True)
    grads = dec.backward(dZ.cuda(), kept)
    P = {k: v.cpu().to(F64).requires_grad_() for k, v in dec.params.items()}
    want = wide_model(dec.cfg, P, x.to(F64), lengths or [37] * 3)
    assert (Z.cpu().to(F64) - want).abs().max() <= 2e-4 * want.abs().max()
    (want * dZ.to(F64)).sum().backward()
    for k, p in P.items():
        err = (grads[k].cpu().to(F64) - p.grad).abs().max().item()
        assert err <= 2e-4 * p.grad.abs().max().item() + 1e-9, (k, err)


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-4), (torch.bfloat16, 0.1)])
def test_streaming_follows_whole_clips(gpu, dtype, tol):
    """A prompt and single frames against the whole clip: in fp32 within the
    bound above, in bfloat16 within the roundings of its activations (2^-8 each,
    a dozen in a row at most on the way)."""
    dec = small(dtype)
    x = torch.randn(3, 30, 2, generator=torch.Generator().manual_seed(2))
    whole, state = dec.forward(x), dec.state(3)
    out = [dec.forward(x[:, :11], state=state)] + [dec.step(x[:, t], state)[:, None] for t in range(11, 30)]
    assert (torch.cat(out, 1) - whole).abs().max() <= tol * whole.abs().max()


def test_fit_lowers_the_loss(gpu):
    dec = small(torch.bfloat16)
    g = torch.Generator().manual_seed(4)
    x = torch.randn(4, 60, 2, generator=g)
    # each frame's target is the mean of the features so far: a memory is needed
    target = (x.cumsum(1) / torch.arange(1, 61)[None, :, None])[..., :1].repeat(1, 1, 9).cuda()
    losses = fit(dec, x, target, steps=60, lr=3e-3, lengths=torch.tensor([60, 50, 7, 60], dtype=torch.int32, device="cuda"))
    assert losses[-1] < 0.2 * losses[0], (losses[0], losses[-1])


def test_a_step_in_a_graph(gpu):
    """A captured step (torch.cuda.graph) replays with new frames and carries
    its state, as eager steps do, with other work between the replays."""
    dec = small(torch.bfloat16)
    x = torch.randn(3, 12, 2, generator=torch.Generator().manual_seed(6)).cuda()
    state = dec.state(3)
    eager = [dec.step(x[:, t], state) for t in range(12)]
    held, frame = dec.state(3), x[:, 0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            dec.step(frame, held)  # libraries set up outside the capture
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = dec.step(frame, held)
    for c, s in held:
        c.zero_()
        s.zero_()
    for t in range(12):
        frame.copy_(x[:, t])
        graph.replay()
        assert torch.equal(out, eager[t]), t
        if t % 3 == 0:
            torch.cuda.synchronize()
            dec.forward(x)  # eager work between replays
    for (c, s), (ce, se) in zip(held, state):
        assert torch.equal(c, ce) and torch.equal(s, se)
