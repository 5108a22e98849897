"""The control decoder with the delta rule for its mixer and with norms, gates
and scales around its branches: passes and gradients against the same model in
64 bits on the CPU with torch's autograd, streaming against whole clips, a
captured step, and fits that take the framework's own optimiser.  Needs a GPU."""
import pytest

torch = pytest.importorskip("torch")

from dgen_hip.decoder import DecoderConfig, RecurrentDecoder, fit, main  # noqa: E402
from test_gpu_decoder import norm  # noqa: E402

pytestmark = pytest.mark.gpu
F64 = torch.float64
KINDS = [("delta", False), ("delta", True), ("scan", True)]


def small(mixer, around, dtype=torch.float32, **kw):
    return RecurrentDecoder(DecoderConfig(controls=9, hidden=40, inner=72, states=8, window=4, rank=6, mlp=50, blocks=2, dtype=dtype,
                                          mixer=mixer, around=around, heads=4, key_heads=2, key=20, **kw))


def conv(u, w, b, live):
    T, W = u.shape[1], w.shape[1]
    u = torch.where(live, u, 0.0)
    pad = torch.cat([torch.zeros(u.shape[0], W - 1, u.shape[2], dtype=F64), u], 1)
    v = sum(pad[:, k:k + T] * w[:, k] for k in range(W)) + b
    return torch.where(live, v * torch.sigmoid(v), 0.0)


def wide_model(c, P, x, lengths):
    """The decoder in 64 bits, frame by frame."""
    B, T, _ = x.shape
    live = torch.tensor([[t < n for t in range(T)] for n in lengths])[..., None]
    r, h, branch = x @ P["in"], None, None

    def join(r, h, branch):
        if h is None:
            return r
        if not c.around or branch is None:
            return r + h
        h, z = h.split(c.hidden, -1)
        return P[branch + "_scale"] * r + torch.sigmoid(z) * norm(h, P[branch + "_norm"])

    def scan(p, y):
        u, z = (y @ P[p + "xz"]).split(c.inner, -1)
        v = conv(u, P[p + "conv"], P[p + "conv_bias"], live)
        low, Bm, Cm = (v @ P[p + "proj"]).split([c.rank, c.states, c.states], -1)
        step = torch.where(live, torch.nn.functional.softplus(low @ P[p + "dt"] + P[p + "dt_bias"]), 0.0)
        A, s, ys = -torch.exp(P[p + "log_A"]), torch.zeros(B, c.inner, c.states, dtype=F64), []
        for t in range(T):
            s = torch.exp(step[:, t, :, None] * A) * s + (step[:, t] * v[:, t])[..., None] * Bm[:, t, None]
            ys.append((s * Cm[:, t, None]).sum(-1))
        return torch.where(live, (torch.stack(ys, 1) + P[p + "D"] * v) * z * torch.sigmoid(z), 0.0)

    def delta(p, y):
        v = conv(y @ P[p + "xz"], P[p + "conv"], P[p + "conv_bias"], live)
        n = c.key_heads * c.key
        q, k, v = (t.unflatten(-1, (-1, d)) for t, d in zip(v.split([n, n, c.inner], -1), (c.key, c.key, c.inner // c.heads)))
        q, k = ((t / torch.sqrt(t.square().sum(-1, keepdim=True) + 1e-6)).repeat_interleave(c.heads // c.key_heads, 2) for t in (q, k))
        a, b = (y @ P[p + "ab"]).split(c.heads, -1)
        g = -torch.exp(P[p + "log_A"]) * torch.nn.functional.softplus(a + P[p + "dt_bias"])
        g, beta = torch.where(live, g, 0.0), torch.where(live, torch.sigmoid(b), 0.0)
        S, ys = torch.zeros(B, c.heads, c.key, c.inner // c.heads, dtype=F64), []
        for t in range(T):
            S = torch.exp(g[:, t])[..., None, None] * S
            u = beta[:, t, :, None] * (v[:, t] - (k[:, t, :, :, None] * S).sum(2))
            S = S + k[:, t, :, :, None] * u[:, :, None]
            ys.append(c.key ** -0.5 * (q[:, t, :, :, None] * S).sum(2))
        return torch.where(live, torch.stack(ys, 1).flatten(2), 0.0)

    for i in range(c.blocks):
        p = f"{i}."
        r = join(r, h, branch)
        s = (scan if c.mixer == "scan" else delta)(p, norm(r, P[p + "norm1"]))
        r = join(r, s @ P[p + "out"], p + "out")
        m = norm(r, P[p + "norm2"])
        g = m @ P[p + "gate"]
        h, branch = (g * torch.sigmoid(g) * (m @ P[p + "up"])) @ P[p + "down"], p + "down"
    return norm(join(r, h, branch), P["norm"]) @ P["heads"] + P["heads_bias"]


@pytest.mark.parametrize("mixer,around", KINDS)
@pytest.mark.parametrize("T,lengths", [(37, None), (37, [37, 0, 20]), (9, [9, 1, 3])])
def test_passes_against_64_bits(gpu, mixer, around, T, lengths):
    """fp32: a few hundred operations deep through two blocks, each within a
    few 2^-24 of its largest values (the bound of the decoder's other test).  A
    branch that is normed is divided by its own length, which magnifies what it is
    off by: in clips that end, whose padding is the smallest branch there is, by
    at most ten."""
    dec = small(mixer, around)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, T, 2, generator=g)
    dZ = torch.randn(3, T, 9, generator=g)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    Z, kept = dec.forward(x, lengths=n, keep=True)
    grads = dec.backward(dZ.cuda(), kept)
    P = {k: v.cpu().to(F64).requires_grad_() for k, v in dec.params.items()}
    want = wide_model(dec.cfg, P, x.to(F64), lengths or [T] * 3)
    tol = 2e-3 if around else 2e-4
    assert (Z.cpu().to(F64) - want).abs().max() <= tol * want.abs().max()
    (want * dZ.to(F64)).sum().backward()
    for k, p in P.items():
        err = (grads[k].cpu().to(F64) - p.grad).abs().max().item()
        assert err <= tol * p.grad.abs().max().item() + 1e-9, (k, err, p.grad.abs().max().item())


@pytest.mark.parametrize("mixer,around", KINDS)
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-3), (torch.bfloat16, 0.15)])
def test_streaming_follows_whole_clips(gpu, mixer, around, dtype, tol):
    """A prompt and single frames against the whole clip: in fp32 within the
    bound above, in bfloat16 within the roundings of its activations (2^-8
    each, some twenty in a row on the way, independent ones: 0.02 of the
    largest; and as often again through the norms)."""
    dec = small(mixer, around, dtype)
    x = torch.randn(3, 50, 2, generator=torch.Generator().manual_seed(2))
    whole, state = dec.forward(x), dec.state(3)
    out = [dec.forward(x[:, :31], state=state)] + [dec.step(x[:, t], state)[:, None] for t in range(31, 50)]
    assert (torch.cat(out, 1) - whole).abs().max() <= tol * whole.abs().max()


@pytest.mark.parametrize("mixer,around", KINDS)
def test_a_captured_step_replays(gpu, mixer, around):
    dec = small(mixer, around, torch.bfloat16)
    frame, state = torch.randn(4, 2, device="cuda"), dec.state(4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        dec.step(frame, state)
    torch.cuda.current_stream().wait_stream(side)
    for pair in state:
        for t in pair:
            t.zero_()
    eager = dec.state(4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = dec.step(frame, state)
    g = torch.Generator().manual_seed(5)
    for k in range(5):
        frame.copy_(torch.randn(4, 2, generator=g))
        want = dec.step(frame, eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(z, want)


@pytest.mark.parametrize("mixer,around", [("scan", False), *KINDS])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_fit_with_the_frameworks_optimiser(gpu, mixer, around, dtype):
    """Runs, keeps every parameter finite, moves each, and ragged clips may be
    padded with anything."""
    dec = small(mixer, around, dtype)
    x = torch.randn(3, 40, 2, generator=torch.Generator().manual_seed(3))
    target = torch.randn(3, 40, 9, device="cuda")
    x[1, 10:], target[1, 10:] = float("nan"), float("nan")
    before = {k: v.clone() for k, v in dec.params.items()}
    losses = fit(dec, x, target, steps=3, lr=1e-2, lengths=torch.tensor([40, 10, 33]), weight_decay=0.01, max_norm=1.0)
    assert len(losses) == 3 and all(l == l and l < float("inf") for l in losses)
    for k, v in dec.params.items():
        assert torch.isfinite(v).all() and not torch.equal(v, before[k]), k


def test_the_optimisers_steps_are_adams(gpu):
    """Without weight decay and far from the bound: the parameters of torch's
    Adam, to roundings of the steps (lr each, 2^-10 of it)."""
    a, b = small("scan", False), small("scan", False)
    x = torch.randn(2, 30, 2, generator=torch.Generator().manual_seed(4))
    target = torch.randn(2, 30, 9, device="cuda")
    fit(a, x, target, steps=1, lr=1e-2)
    fit(b, x, target, steps=1, lr=1e-2, max_norm=1e6)
    for k in a.params:
        assert (a.params[k] - b.params[k]).abs().max() <= 1e-2 * 2.0 ** -10 + 1e-6 * a.params[k].abs().max(), k


def test_the_command_runs(gpu, capsys):
    main(["--mixer", "delta", "--around", "--steps", "2", "--weight-decay", "0.01", "--max-norm", "1"])
    out = capsys.readouterr().out
    assert "fit: loss" in out and "stream: 500 single frames" in out


def test_refusals():
    with pytest.raises(ValueError, match="mixer"):
        RecurrentDecoder(DecoderConfig(mixer="other"), device="cpu")
    with pytest.raises(ValueError, match="heads"):
        RecurrentDecoder(DecoderConfig(mixer="delta", heads=6, key_heads=4), device="cpu")
    with pytest.raises(ValueError, match="heads"):
        RecurrentDecoder(DecoderConfig(mixer="delta", inner=100, heads=8), device="cpu")
