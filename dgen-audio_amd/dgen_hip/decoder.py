"""A recurrent control decoder: per-frame features of a clip to synth controls,
with a memory of the frames before (the reference's decoder,
Examples/HarmonicE2E/Model.swift:96-120, sees one frame at a time).

Each block adds two branches to a residual stream kept in 32 bits:

    norm -> projection to (x, z) -> causal convolution -> projection to
    (step, B, C) -> selective scan, gated by z -> projection back
    norm -> gated feed-forward block -> projection back

and a last norm and projection give the head pre-activations (the Z of the
harmonic synth's heads: amplitudes, gains, taps; the synth's own training
session makes its Z with its own decoder, and what fits this one here is a loss
on control tracks).  The parts are the operators
of :mod:`dgen_hip.sequence`; plain projections are library products.

    python -m dgen_hip.decoder          # fits control tracks, then streams them

``forward`` and ``backward`` train on whole clips (of unequal length, if
wanted); ``step`` takes one frame of every voice and carries its state.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import sequence as Q


@dataclass
class DecoderConfig:
    features: int = 2      # f0 and loudness, as HarmonicConfig.din
    controls: int = 127    # HarmonicConfig.NC
    hidden: int = 512
    inner: int = 1024      # channels of the convolution and the scan
    states: int = 16
    window: int = 4
    rank: int = 32         # of the step's projection
    mlp: int = 1408
    blocks: int = 2
    activation: str = "silu"
    dtype: torch.dtype = torch.bfloat16  # of activations and projections
    seed: int = 5


def _mm(x, w):
    """x [..., k] times w [k][n]."""
    return (x.reshape(-1, x.shape[-1]) @ w).view(*x.shape[:-1], w.shape[1])


def _mm_grads(dy, x, w):
    """Gradients of _mm by x and w."""
    d, f = dy.reshape(-1, dy.shape[-1]), x.reshape(-1, x.shape[-1])
    return (d @ w.t()).view(x.shape), f.t() @ d


class RecurrentDecoder:
    """Parameters (``params``, by name) and passes of the decoder."""

    def __init__(self, cfg: DecoderConfig = DecoderConfig(), device: str | torch.device = "cuda"):
        self.cfg, self.device = cfg, torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        g = torch.Generator().manual_seed(cfg.seed)
        f32, ty, D, E, N = torch.float32, cfg.dtype, cfg.hidden, cfg.inner, cfg.states
        self.params: dict[str, torch.Tensor] = {}

        def put(name, t, dtype):
            self.params[name] = t.to(device=self.device, dtype=dtype)

        def linear(name, k, n, gain=1.0):
            put(name, torch.randn(k, n, generator=g) * (gain / math.sqrt(k)), ty)

        linear("in", cfg.features, D)
        for i in range(cfg.blocks):
            p = f"{i}."
            put(p + "norm1", torch.ones(D), f32)
            linear(p + "xz", D, 2 * E)
            put(p + "conv", (torch.rand(E, cfg.window, generator=g) * 2 - 1) / math.sqrt(cfg.window), f32)
            put(p + "conv_bias", torch.zeros(E), f32)
            linear(p + "proj", E, cfg.rank + 2 * N)
            linear(p + "dt", cfg.rank, E)
            step = torch.exp(torch.rand(E, generator=g) * math.log(100.0) + math.log(1e-3))  # 1e-3 .. 0.1
            put(p + "dt_bias", step + torch.log(-torch.expm1(-step)), f32)
            put(p + "log_A", torch.log(torch.arange(1, N + 1, dtype=f32)).repeat(E, 1), f32)
            put(p + "D", torch.ones(E), f32)
            linear(p + "out", E, D, 1 / math.sqrt(2 * cfg.blocks))
            put(p + "norm2", torch.ones(D), f32)
            linear(p + "gate", D, cfg.mlp)
            linear(p + "up", D, cfg.mlp)
            linear(p + "down", cfg.mlp, D, 1 / math.sqrt(2 * cfg.blocks))
        put("norm", torch.ones(D), f32)
        linear("heads", D, cfg.controls)
        put("heads_bias", torch.zeros(cfg.controls), f32)

    # ------------------------------------------------------------- passes
    def state(self, voices: int) -> list[tuple[torch.Tensor, torch.Tensor]]:
        """Zero state of ``voices`` sequences: per block, the convolution's
        frames and the scan's states."""
        c = self.cfg
        return [(torch.zeros(voices, c.window - 1, c.inner, dtype=c.dtype, device=self.device),
                 torch.zeros(voices, c.inner, c.states, device=self.device)) for _ in range(c.blocks)]

    def forward(self, x, lengths=None, state=None, keep: bool = False):
        """Head pre-activations [batch][frames][controls] (float32) of features
        [batch][frames][features].  ``state`` (from :meth:`state`) is read and
        moved on; with ``keep`` the result is (Z, saved) for :meth:`backward`,
        to which the state counts as given (a copy of it is kept).  Frames past
        a clip's end pass through the parts that see one frame at a time, as any
        others: a program pads with finite features and gives them no gradient."""
        c, P = self.cfg, self.params
        if x.dim() != 3 or x.shape[2] != c.features:
            raise ValueError(f"features: [batch][frames][{c.features}] expected, got {tuple(x.shape)}")
        x = x.to(device=self.device, dtype=c.dtype)
        r = _mm(x, P["in"]).float()
        h = torch.zeros_like(r, dtype=c.dtype)
        saved = []
        for i in range(c.blocks):
            p = f"{i}."
            y1, r1 = Q.rms_norm(h, P[p + "norm1"], residual=r)
            xz = _mm(y1, P[p + "xz"])
            u, z = xz[..., :c.inner], xz[..., c.inner:]
            conv, scan = (None, None) if state is None else state[i]
            start = (conv, scan)
            if keep and state is not None:  # (the calls below move it on in place)
                start = (conv.clone(), scan.clone())
            v = Q.causal_conv(u, P[p + "conv"], P[p + "conv_bias"], state=conv, state_out=conv, lengths=lengths)
            q = _mm(v, P[p + "proj"])
            low, B, C = q[..., :c.rank], q[..., c.rank:c.rank + c.states], q[..., c.rank + c.states:]
            dt = _mm(low, P[p + "dt"])
            A = -torch.exp(P[p + "log_A"])
            s = Q.selective_scan(v, dt, A, B, C, D=P[p + "D"], z=z, dt_bias=P[p + "dt_bias"], state=scan,
                                 state_out=scan, lengths=lengths)
            y2, r = Q.rms_norm(_mm(s, P[p + "out"]), P[p + "norm2"], residual=r1)
            g = Q.gated_mlp(y2, P[p + "gate"], P[p + "up"], activation=c.activation)
            h = _mm(g, P[p + "down"])
            if keep:
                saved.append((y1, r1, xz, v, q, dt, A, s, y2, r, g, start))
        y, r = Q.rms_norm(h, P["norm"], residual=r)
        Z = _mm(y, P["heads"]).float() + P["heads_bias"]
        return (Z, (x, lengths, saved, y, r)) if keep else Z

    def backward(self, dZ, kept) -> dict[str, torch.Tensor]:
        """Gradients of every parameter, by name (float32), from those of Z."""
        c, P, G = self.cfg, self.params, {}
        x, lengths, saved, y, r = kept
        G["heads_bias"] = dZ.sum((0, 1))
        dy, G["heads"] = _mm_grads(dZ.to(c.dtype), y, P["heads"])
        dr, G["norm"] = Q.rms_norm_backward(dy, r, P["norm"])
        for i in reversed(range(c.blocks)):
            p = f"{i}."
            y1, r1, xz, v, q, dt, A, s, y2, r2, g, (conv, scan) = saved[i]
            # dr: of the stream after the block, hence of its last branch too
            dg, G[p + "down"] = _mm_grads(dr.to(c.dtype), g, P[p + "down"])
            dy2, G[p + "gate"], G[p + "up"] = Q.gated_mlp_backward(dg, y2, P[p + "gate"], P[p + "up"],
                                                                   activation=c.activation)
            dr, G[p + "norm2"] = Q.rms_norm_backward(dy2, r2, P[p + "norm2"], ds=dr)
            ds, G[p + "out"] = _mm_grads(dr.to(c.dtype), s, P[p + "out"])
            low, B, C = q[..., :c.rank], q[..., c.rank:c.rank + c.states], q[..., c.rank + c.states:]
            t = Q.selective_scan_backward(ds, v, dt, A, B, C, D=P[p + "D"], z=xz[..., c.inner:],
                                          dt_bias=P[p + "dt_bias"], state=scan, lengths=lengths)
            G[p + "log_A"], G[p + "D"], G[p + "dt_bias"] = t.dA * A, t.dD, t.ddt_bias
            dlow, G[p + "dt"] = _mm_grads(t.ddt, low, P[p + "dt"])
            dv, G[p + "proj"] = _mm_grads(torch.cat([dlow, t.dB, t.dC], -1), v, P[p + "proj"])
            du, G[p + "conv"], G[p + "conv_bias"] = Q.causal_conv_backward(
                dv + t.dx, xz[..., :c.inner], P[p + "conv"], P[p + "conv_bias"], state=conv, lengths=lengths)
            dy1, G[p + "xz"] = _mm_grads(torch.cat([du, t.dz], -1), y1, P[p + "xz"])
            dr, G[p + "norm1"] = Q.rms_norm_backward(dy1, r1, P[p + "norm1"], ds=dr)
        _, G["in"] = _mm_grads(dr.to(c.dtype), x, P["in"])
        return {k: G[k].float() for k in P}

    def step(self, frame, state):
        """One frame [voices][features] of every voice: Z [voices][controls];
        ``state`` moves on in place."""
        return self.forward(frame[:, None], state=state)[:, 0]


def fit(decoder: RecurrentDecoder, x, target, steps: int, lr: float = 1e-3, lengths=None) -> list[float]:
    """Adam on the mean squared error of Z over the sequences' own frames
    (``lengths``: on the host or the device; what lies past a sequence's end
    may be anything); the losses of the steps.  Parameters are kept in 32 bits
    and rounded to their own type for each pass."""
    master = {k: v.float().clone().requires_grad_() for k, v in decoder.params.items()}
    opt = torch.optim.Adam(master.values(), lr=lr)
    inside, count = None, target.numel()
    if lengths is not None:
        lengths = lengths.to(device=decoder.device, dtype=torch.int32)
        x = x.to(decoder.device)
        inside = (torch.arange(x.shape[1], device=decoder.device) < lengths[:, None])[..., None]
        # (padded frames pass through the frame-wise parts: with finite values and no gradient they count for nothing)
        x = torch.where(inside, x, 0.0)
        count = max(1, int(inside.sum())) * target.shape[2]
    losses = []
    for _ in range(steps):
        Z, kept = decoder.forward(x, lengths=lengths, keep=True)
        d = Z - target
        if inside is not None:
            d = torch.where(inside, d, 0.0)
        losses.append(float(d.square().sum() / count))
        grads = decoder.backward(d * (2.0 / count), kept)
        for k, p in master.items():
            p.grad = grads[k]
        opt.step()
        with torch.no_grad():
            for k, p in master.items():
                decoder.params[k].copy_(p)
    return losses


def main() -> None:
    """Fits a decoder to synthetic control tracks that lag behind the features
    (an envelope follower of the loudness, which no frame alone determines),
    then renders them frame by frame and compares with the whole clips."""
    voices, frames = 8, 500
    dec = RecurrentDecoder(DecoderConfig(controls=16, hidden=128, inner=256, mlp=352, rank=8))
    g = torch.Generator().manual_seed(3)
    t = torch.arange(frames)[None] / frames
    loud = 0.5 + 0.5 * torch.sin(2 * math.pi * (1 + 3 * torch.rand(voices, 1, generator=g)) * t)
    f0 = torch.rand(voices, 1, generator=g) + 0.1 * torch.sin(2 * math.pi * 5 * t)
    x = torch.stack([f0, loud], -1)
    follow, env = [], torch.zeros(voices)
    for k in range(frames):
        env = env + 0.05 * (loud[:, k] - env)
        follow.append(env)
    env = torch.stack(follow, 1)
    target = torch.stack([env * math.cos(j) + f0 * math.sin(j) for j in range(16)], -1).to(dec.device)
    losses = fit(dec, x, target, steps=200)
    print(f"fit: loss {losses[0]:.4f} -> {losses[-1]:.6f} in {len(losses)} steps")
    whole, state = dec.forward(x), dec.state(voices)
    frames_out = torch.stack([dec.step(x[:, k], state) for k in range(frames)], 1)
    print(f"stream: {frames} single frames of {voices} voices, largest difference to the whole clips "
          f"{float((frames_out - whole).abs().max()):.2e}")


if __name__ == "__main__":
    main()
