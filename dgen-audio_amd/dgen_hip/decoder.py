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

Two things may be otherwise.  With ``mixer`` "delta" the first branch is

    norm -> projection to (q, k, v), causal convolution; projection to (decay,
    strength) -> gated delta rule -> projection back

whose memory of the frames before is overwritten key by key.  With ``around``
every branch ends in a norm, a gate and a scale of the stream of its own
(:func:`dgen_hip.sequence.block_norm`), for stacks of many blocks.

    python -m dgen_hip.decoder          # fits control tracks, then streams them
    python -m dgen_hip.decoder --mixer delta --around --weight-decay 0.01 --max-norm 1

``forward`` and ``backward`` train on whole clips (of unequal length, if
wanted); ``step`` takes one frame of every voice and carries its state.
"""
from __future__ import annotations

import argparse
import math
from dataclasses import dataclass

import torch

from . import optim
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
    mixer: str = "scan"    # or "delta"
    around: bool = False   # norms, gates and scales around the branches
    heads: int = 8         # of the delta rule: of its values,
    key_heads: int = 4     # of its keys and queries,
    key: int = 64          # channels of each of these


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

        if cfg.mixer not in ("scan", "delta"):
            raise ValueError(f"mixer {cfg.mixer!r}: one of ['delta', 'scan']")
        if cfg.mixer == "delta":
            if min(cfg.heads, cfg.key_heads) < 1 or E % cfg.heads or cfg.heads % cfg.key_heads:
                raise ValueError(f"{E} channels, {cfg.heads} heads, {cfg.key_heads} key heads: each divides the one before")
            if not 1 <= cfg.key <= 128 or not 1 <= E // cfg.heads <= 1024:
                raise ValueError(f"{cfg.key} channels of a key head, {E // cfg.heads} of a head: 1 to 128 and 1 to 1024")

        def back(name, k):
            """A branch's projection to the stream; with a gate beside it, a norm
            and the stream's scale."""
            linear(name, k, 2 * D if cfg.around else D, 1 / math.sqrt(2 * cfg.blocks))
            if cfg.around:
                put(name + "_norm", torch.full((D,), 1 / math.sqrt(2 * cfg.blocks)), f32)
                put(name + "_scale", torch.ones(D), f32)

        def steps(n):
            """Biases whose softplus lies between 1e-3 and 0.1."""
            step = torch.exp(torch.rand(n, generator=g) * math.log(100.0) + math.log(1e-3))
            return step + torch.log(-torch.expm1(-step))

        linear("in", cfg.features, D)
        for i in range(cfg.blocks):
            p = f"{i}."
            put(p + "norm1", torch.ones(D), f32)
            ch = E if cfg.mixer == "scan" else 2 * cfg.key_heads * cfg.key + E  # of the convolution
            linear(p + "xz", D, 2 * E if cfg.mixer == "scan" else ch)
            put(p + "conv", (torch.rand(ch, cfg.window, generator=g) * 2 - 1) / math.sqrt(cfg.window), f32)
            put(p + "conv_bias", torch.zeros(ch), f32)
            if cfg.mixer == "scan":
                linear(p + "proj", E, cfg.rank + 2 * N)
                linear(p + "dt", cfg.rank, E)
                put(p + "dt_bias", steps(E), f32)
                put(p + "log_A", torch.log(torch.arange(1, N + 1, dtype=f32)).repeat(E, 1), f32)
                put(p + "D", torch.ones(E), f32)
            else:
                linear(p + "ab", D, 2 * cfg.heads)
                put(p + "dt_bias", steps(cfg.heads), f32)
                put(p + "log_A", torch.zeros(cfg.heads), f32)
            back(p + "out", E)
            put(p + "norm2", torch.ones(D), f32)
            linear(p + "gate", D, cfg.mlp)
            linear(p + "up", D, cfg.mlp)
            back(p + "down", cfg.mlp)
        put("norm", torch.ones(D), f32)
        linear("heads", D, cfg.controls)
        put("heads_bias", torch.zeros(cfg.controls), f32)

    # ------------------------------------------------------------- passes
    def state(self, voices: int) -> list[tuple[torch.Tensor, torch.Tensor]]:
        """Zero state of ``voices`` sequences: per block, the convolution's
        frames and the scan's states or the delta rule's memory."""
        c = self.cfg
        ch, memory = c.inner, (c.inner, c.states)
        if c.mixer == "delta":
            ch, memory = 2 * c.key_heads * c.key + c.inner, (c.heads, c.key, c.inner // c.heads)
        return [(torch.zeros(voices, c.window - 1, ch, dtype=c.dtype, device=self.device),
                 torch.zeros(voices, *memory, device=self.device)) for _ in range(c.blocks)]

    def _join(self, h, r, branch, norm):
        """The stream after a branch's output h, and the next branch's input."""
        P, D = self.params, self.cfg.hidden
        if branch is None or not self.cfg.around:
            return Q.rms_norm(h, P[norm], residual=r)
        return Q.block_norm(h[..., :D], P[branch + "_norm"], r, P[norm], gate=h[..., D:], residual_scale=P[branch + "_scale"])

    def _join_backward(self, dy, dr, h, r, s, branch, norm, G):
        """(gradient of the stream before, of h): dr is the gradient that
        reaches the stream s after the join from elsewhere (None: nothing)."""
        P, D = self.params, self.cfg.hidden
        if branch is None or not self.cfg.around:
            dr, G[norm] = Q.rms_norm_backward(dy, s, P[norm], ds=dr)
            return dr, dr.to(self.cfg.dtype)
        t = Q.block_norm_backward(dy, h[..., :D], r, s, P[branch + "_norm"], P[norm], gate=h[..., D:],
                                  residual_scale=P[branch + "_scale"], ds=dr)
        G[norm], G[branch + "_norm"], G[branch + "_scale"] = t.dpre, t.dpost, t.dresidual_scale
        return t.dresidual, torch.cat([t.dx, t.dgate], -1)

    def _heads(self, v):
        """Queries, keys and values of the convolution's channels."""
        c = self.cfg
        n = c.key_heads * c.key
        return (v[..., :n].unflatten(-1, (c.key_heads, c.key)), v[..., n:2 * n].unflatten(-1, (c.key_heads, c.key)),
                v[..., 2 * n:].unflatten(-1, (c.heads, c.inner // c.heads)))

    def _scan(self, p, y, state, memory, lengths):
        """The scan's branch up to its projection back: (result, what its
        gradient takes)."""
        c, P = self.cfg, self.params
        xz = _mm(y, P[p + "xz"])
        u, z = xz[..., :c.inner], xz[..., c.inner:]
        v = Q.causal_conv(u, P[p + "conv"], P[p + "conv_bias"], state=state, state_out=state, lengths=lengths)
        q = _mm(v, P[p + "proj"])
        low, B, C = q[..., :c.rank], q[..., c.rank:c.rank + c.states], q[..., c.rank + c.states:]
        dt = _mm(low, P[p + "dt"])
        A = -torch.exp(P[p + "log_A"])
        s = Q.selective_scan(v, dt, A, B, C, D=P[p + "D"], z=z, dt_bias=P[p + "dt_bias"], state=memory, state_out=memory,
                             lengths=lengths)
        return s, (xz, v, q, dt, A)

    def _scan_backward(self, p, ds, y, kept, state, memory, lengths, G):
        c, P = self.cfg, self.params
        xz, v, q, dt, A = kept
        low, B, C = q[..., :c.rank], q[..., c.rank:c.rank + c.states], q[..., c.rank + c.states:]
        t = Q.selective_scan_backward(ds, v, dt, A, B, C, D=P[p + "D"], z=xz[..., c.inner:], dt_bias=P[p + "dt_bias"],
                                      state=memory, lengths=lengths)
        G[p + "log_A"], G[p + "D"], G[p + "dt_bias"] = t.dA * A, t.dD, t.ddt_bias
        dlow, G[p + "dt"] = _mm_grads(t.ddt, low, P[p + "dt"])
        dv, G[p + "proj"] = _mm_grads(torch.cat([dlow, t.dB, t.dC], -1), v, P[p + "proj"])
        du, G[p + "conv"], G[p + "conv_bias"] = Q.causal_conv_backward(
            dv + t.dx, xz[..., :c.inner], P[p + "conv"], P[p + "conv_bias"], state=state, lengths=lengths)
        dy, G[p + "xz"] = _mm_grads(torch.cat([du, t.dz], -1), y, P[p + "xz"])
        return dy

    def _delta(self, p, y, state, memory, lengths):
        """The same of the delta rule's."""
        c, P = self.cfg, self.params
        u = _mm(y, P[p + "xz"])
        v = Q.causal_conv(u, P[p + "conv"], P[p + "conv_bias"], state=state, state_out=state, lengths=lengths)
        ab = _mm(y, P[p + "ab"]).float()
        g = -torch.exp(P[p + "log_A"]) * torch.nn.functional.softplus(ab[..., :c.heads] + P[p + "dt_bias"])
        beta = torch.sigmoid(ab[..., c.heads:])
        s = Q.gated_delta_rule(*self._heads(v), g, beta, state=memory, state_out=memory, lengths=lengths)
        return s.flatten(2), (u, v, ab, g, beta)

    def _delta_backward(self, p, ds, y, kept, state, memory, lengths, G):
        c, P = self.cfg, self.params
        u, v, ab, g, beta = kept
        t = Q.gated_delta_rule_backward(ds.unflatten(-1, (c.heads, c.inner // c.heads)), *self._heads(v), g, beta, state=memory,
                                        lengths=lengths)
        # (a gate that lets nothing through has no gradient, however steep the way to it: -infinity's is not 0 times that)
        shut = t.dg == 0
        da = torch.where(shut, 0.0, -t.dg * torch.exp(P[p + "log_A"]) * torch.sigmoid(ab[..., :c.heads] + P[p + "dt_bias"]))
        G[p + "log_A"], G[p + "dt_bias"] = torch.where(shut, 0.0, t.dg * g).sum((0, 1)), da.sum((0, 1))
        dy, G[p + "ab"] = _mm_grads(torch.cat([da, t.dbeta * beta * (1 - beta)], -1).to(c.dtype), y, P[p + "ab"])
        du, G[p + "conv"], G[p + "conv_bias"] = Q.causal_conv_backward(
            torch.cat([t.dq.flatten(2), t.dk.flatten(2), t.dv.flatten(2)], -1), u, P[p + "conv"], P[p + "conv_bias"],
            state=state, lengths=lengths)
        dyu, G[p + "xz"] = _mm_grads(du, y, P[p + "xz"])
        return dy + dyu

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
        h, branch = torch.zeros_like(r, dtype=c.dtype), None
        mixer = self._scan if c.mixer == "scan" else self._delta
        saved = []
        for i in range(c.blocks):
            p = f"{i}."
            y1, r1 = self._join(h, r, branch, p + "norm1")
            conv, memory = (None, None) if state is None else state[i]
            start = (conv, memory)
            if keep and state is not None:  # (the calls below move it on in place)
                start = (conv.clone(), memory.clone())
            s, kept = mixer(p, y1, conv, memory, lengths)
            # (what went into a join is kept where its gradient reads it)
            h2, entering = _mm(s, P[p + "out"]), (h, r) if c.around and branch else (None, None)
            y2, r = self._join(h2, r1, p + "out", p + "norm2")
            g = Q.gated_mlp(y2, P[p + "gate"], P[p + "up"], activation=c.activation)
            h, branch = _mm(g, P[p + "down"]), p + "down"
            if keep:
                saved.append((*entering, y1, r1, s, kept, h2 if c.around else None, y2, r, g, start))
        y, last = self._join(h, r, branch, "norm")
        Z = _mm(y, P["heads"]).float() + P["heads_bias"]
        if not c.around:
            h = r = None
        return (Z, (x, lengths, saved, h, r, y, last)) if keep else Z

    def backward(self, dZ, kept) -> dict[str, torch.Tensor]:
        """Gradients of every parameter, by name (float32), from those of Z."""
        c, P, G = self.cfg, self.params, {}
        x, lengths, saved, h, r, y, last = kept
        mixer = self._scan_backward if c.mixer == "scan" else self._delta_backward
        G["heads_bias"] = dZ.sum((0, 1))
        dy, G["heads"] = _mm_grads(dZ.to(c.dtype), y, P["heads"])
        # dr: of the stream; dh: of the branch that ends in it
        dr, dh = self._join_backward(dy, None, h, r, last, f"{c.blocks - 1}.down" if c.blocks else None, "norm", G)
        for i in reversed(range(c.blocks)):
            p = f"{i}."
            before, r0, y1, r1, s, kept, h2, y2, r2, g, (conv, memory) = saved[i]
            dg, G[p + "down"] = _mm_grads(dh, g, P[p + "down"])
            dy2, G[p + "gate"], G[p + "up"] = Q.gated_mlp_backward(dg, y2, P[p + "gate"], P[p + "up"],
                                                                   activation=c.activation)
            dr, dh = self._join_backward(dy2, dr, h2, r1, r2, p + "out", p + "norm2", G)
            ds, G[p + "out"] = _mm_grads(dh, s, P[p + "out"])
            dy1 = mixer(p, ds, y1, kept, conv, memory, lengths, G)
            dr, dh = self._join_backward(dy1, dr, before, r0, r1, f"{i - 1}.down" if i else None, p + "norm1", G)
        _, G["in"] = _mm_grads(dr.to(c.dtype), x, P["in"])
        return {k: G[k].float() for k in P}

    def step(self, frame, state):
        """One frame [voices][features] of every voice: Z [voices][controls];
        ``state`` moves on in place."""
        return self.forward(frame[:, None], state=state)[:, 0]


def fit(decoder: RecurrentDecoder, x, target, steps: int, lr: float = 1e-3, lengths=None, weight_decay: float | None = None,
        max_norm: float | None = None) -> list[float]:
    """Adam on the mean squared error of Z over the sequences' own frames
    (``lengths``: on the host or the device; what lies past a sequence's end
    may be anything); the losses of the steps.  Parameters are kept in 32 bits
    and rounded to their own type for each pass.  With ``weight_decay`` or
    ``max_norm`` (of all gradients) the steps are those of
    :class:`dgen_hip.optim.AdamW`, whose decay takes every parameter alike: norms'
    weights, scales, biases and the mixers' decays and steps too."""
    own = None
    if weight_decay is None and max_norm is None:
        master = {k: v.float().clone().requires_grad_() for k, v in decoder.params.items()}
        opt = torch.optim.Adam(master.values(), lr=lr)
    else:
        names = list(decoder.params)
        half = [v if v.dtype is torch.bfloat16 else None for v in decoder.params.values()]
        own = optim.AdamW([v.float() for v in decoder.params.values()], lr=lr, weight_decay=weight_decay or 0.0,
                          max_norm=max_norm, copies=half)
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
        if own is not None:
            own.step([grads[k] for k in names])
            continue
        for k, p in master.items():
            p.grad = grads[k]
        opt.step()
        with torch.no_grad():
            for k, p in master.items():
                decoder.params[k].copy_(p)
    return losses


def main(args: list[str] | None = None) -> None:
    """Fits a decoder to synthetic control tracks that lag behind the features
    (an envelope follower of the loudness, which no frame alone determines),
    then renders them frame by frame and compares with the whole clips."""
    ap = argparse.ArgumentParser(description=main.__doc__)
    ap.add_argument("--mixer", choices=("scan", "delta"), default="scan")
    ap.add_argument("--around", action="store_true", help="norms, gates and scales around the branches")
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--weight-decay", type=float, default=None)
    ap.add_argument("--max-norm", type=float, default=None)
    a = ap.parse_args(args)
    voices, frames = 8, 500
    dec = RecurrentDecoder(DecoderConfig(controls=16, hidden=128, inner=256, mlp=352, rank=8, mixer=a.mixer, around=a.around,
                                         heads=4, key_heads=2, key=32))
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
    losses = fit(dec, x, target, steps=a.steps, weight_decay=a.weight_decay, max_norm=a.max_norm)
    print(f"fit: loss {losses[0]:.4f} -> {losses[-1]:.6f} in {len(losses)} steps")
    whole, state = dec.forward(x), dec.state(voices)
    frames_out = torch.stack([dec.step(x[:, k], state) for k in range(frames)], 1)
    print(f"stream: {frames} single frames of {voices} voices, largest difference to the whole clips "
          f"{float((frames_out - whole).abs().max()):.2e}")


if __name__ == "__main__":
    main()
