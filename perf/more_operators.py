"""More operators of the recurrent control decoder as a program calls them, in
training (whole clips, gradients, the optimiser's step) and in rendering (clips
of unequal length, one control frame at a time).

- ``delta``: gated delta rule, a matrix-valued memory per head
- ``block``: the norm after a block, its gate, the residual's scale and addition
  and the norm before the next block
- ``adamw``: one AdamW step over all of a model's tensors

With ``own`` false, ``run`` computes them from elementary torch operations in
32 bits (the decays' running sums in 64), rounded once at the end; with ``own``
true it calls the framework.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

EPS = 1e-5
UNIT_EPS = 1e-6  # of the keys' and queries' norms
CHUNK = 64
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # a live voice bank: one new control frame for 32 voices; the memory's
        # reading and writing counts
        dict(name="delta_step", kind="delta", back=False, B=32, T=1, heads=8, shared=1, K=128, V=128, type="fp32",
             ragged=False, state=True),
        # rendering a few clips of unequal length, keys shared by three heads,
        # odd sizes
        dict(name="delta_ragged", kind="delta", back=False, B=7, T=777, heads=6, shared=3, K=40, V=77, type="bf16",
             ragged=True, state=True),
        # a training batch, 32 clips of 1000 control frames, 1024 channels
        dict(name="delta_forward", kind="delta", back=False, B=32, T=1000, heads=8, shared=1, K=128, V=128, type="bf16",
             ragged=False, state=False),
        # its gradients
        dict(name="delta_backward", kind="delta", back=True, B=32, T=1000, heads=8, shared=1, K=128, V=128, type="bf16",
             ragged=False, state=False),
        # one long signal at audio rate: few heads, long axis
        dict(name="delta_long", kind="delta", back=False, B=1, T=65536, heads=4, shared=1, K=64, V=64, type="fp32",
             ragged=False, state=False),
        # gradients of three short clips of unequal length, shared keys, odd sizes
        dict(name="delta_backward_odd", kind="delta", back=True, B=3, T=1001, heads=6, shared=2, K=33, V=50, type="fp32",
             ragged=True, state=False),
        # one control frame of 32 voices
        dict(name="block_step", kind="block", back=False, B=32, T=1, width=512, type="bf16", res="fp32", gate="rows",
             scale=True),
        # the residual stream of a training batch, kept in 32 bits beside bf16
        # activations, gated frame by frame
        dict(name="block_forward", kind="block", back=False, B=32, T=1000, width=512, type="bf16", res="fp32",
             gate="rows", scale=True),
        # its gradients, with one gate for each clip
        dict(name="block_backward", kind="block", back=True, B=32, T=1000, width=512, type="bf16", res="fp32",
             gate="clips", scale=True),
        # gradients of odd sizes in 32 bits
        dict(name="block_backward_odd", kind="block", back=True, B=3, T=1333, width=1023, type="fp32", res="fp32",
             gate="rows", scale=True),
        # the decoder's default sizes: 34 tensors, many of them small
        dict(name="adamw_decoder", kind="adamw", hidden=512, inner=1024, mlp=1408, blocks=2, states=16, grad="fp32",
             copies=True, clip=False),
        # a decoder of 240 M parameters, gradients of the activations' type, with
        # the gradients' norm held to a bound
        dict(name="adamw_large", kind="adamw", hidden=2048, inner=4096, mlp=5632, blocks=4, states=16, grad="bf16",
             copies=True, clip=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["delta", "delta", "delta", "block", "adamw"])
    back, t = rng.random() < 0.5, rng.choice(["fp32", "bf16"])
    if kind == "adamw":
        return dict(kind=kind, hidden=_log(rng, 16, 1500), inner=_log(rng, 16, 3000), mlp=_log(rng, 16, 4000),
                    blocks=rng.choice([1, 2, 3, 4]), states=rng.choice([4, 12, 16]), grad=t,
                    copies=rng.random() < 0.5, clip=rng.random() < 0.5)
    T = 1 if not back and rng.random() < 0.25 else _log(rng, 2, 65536)
    if kind == "block":
        width = _log(rng, 16, 2048)
        B = max(1, min(_log(rng, 1, 48), 16_000_000 // (T * width)))
        return dict(kind=kind, back=back, B=B, T=min(T, 16_000_000 // width), width=width, type=t,
                    res=rng.choice(["fp32", t]), gate=rng.choice(["none", "rows", "clips"]), scale=rng.random() < 0.5)
    K, V, shared = _log(rng, 8, 128), _log(rng, 8, 160), rng.choice([1, 1, 2, 3])
    if rng.random() < 0.5:
        K, V = -(-K // 32) * 32, -(-V // 32) * 32
    most = (8_000_000 if back else 32_000_000) // max(K, V)  # frames and heads
    heads = shared * max(1, min(_log(rng, 1, 8), most // (T * shared)))
    B = max(1, min(_log(rng, 1, 48), most // (T * heads)))
    return dict(kind=kind, back=back, B=B, T=T, heads=heads, shared=shared, K=K, V=V, type=t,
                ragged=T > 1 and rng.random() < 0.4, state=T == 1 or rng.random() < 0.3)


# ------------------------------------------------------------------ inputs
def _shapes(case):
    """The tensors of a decoder of these sizes."""
    D, E, M, N, R = case["hidden"], case["inner"], case["mlp"], case["states"], 32
    block = [(D,), (D, 2 * E), (E, 4), (E,), (E, R + 2 * N), (R, E), (E,), (E, N), (E,), (E, D), (D,), (D, M), (D, M),
             (M, D)]
    return [(2, D), *block * case["blocks"], (D,), (D, 127), (127,)]


def _inputs(case, seed):
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    g = torch.Generator(device=dev)
    g.manual_seed((int(seed) * 1000003 + sum(map(ord, case["kind"]))) & 0x7FFFFFFF)

    def normal(*shape, scale=1.0, type=torch.float32):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(type)

    def uniform(*shape, lo=0.0, hi=1.0):
        return torch.rand(*shape, generator=g, device=dev) * (hi - lo) + lo

    if case["kind"] == "adamw":
        shapes = _shapes(case)
        n = sum(map(math.prod, shapes))
        # (a thousand steps in: moments of the gradients' size)
        return dict(params=normal(n, scale=0.05), m=normal(n, scale=1e-4), v=uniform(n, hi=1e-6).square() * 1e6,
                    grads=[normal(*s, scale=1e-3, type=TYPES[case["grad"]]) for s in shapes])
    ty, B, T = TYPES[case["type"]], case["B"], case["T"]
    if case["kind"] == "block":
        n, rt = case["width"], TYPES[case["res"]]
        d = dict(x=normal(B, T, n, type=ty), residual=normal(B, T, n, scale=2.0, type=rt), gate=None, scale=None,
                 post=uniform(n, lo=0.5, hi=1.5), pre=uniform(n, lo=0.5, hi=1.5))
        if case["gate"] != "none":
            d["gate"] = normal(B, T if case["gate"] == "rows" else 1, n, type=ty)
        if case["scale"]:
            d["scale"] = uniform(n, lo=0.8, hi=1.2)
        if case["back"]:
            # (s: the sum that the forward pass handed on)
            d.update(dy=normal(B, T, n, type=ty), ds=normal(B, T, n, type=rt), s=_block_sum(d)[0].to(rt))
        return d
    H, G, K, V = case["heads"], case["heads"] // case["shared"], case["K"], case["V"]
    # queries, keys and values are parts of one projection's output, decays and
    # write strengths of another's
    qkv = normal(B, T, 2 * G * K + H * V, type=ty)
    rate = torch.exp(uniform(H, lo=math.log(1e-3), hi=math.log(0.5)))
    d = dict(q=qkv[..., :G * K].unflatten(-1, (G, K)), k=qkv[..., G * K:2 * G * K].unflatten(-1, (G, K)),
             v=qkv[..., 2 * G * K:].unflatten(-1, (H, V)), g=-rate * torch.exp(normal(B, T, H, scale=0.5)),
             beta=torch.sigmoid(normal(B, T, H)), lengths=None, state=None)
    if case["ragged"]:
        d["lengths"] = torch.randint(0, T + 1, (B,), generator=g, device=dev, dtype=torch.int32)
    if case["state"]:
        d["state"] = normal(B, H, K, V, scale=0.3)
    if case["back"]:
        d["dy"] = normal(B, T, H, V, type=ty)
    return d


ADAMW = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
ADAMW_STEP = 1000


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if case["kind"] == "adamw":
        # the tensors are views of one buffer, the results go to a second one (a
        # program that can take a step back keeps two); the copies are what the
        # next pass multiplies with
        sizes = [math.prod(x) for x in _shapes(case)]
        for k in ("params", "m", "v"):
            s[k + "_out"] = torch.empty_like(s[k])
        s["copies"] = torch.empty_like(s["params"], dtype=torch.bfloat16) if case["copies"] else None
        for k in ("params", "m", "v", "params_out", "m_out", "v_out", "copies"):
            if s[k] is not None:
                s[k + "_list"] = [t.view(x) for t, x in zip(s[k].split(sizes), _shapes(case))]
    elif case["kind"] == "delta" and not case["back"]:
        s["state_out"] = torch.empty(case["B"], case["heads"], case["K"], case["V"], device=s["q"].device)
    return s


# ------------------------------------------------------------- plain forms
def _unit(x):
    """x over its length, and what it was multiplied by."""
    r = torch.rsqrt((x * x).sum(-1, keepdim=True) + UNIT_EPS)
    return x * r, r


def _inverse(A):
    """(I + A)^-1 of strictly lower triangular A, by blocks of twice the size."""
    at = torch.arange(A.shape[-1], device=A.device)
    X, n = torch.eye(A.shape[-1], device=A.device).expand_as(A), 1
    while n < A.shape[-1]:
        low = (at[:, None] // (2 * n) == at // (2 * n)) & (at[:, None] // n != at // n)
        X = X - X @ torch.where(low, A, 0.0) @ X
        n *= 2
    return X


def _affine(P, E):
    """S[c] = P[c] S[c-1] + E[c] along axis 2, S[-1] = 0, by doubling."""
    n = 1
    while n < P.shape[2]:
        E = torch.cat([E[:, :, :n], E[:, :, n:] + P[:, :, n:] @ E[:, :, :-n]], 2)
        P = torch.cat([P[:, :, :n], P[:, :, n:] @ P[:, :, :-n]], 2)
        n *= 2
    return E


def _delta_frame(s):
    """One frame."""
    shared, first = s["case"]["shared"], s["state"]
    (q, _), (k, _) = (_unit(s[x][:, 0].float().repeat_interleave(shared, 1)[..., None].mT) for x in "qk")
    S = torch.exp(s["g"][:, 0])[..., None, None] * first
    S = S + k.mT * (s["beta"][:, 0, :, None, None] * (s["v"][:, 0, :, None].float() - k @ S))
    return dict(y=(q * s["case"]["K"] ** -0.5 @ S).transpose(1, 2).to(s["v"].dtype), state=S)


def _delta_plain(s):
    """Chunks of frames: within one, the frames' writes solve a triangular
    system; between them, the memory is an affine function of the entering one."""
    c, v = s["case"], s["v"]
    if c["T"] == 1 and c["state"] and not c["ragged"] and not c["back"]:
        return _delta_frame(s)
    B, T, H, V = v.shape
    K, ty, shared = c["K"], v.dtype, c["shared"]
    C, N = CHUNK, -(-T // CHUNK)
    n = torch.full((B,), T, device=v.device) if s["lengths"] is None else s["lengths"].long()
    ok = torch.arange(T, device=v.device) < n[:, None]

    def cut(x, heads=1):
        """[B][T][heads][.] to [B][H][N][C][.], 0 behind the sequences."""
        x = torch.where(ok[..., None, None], x.float(), 0.0)
        x = torch.cat([x, x.new_zeros(B, N * C - T, *x.shape[2:])], 1)
        x = x.repeat_interleave(heads, 2) if heads > 1 else x
        return x.unflatten(1, (N, C)).permute(0, 3, 1, 2, 4)

    def joined(x):
        return x.permute(0, 2, 3, 1, 4).reshape(B, N * C, H, -1)[:, :T]

    (q, rq), (k, rk) = (_unit(cut(s[x], shared)) for x in "qk")
    q = q * K ** -0.5
    v, beta = cut(v), cut(s["beta"][..., None])
    G = cut(s["g"][..., None]).double().cumsum(3)
    between = (G - G.mT).float()
    D = torch.where(torch.ones(C, C, device=v.device).tril() > 0, torch.exp(between.clamp(max=0.0)), 0.0)
    into, rest, whole = torch.exp(G.float()), torch.exp((G[..., -1:, :] - G).float()), torch.exp(G[..., -1:, :].float())
    L = ((k @ k.mT) * D).tril(-1)
    X, M = _inverse(beta * L), (q @ k.mT) * D
    kt = (k * rest).mT
    P = whole * torch.eye(K, device=v.device) - kt @ (X @ (beta * into * k))
    E = kt @ (X @ (beta * v))
    first = torch.zeros_like(E[:, :, 0]) if s["state"] is None else s["state"]
    E[:, :, 0] += P[:, :, 0] @ first
    after = _affine(P, E)
    S = torch.cat([first[:, :, None], after[:, :, :-1]], 2)
    U = X @ (beta * (v - into * (k @ S)))
    if not c["back"]:
        return dict(y=joined(into * (q @ S) + M @ U).to(ty), state=after[:, :, -1])
    dy = cut(s["dy"])
    # adjoint of the memory after each chunk
    dE = (into * q).mT @ dy - (beta * into * k).mT @ (X.mT @ (M.mT @ dy))
    dS = _affine(P.mT.flip(2), dE.flip(2)).flip(2)
    dS = torch.cat([dS[:, :, 1:], torch.zeros_like(dS[:, :, :1])], 2)
    dR = X.mT @ (M.mT @ dy + rest * (k @ dS))
    dM, dA = (dy @ U.mT) * D, -((dR @ U.mT) * D).tril(-1)
    dq = into * (dy @ S.mT) + dM @ k
    read = dA @ k - into * (dR @ S.mT)
    write = dM.mT @ q + (beta * dA).mT @ k + rest * (U @ dS.mT)
    dbeta = (dR * v).sum(-1, keepdim=True) + (k * read).sum(-1, keepdim=True)
    at = (q * dq).sum(-1, keepdim=True) + beta * (k * read).sum(-1, keepdim=True) - (k * write).sum(-1, keepdim=True)
    dg = at.flip(3).cumsum(3).flip(3) + (after * dS).sum((-1, -2))[..., None, None]
    dk, dq = beta * read + write, dq * K ** -0.5
    dk = rk * (dk - k * (k * dk).sum(-1, keepdim=True))
    qu = q * K ** 0.5
    dq = rq * (dq - qu * (qu * dq).sum(-1, keepdim=True))
    dq, dk = (joined(t).unflatten(2, (H // shared, shared)).sum(3).to(ty) for t in (dq, dk))
    live = ok[..., None]
    return dict(dq=dq, dk=dk, dv=joined(beta * dR).to(ty), dg=torch.where(live, joined(dg)[..., 0], 0.0),
                dbeta=torch.where(live, joined(dbeta)[..., 0], 0.0))


def _block_sum(s):
    """The new residual, and what it was made of."""
    x, r = s["x"].float(), s["residual"].float()
    gate = 1.0 if s["gate"] is None else 1 / (1 + torch.exp(-s["gate"].float()))
    scale = 1.0 if s["scale"] is None else s["scale"]
    rx = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    n = x * rx
    p = n * s["post"]
    return scale * r + gate * p, r, gate, scale, rx, n, p


def _block_plain(s):
    c = s["case"]
    a, r, gate, scale, rx, n, p = _block_sum(s)
    if not c["back"]:
        ra = torch.rsqrt((a * a).mean(-1, keepdim=True) + EPS)
        return dict(y=(a * ra * s["pre"]).to(s["x"].dtype), s=a.to(s["residual"].dtype))
    a = s["s"].float()
    ra = torch.rsqrt((a * a).mean(-1, keepdim=True) + EPS)
    dy = s["dy"].float()
    na, dn = a * ra, dy * s["pre"]
    da = ra * (dn - na * (dn * na).mean(-1, keepdim=True)) + s["ds"].float()
    dp = da * gate
    dw = dp * s["post"]
    out = dict(dx=(rx * (dw - n * (dw * n).mean(-1, keepdim=True))).to(s["x"].dtype),
               dresidual=(da * scale).to(s["residual"].dtype), dpost=(dp * n).sum((0, 1)), dpre=(dy * na).sum((0, 1)))
    if s["gate"] is not None:
        dgate = da * p * gate * (1 - gate)
        out["dgate"] = (dgate.sum(1, keepdim=True) if c["gate"] == "clips" else dgate).to(s["x"].dtype)
    if s["scale"] is not None:
        out["dscale"] = (da * r).sum((0, 1))
    return out


def _adamw_plain(s):
    c, (b1, b2), t, lr = s["case"], ADAMW["betas"], ADAMW_STEP, ADAMW["lr"]
    g, norm = torch.cat([x.reshape(-1) for x in s["grads"]]).float(), None
    if c["clip"]:
        norm = (g * g).sum().sqrt()
        g = g * (1.0 / (norm + 1e-6)).clamp(max=1.0)
    m = s["m"] * b1 + g * (1 - b1)
    v = s["v"] * b2 + g * g * (1 - b2)
    step = (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + ADAMW["eps"])
    p = s["params"] * (1 - lr * ADAMW["weight_decay"]) - lr * step
    for k, x in (("params_out", p), ("m_out", m), ("v_out", v), ("copies", p)):
        if s[k] is not None:
            s[k].copy_(x)
    return _adamw_results(s, norm)


def _adamw_results(s, norm):
    out = dict(params=s["params_out"], m=s["m_out"], v=s["v_out"])
    if s["copies"] is not None:
        out["copies"] = s["copies"]
    if norm is not None:
        out["norm"] = norm
    return out


PLAIN = {"delta": _delta_plain, "block": _block_plain, "adamw": _adamw_plain}


# ------------------------------------------------------ the framework's calls
def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dgen-audio_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from dgen_hip import optim, sequence
    return sequence, optim


def _delta_own(s):
    q, _ = _package()
    if not s["case"]["back"]:
        y = q.gated_delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], state=s["state"], state_out=s["state_out"],
                               lengths=s["lengths"])
        return dict(y=y, state=s["state_out"])
    return q.gated_delta_rule_backward(s["dy"], s["q"], s["k"], s["v"], s["g"], s["beta"], state=s["state"],
                                       lengths=s["lengths"])._asdict()


def _block_own(s):
    q, _ = _package()
    gate = dict(gate=s["gate"], gate_activation="sigmoid", residual_scale=s["scale"], eps=EPS)
    if not s["case"]["back"]:
        y, a = q.block_norm(s["x"], s["post"], s["residual"], s["pre"], **gate)
        return dict(y=y, s=a)
    r = q.block_norm_backward(s["dy"], s["x"], s["residual"], s["s"], s["post"], s["pre"], ds=s["ds"], **gate)
    out = dict(dx=r.dx, dresidual=r.dresidual, dpost=r.dpost, dpre=r.dpre)
    if r.dgate is not None:
        out["dgate"] = r.dgate
    if r.dresidual_scale is not None:
        out["dscale"] = r.dresidual_scale
    return out


def _adamw_own(s):
    _, o = _package()
    norm = o.adamw(s["params_list"], s["grads"], s["m_list"], s["v_list"], ADAMW_STEP, **ADAMW,
                   max_norm=1.0 if s["case"]["clip"] else None, copies=s.get("copies_list"),
                   out=(s["params_out_list"], s["m_out_list"], s["v_out_list"]))
    return _adamw_results(s, norm)


OWN = {"delta": _delta_own, "block": _block_own, "adamw": _adamw_own}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["kind"]](state)


# -------------------------------------------------------------------- work
def work(case):
    e = {"fp32": 4.0, "bf16": 2.0}
    if case["kind"] == "adamw":
        n = float(sum(map(math.prod, _shapes(case))))
        t = e[case["grad"]]
        return dict(bytes=n * (24 + t + (2 if case["copies"] else 0)), flops=n * (14.0 + (2 if case["clip"] else 0)))
    t, B, T, back = e[case["type"]], case["B"], case["T"], case["back"]
    if case["kind"] == "block":
        n, w = float(B * T * case["width"]), case["width"]
        r, scale = e[case["res"]], 1 if case["scale"] else 0
        gate = {"none": 0.0, "rows": n, "clips": float(B * w)}[case["gate"]] * t
        if back:
            return dict(bytes=n * (3 * t + 4 * r) + n * r * scale + 2 * gate + 4.0 * w * (4 + 2 * scale),
                        flops=n * (30.0 + (8 if gate else 0)))
        return dict(bytes=n * (2 * t + 2 * r) + gate + 4.0 * w * (2 + scale), flops=n * (12.0 + (5 if gate else 0)))
    H, K, V = case["heads"], case["K"], case["V"]
    G = H // case["shared"]
    frames = float(B * T)
    state = 4.0 * B * H * K * V * ((1 if case["state"] else 0) + (0 if back else 1))
    if back:
        # q, k, v, dy, decays and strengths in; their gradients out
        return dict(bytes=frames * (4 * G * K + 3 * H * V) * t + frames * H * 16 + state, flops=frames * H * K * V * 19.0)
    return dict(bytes=frames * (2 * G * K + 2 * H * V) * t + frames * H * 8 + state, flops=frames * H * K * V * 7.0)


# ------------------------------------------------- the same in 64 bits
def _exact_delta(s, c):
    """Frame by frame: the memory decays, the key reads it, the rest of the
    value is written, the query reads."""
    shared, K = c["shared"], c["K"]
    B, T, H, V = s["v"].shape
    q0, k0 = (s[x].double().repeat_interleave(shared, 2) for x in "qk")
    lq, lk = (torch.sqrt(x.square().sum(-1, keepdim=True) + UNIT_EPS) for x in (q0, k0))
    q, k, v = q0 / lq / math.sqrt(K), k0 / lk, s["v"].double()
    n = [T] * B if s["lengths"] is None else s["lengths"].tolist()
    live = torch.tensor([[t < m for m in n] for t in range(T)], device=v.device)  # [T][B]
    decay = torch.where(live.T[..., None], s["g"].double(), 0.0).exp()
    beta = torch.where(live.T[..., None], s["beta"].double(), 0.0)
    S = torch.zeros(B, H, K, V, dtype=torch.float64, device=v.device)
    if s["state"] is not None:
        S = s["state"].double()
    y, kept = torch.zeros_like(v), []
    for t in range(T):
        if c["back"]:
            kept.append(S)
        S = S * decay[:, t, :, None, None]
        u = beta[:, t, :, None] * (v[:, t] - (k[:, t, :, None] @ S)[:, :, 0])
        S = S + k[:, t, :, :, None] * u[:, :, None]
        if not c["back"]:
            y[:, t] = (q[:, t, :, None] @ S)[:, :, 0]
    mask = live.T[..., None, None]
    if not c["back"]:
        return dict(y=torch.where(mask, y, 0.0), state=S)
    dy = torch.where(mask, s["dy"].double(), 0.0)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    dg, dbeta = torch.zeros_like(decay), torch.zeros_like(beta)
    dS = torch.zeros_like(S)
    for t in reversed(range(T)):
        before = kept.pop() * decay[:, t, :, None, None]
        miss = v[:, t] - (k[:, t, :, None] @ before)[:, :, 0]
        u = beta[:, t, :, None] * miss
        S = before + k[:, t, :, :, None] * u[:, :, None]
        dS = dS + q[:, t, :, :, None] * dy[:, t, :, None]
        dq[:, t] = (S @ dy[:, t, :, :, None])[..., 0]
        du = (k[:, t, :, None] @ dS)[:, :, 0]
        dbeta[:, t] = (du * miss).sum(-1)
        dmiss = beta[:, t, :, None] * du
        dv[:, t] = dmiss
        dk[:, t] = (dS @ u[..., None])[..., 0] - (before @ dmiss[..., None])[..., 0]
        dS = dS - k[:, t, :, :, None] * dmiss[:, :, None]
        dg[:, t] = (before * dS).sum((-1, -2))
        dS = dS * decay[:, t, :, None, None]
    dq = dq / math.sqrt(K)
    dq, dk = (d / l - x * (x * d).sum(-1, keepdim=True) / l ** 3 for d, x, l in ((dq, q0, lq), (dk, k0, lk)))
    dq, dk = (torch.where(mask, d.reshape(B, T, H // shared, shared, K).sum(3), 0.0) for d in (dq, dk))
    out = live.T[..., None]
    return dict(dq=dq, dk=dk, dv=torch.where(mask, dv, 0.0), dg=torch.where(out, dg, 0.0),
                dbeta=torch.where(out, dbeta, 0.0))


def _exact_block(s, c):
    """The gradients with sums of squares as they stand in the formula."""
    x, r, w1, w2 = s["x"].double(), s["residual"].double(), s["post"].double(), s["pre"].double()
    n = x.shape[-1]
    gate = torch.ones_like(x[..., :1]) if s["gate"] is None else torch.sigmoid(s["gate"].double())
    scale = torch.ones_like(w1) if s["scale"] is None else s["scale"].double()
    vx = x.square().sum(-1, keepdim=True) / n + EPS
    a = scale * r + gate * w1 * x / vx.sqrt()
    if not c["back"]:
        return dict(y=w2 * a / torch.sqrt(a.square().sum(-1, keepdim=True) / n + EPS), s=a)
    a = s["s"].double()
    va = a.square().sum(-1, keepdim=True) / n + EPS
    dy = s["dy"].double()
    da = dy * w2 * va ** -0.5 - a * (dy * w2 * a).sum(-1, keepdim=True) * va ** -1.5 / n + s["ds"].double()
    dn = da * gate * w1
    out = dict(dx=dn * vx ** -0.5 - x * (dn * x).sum(-1, keepdim=True) * vx ** -1.5 / n, dresidual=da * scale,
               dpost=(da * gate * x * vx ** -0.5).sum((0, 1)), dpre=(dy * a * va ** -0.5).sum((0, 1)))
    if s["gate"] is not None:
        d = da * w1 * x * vx ** -0.5 * gate * (1 - gate)
        out["dgate"] = d.sum(1, keepdim=True) if c["gate"] == "clips" else d
    if s["scale"] is not None:
        out["dscale"] = (da * r).sum((0, 1))
    return out


def _exact_adamw(s, c):
    g = torch.cat([t.double().reshape(-1) for t in s["grads"]])
    norm = g.square().sum().sqrt()
    if c["clip"]:
        g = g * min(1.0, 1.0 / (float(norm) + 1e-6))
    (b1, b2), lr, t = ADAMW["betas"], ADAMW["lr"], ADAMW_STEP
    m, v = s["m"].double(), s["v"].double()
    m, v = m + (1 - b1) * (g - m), v + (1 - b2) * (g.square() - v)
    p = s["params"].double()
    p = p - lr * (ADAMW["weight_decay"] * p + m / (1 - b1 ** t) / ((v / (1 - b2 ** t)).sqrt() + ADAMW["eps"]))
    out = dict(params=p, m=m, v=v)
    if c["copies"]:
        out["copies"] = p
    if c["clip"]:
        out["norm"] = norm
    return out


def exact(case, seed):
    if case["kind"] == "delta" and case["T"] > (20000 if case["back"] else 70000):
        return None  # (too many frames one by one)
    s = _inputs(case, seed)
    return {"delta": _exact_delta, "block": _exact_block, "adamw": _exact_adamw}[case["kind"]](s, case)
