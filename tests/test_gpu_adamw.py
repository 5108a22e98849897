"""AdamW over many tensors (dgen_hip.optim) against the formula in 64 bits, and
over steps against torch's own.  Needs a GPU.

Tolerances, in roundings of fp32 (2^-24) relative to what a number is made of: a
moment is three operations, the parameter's change about ten; the gradients' norm, a sum in 64 bits of sums of
up to 64 squares in a row, 70."""
import pytest

torch = pytest.importorskip("torch")

from dgen_hip import optim  # noqa: E402
from test_gpu_sequence import F64, Data, close  # noqa: E402

pytestmark = pytest.mark.gpu
SHAPES = [(1,), (3, 5), (0, 4), (4096,), (4097,), (17, 241), (2, 3, 4), (12289,), (64, 64), (100000,), ()]
ARGS = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.02)


def tensors(seed, shapes=SHAPES, grad=torch.float32, odd=False):
    d = Data(seed)

    def at(t):  # at an address of an odd number of elements
        if not odd or not t.numel():
            return t.cuda()
        full = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")
        v = full[1:].view(t.shape)
        v.copy_(t)
        return v

    def all_of(make, **kw):
        return [at(make(*(s or (1,)), **kw).reshape(s)) for s in shapes]

    return (all_of(d.normal, scale=0.1), all_of(d.normal, type=grad, scale=1e-2), all_of(d.normal, scale=1e-3),
            all_of(d.uniform, hi=1e-4))


def formula(p, g, m, v, step, lr, betas, eps, weight_decay, max_norm=None):
    p, g, m, v = ([t.to(F64) for t in x] for x in (p, g, m, v))
    norm = torch.stack([t.square().sum() for t in g]).sum().sqrt()
    f = 1.0 if max_norm is None else min(1.0, max_norm / (norm.item() + 1e-6))
    # a rounding of m is relative to its two terms, which can cancel: |m'| may be far below beta1 |m| + (1 - beta1) |g|,
    # and what it is off by reaches p' times lr / (1 - beta1^t) / (sqrt(v^) + eps)
    terms = [betas[0] * a.abs() + (1 - betas[0]) * b.abs() * f for a, b in zip(m, g)]
    m = [betas[0] * a + (1 - betas[0]) * b * f for a, b in zip(m, g)]
    v = [betas[1] * a + (1 - betas[1]) * (b * f) ** 2 for a, b in zip(v, g)]
    sizes = [a.abs() + lr * (b / (1 - betas[0] ** step)) / ((c / (1 - betas[1] ** step)).sqrt() + eps)
             for a, b, c in zip(p, terms, v)]
    p = [(1 - lr * weight_decay) * a - lr * (b / (1 - betas[0] ** step)) / ((c / (1 - betas[1] ** step)).sqrt() + eps)
         for a, b, c in zip(p, m, v)]
    return p, m, v, norm, (sizes, terms, v)


def check(got, want, where=""):
    for name, x, y, ops, sizes in zip(("param", "exp_avg", "exp_avg_sq"), got, want, (16, 6, 8), want[4]):
        for i, (a, b, c) in enumerate(zip(x, y, sizes)):
            close(a, b.cpu(), ops, f"{name}[{i}] {where}", c.max().item() if c.numel() else None)


@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("step", [1, 7, 100000])
@pytest.mark.parametrize("max_norm", [None, 0.5, 1e6])
@pytest.mark.parametrize("odd", [False, True])
def test_one_step(gpu, grad, step, max_norm, odd):
    p, g, m, v = tensors(step, grad=grad, odd=odd)
    want = formula(p, g, m, v, step, max_norm=max_norm, **ARGS)
    copies = [torch.full(t.shape, 9.0, dtype=torch.bfloat16, device="cuda") for t in p]
    old = [t.clone() for t in (*p, *m, *v)]
    out = [[torch.full_like(t, 9.0) for t in x] for x in (p, m, v)]
    norm = optim.adamw(p, g, m, v, step, max_norm=max_norm, copies=copies, out=out, **ARGS)
    check(out, want)
    assert all(torch.equal(a, b) for a, b in zip(old, (*p, *m, *v)))  # left as they were
    assert all(torch.equal(a, b.bfloat16()) for a, b in zip(copies, out[0]))
    assert (norm is None) == (max_norm is None)
    if norm is not None:
        close(norm, want[3].cpu(), 70, "norm")
    # in place, the same bits; and with the count on the device, to its own rounding
    optim.adamw(p, g, m, v, step, max_norm=max_norm, **ARGS)
    assert all(torch.equal(a, b) for x, y in zip((p, m, v), out) for a, b in zip(x, y))
    p, g, m, v = tensors(step, grad=grad, odd=odd)
    optim.adamw(p, g, m, v, torch.tensor(step, device="cuda"), max_norm=max_norm, **ARGS)
    check((p, m, v), want, "counted there")


def test_many_tensors(gpu):
    """More than one launch takes, some of them empty."""
    shapes = [(i * 7 % 90, 3) for i in range(137)]
    p, g, m, v = tensors(3, shapes)
    want = formula(p, g, m, v, 5, max_norm=0.1, **ARGS)
    norm = optim.adamw(p, g, m, v, 5, max_norm=0.1, **ARGS)
    check((p, m, v), want)
    close(norm, want[3].cpu(), 70, "norm")


def test_steps_against_torch(gpu):
    p, _, _, _ = tensors(11, [(33, 20), (5,), (4100,)])
    theirs = [t.clone().requires_grad_() for t in p]
    copies = [t.bfloat16() for t in p]
    own = optim.AdamW(p, lr=1e-2, weight_decay=0.1, max_norm=0.7, copies=copies)
    opt = torch.optim.AdamW(theirs, lr=1e-2, weight_decay=0.1)
    for k in range(20):
        grads = tensors(100 + k, [(33, 20), (5,), (4100,)])[1]
        norm = own.step(grads)
        for t, x in zip(theirs, grads):
            t.grad = x.clone()
        assert torch.allclose(norm, torch.nn.utils.clip_grad_norm_(theirs, 0.7), rtol=1e-5)
        opt.step()
    for a, b, c in zip(p, theirs, copies):
        # (a step of lr 1e-2 each way, its direction to a few roundings where the gradients are not tiny)
        assert torch.allclose(a, b, atol=20 * 1e-2 * 2e-4) and torch.equal(c, a.bfloat16())
    assert int(own.count) == 20


def test_captured_steps_count_on(gpu):
    shapes = [(30, 7), (5000,)]
    p, g, _, _ = tensors(4, shapes)
    eager = optim.AdamW([t.clone() for t in p], max_norm=0.3)
    own = optim.AdamW(p, max_norm=0.3)
    start = [t.clone() for t in p]
    own.step(g)  # (loads the library)
    for t, s in zip(p, start):
        t.copy_(s)
    for t in (*own.exp_avg, *own.exp_avg_sq, own.count):
        t.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = own.step(g)
    for k in range(4):
        for t, x in zip(g, tensors(50 + k, shapes)[1]):
            t.copy_(x)
        want = eager.step(g)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want) and int(own.count) == k + 1
        assert all(torch.equal(a, b) for a, b in zip(own.params, eager.params))


def test_gradients_that_are_no_numbers(gpu):
    p, g, m, v = tensors(5, [(40,), (5000,)])
    g[0][3] = float("nan")
    before = p[1].clone()
    optim.adamw(p, g, m, v, 1, **ARGS)
    assert torch.isnan(p[0][3]) and torch.isfinite(p[0][4:]).all() and torch.isfinite(p[1]).all()
    # the norm is none either, and says so
    p[1].copy_(before)
    assert torch.isnan(optim.adamw(p, g, m, v, 1, max_norm=1.0, **ARGS))
    g[0][3] = float("inf")
    p, _, m, v = tensors(5, [(40,), (5000,)])
    assert torch.isinf(optim.adamw(p, g, m, v, 1, max_norm=1.0, **ARGS))
    assert torch.isnan(p[0][3]) and torch.isfinite(p[1]).all()


def test_streams(gpu):
    p, g, m, v = tensors(6)
    a = [[t.clone() for t in x] for x in (p, m, v)]
    optim.adamw(p, g, m, v, 3, max_norm=1.0, **ARGS)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        optim.adamw(a[0], g, a[1], a[2], 3, max_norm=1.0, **ARGS)
    side.synchronize()
    assert all(torch.equal(x, y) for q, r in zip((p, m, v), a) for x, y in zip(q, r))


def test_refusals(gpu):
    p, g, m, v = tensors(7, [(4, 5), (6,)])
    ok = dict(params=p, grads=g, exp_avg=m, exp_avg_sq=v, step=1)
    optim.adamw(**ok)
    half = [t.bfloat16() for t in p]
    for wrong in (dict(params=[]), dict(params=p[:1]), dict(params=[t.cpu() for t in p]), dict(params=half), dict(grads=[g[0], half[1]]),
                  dict(grads=[g[0].t().contiguous().t(), g[1]]), dict(grads=[g[0].reshape(5, 4), g[1]]), dict(exp_avg=m[:1]), dict(exp_avg=None),
                  dict(step=0), dict(step=torch.tensor(1.0, device="cuda")), dict(step=torch.tensor(1)), dict(lr=-1.0),
                  dict(lr=float("nan")), dict(betas=(0.9, 1.0)), dict(eps=-1.0), dict(weight_decay=-1.0), dict(max_norm=0.0),
                  dict(max_norm=float("nan")), dict(copies=p), dict(copies=half[:1]), dict(out=(p, m)), dict(out=(p, m, m)),
                  dict(out=(m, p, v)), dict(exp_avg=p), dict(exp_avg=[m[0], m[0].flatten()[:6]]), dict(exp_avg_sq=m),
                  dict(params=[p[0], p[0].flatten()[:6]])):
        with pytest.raises((ValueError, TypeError)):
            optim.adamw(**{**ok, **wrong})
