"""The sequence operators record nothing for autograd: an operand that requires
a gradient is taken with a warning, so that no graph is cut unseen."""
import warnings

import pytest

torch = pytest.importorskip("torch")

from dgen_hip import sequence as Q  # noqa: E402

pytestmark = pytest.mark.gpu


def calls(make):
    """(name of the operand, call) for every operand of every operator."""
    g = torch.Generator().manual_seed(1)

    def t(*shape):
        return torch.randn(*shape, generator=g).cuda()

    norm = dict(x=t(4, 8), weight=t(8), residual=t(4, 8))
    conv = dict(x=t(2, 5, 8), weight=t(8, 4), bias=t(8), state=t(2, 3, 8))
    scan = dict(x=t(2, 5, 8), dt=t(2, 5, 8), A=-t(8, 4).abs(), B=t(2, 5, 4), C=t(2, 5, 4), D=t(8), z=t(2, 5, 8),
                dt_bias=t(8), state=t(2, 8, 4))
    mlp = dict(x=t(4, 8), w_gate=t(8, 6), w_up=t(8, 6))
    for op, args in ((Q.rms_norm, norm), (Q.causal_conv, conv), (Q.selective_scan, scan), (Q.gated_mlp, mlp),
                     (Q.rms_norm_backward, dict(dy=t(4, 8), s=t(4, 8), weight=t(8), ds=t(4, 8))),
                     (Q.causal_conv_backward, dict(conv, dy=t(2, 5, 8))),
                     (Q.selective_scan_backward, dict(scan, dy=t(2, 5, 8))),
                     (Q.gated_mlp_backward, dict(mlp, dh=t(4, 6)))):
        for name in args:
            yield name, op, args, {**args, name: make(args[name])}


def flat(r):
    return [r] if isinstance(r, torch.Tensor) else [t for t in r if t is not None]


def test_a_warning_and_the_same_result(gpu):
    for name, op, plain, args in calls(lambda t: t.clone().requires_grad_()):
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            want = flat(op(**plain))
            with torch.no_grad():
                quiet = flat(op(**args))
        with pytest.warns(UserWarning, match=f"^{name} requires a gradient") as seen:
            got = flat(op(**args))
        assert seen[0].filename == __file__
        for a, b, c in zip(got, want, quiet):
            assert torch.equal(a, b) and torch.equal(b, c) and not a.requires_grad
