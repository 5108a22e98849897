"""The control decoder at its ends: heads of the delta rule that forget, their decays'
gradients against the model in 64 bits up to gates that are -infinity, and no blocks.  Needs a
GPU."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_decoder import norm  # noqa: E402
from test_gpu_decoder_blocks import F64, small, wide_model  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("log_A", [5.0, 20.0, 60.0, 100.0])
@pytest.mark.parametrize("lengths", [None, [70, 0, 33]])
def test_heads_that_forget(gpu, log_A, lengths):
    """Within the bound of the decoder's other passes (test_gpu_decoder_blocks),
    and that head's own parameters, whose gradients end at 0, too."""
    dec, T = small("delta", False), 70
    for i in range(2):
        dec.params[f"{i}.log_A"][1] = log_A
    g = torch.Generator().manual_seed(6)
    x, dZ = torch.randn(3, T, 2, generator=g), torch.randn(3, T, 9, generator=g)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    Z, kept = dec.forward(x, lengths=n, keep=True)
    grads = dec.backward(dZ.cuda(), kept)
    P = {k: v.cpu().to(F64).requires_grad_() for k, v in dec.params.items()}
    want = wide_model(dec.cfg, P, x.to(F64), lengths or [T] * 3)
    assert (Z.cpu().to(F64) - want).abs().max() <= 2e-4 * want.abs().max()
    (want * dZ.to(F64)).sum().backward()
    for k, p in P.items():
        assert torch.isfinite(grads[k]).all(), k
        err = (grads[k].cpu().to(F64) - p.grad).abs().max().item()
        assert err <= 2e-4 * p.grad.abs().max().item() + 1e-9, (k, err, p.grad.abs().max().item())
    if log_A >= 60.0:
        for i in range(2):
            assert grads[f"{i}.log_A"][1] == 0 and grads[f"{i}.dt_bias"][1] == 0


@pytest.mark.parametrize("mixer", ["scan", "delta"])
@pytest.mark.parametrize("around", [False, True])
def test_a_decoder_of_no_blocks(gpu, mixer, around):
    """Two projections and a norm: as the others, within the plain decoder's
    bound."""
    from dgen_hip.decoder import DecoderConfig, RecurrentDecoder
    dec = RecurrentDecoder(DecoderConfig(controls=9, hidden=40, inner=72, blocks=0, dtype=torch.float32, mixer=mixer, around=around, heads=4))
    x, dZ = torch.randn(2, 5, 2, generator=torch.Generator().manual_seed(1)), torch.randn(2, 5, 9, device="cuda")
    Z, kept = dec.forward(x, keep=True)
    grads = dec.backward(dZ, kept)
    P = {k: v.cpu().to(F64).requires_grad_() for k, v in dec.params.items()}
    want = norm(x.to(F64) @ P["in"], P["norm"]) @ P["heads"] + P["heads_bias"]
    assert (Z.cpu().to(F64) - want).abs().max() <= 2e-4 * want.abs().max()
    (want * dZ.cpu().to(F64)).sum().backward()
    for k, p in P.items():
        assert (grads[k].cpu().to(F64) - p.grad).abs().max() <= 2e-4 * p.grad.abs().max() + 1e-9, k
