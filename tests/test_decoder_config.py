"""Decoders that cannot be made, on any host."""
import pytest

pytest.importorskip("torch")

from dgen_hip.decoder import DecoderConfig, RecurrentDecoder  # noqa: E402


@pytest.mark.parametrize("kw", [dict(heads=0), dict(key_heads=0), dict(heads=-8), dict(key=0), dict(heads=8, key_heads=3), dict(key=129),
                                dict(inner=2050 * 8)], ids=str)
def test_heads_that_do_not_fit(kw):
    with pytest.raises(ValueError, match="head|key"):
        RecurrentDecoder(DecoderConfig(mixer="delta", **kw), device="cpu")
    if "inner" not in kw:
        RecurrentDecoder(DecoderConfig(mixer="scan", hidden=8, inner=16, mlp=8, **kw), device="cpu")
