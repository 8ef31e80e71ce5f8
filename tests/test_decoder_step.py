"""Decoder step: what is refused before a layer runs."""
import pytest
import torch

from tattletale_b200.decoder import DecoderStack


@pytest.mark.parametrize("fused", [False, True])
def test_settings_without_random_numbers(fused):
    """Without ``u`` a step is greedy: settings of the sampler would be dropped, misspelled ones too."""
    stack = DecoderStack.__new__(DecoderStack)  # (no layers, no device)
    stack.world, stack.fused_glue = 1, fused
    for settings in (dict(temperature=0.8), dict(top_p=0.9, top_k=3), dict(unknown=1)):
        with pytest.raises(ValueError, match=next(iter(settings))):
            stack.step(torch.zeros(1, dtype=torch.long), **settings)
