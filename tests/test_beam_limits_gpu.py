"""Beam selection's limits at the public call: refused before anything is read or launched."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('beams,vocab', [(1, 2 ** 31 - 2 ** 16 + 1), (1, 3_000_000_000), (2, 2 ** 31)])
def test_vocabularies_past_32_bit_indices_are_refused(beams, vocab):
    from bdm_b200 import beam_select
    logits = torch.zeros(1, 1, 1, dtype=torch.bfloat16, device='cuda').expand(1, beams, vocab)  # no memory behind it
    with pytest.raises(NotImplementedError):
        beam_select(logits, torch.zeros(1, beams, device='cuda'))
