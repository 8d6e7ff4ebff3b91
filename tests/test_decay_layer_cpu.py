"""The decay-attention layer's decays: FP32 on the module's device, in its checkpoints, loadable from older ones."""
import copy

import pytest
import torch

from bdm_b200 import BSDMConfig, DecayAttention, HybridLanguageModel, LanguageModelConfig

CPU = torch.device('cpu')


def test_a_checkpoint_carries_the_decays():
    a = DecayAttention(64, 4, min_exponent=2.0, max_exponent=5.0)
    b = DecayAttention(64, 4, seed=1)
    assert not torch.equal(a.log_decay(CPU), b.log_decay(CPU))
    b.load_state_dict(a.state_dict())
    assert torch.equal(a.log_decay(CPU), b.log_decay(CPU))


def test_a_checkpoint_without_them_still_loads():
    a, b = DecayAttention(64, 4), DecayAttention(64, 4, seed=1)
    older = {k: v for k, v in a.state_dict().items() if 'decay' not in k}
    assert len(older) == 3
    b.load_state_dict(older)
    assert torch.equal(a.log_decay(CPU), b.log_decay(CPU)) and torch.equal(a.in_proj.weight, b.in_proj.weight)
    cfg = LanguageModelConfig(memory=BSDMConfig(dim=64, bank_count=64, bank_size=8, selected_banks=4, value_width=64,
                                                num_heads=2), vocab_size=50, layers=2)
    m, n = HybridLanguageModel(cfg), HybridLanguageModel(cfg)
    n.load_state_dict({k: v for k, v in m.state_dict().items() if 'decay' not in k})
    with pytest.raises(RuntimeError):
        b.load_state_dict({k: v for k, v in older.items() if 'in_proj' not in k})


@pytest.mark.parametrize('move', [lambda m: m.bfloat16(), lambda m: m.double(), lambda m: m.half().float(),
                                  lambda m: copy.deepcopy(m).bfloat16(), lambda m: m.to(torch.bfloat16)])
def test_they_stay_fp32(move):
    want = DecayAttention(64, 4).log_decay(CPU)
    m = move(DecayAttention(64, 4))
    assert m.log_decay(CPU).dtype == torch.float32 and torch.equal(m.log_decay(CPU), want)


def test_they_follow_the_module():
    assert DecayAttention(64, 4).to('meta').log_decay(torch.device('meta')).is_meta
    with torch.device('meta'):
        m = DecayAttention(64, 4)
    m = m.to_empty(device='cpu')
    assert torch.equal(m.log_decay(CPU), DecayAttention(64, 4).log_decay(CPU))
    with torch.inference_mode():
        m = DecayAttention(64, 4).bfloat16()
    assert not m.log_decay(CPU).is_inference()


def test_they_are_no_parameters():
    m = DecayAttention(64, 4)
    assert len(list(m.parameters())) == 3 and not m.log_decay(CPU).requires_grad
