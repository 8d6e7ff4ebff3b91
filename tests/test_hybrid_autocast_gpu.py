"""The hybrid language model under autocast, where its projections are BF16 and its norms FP32."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def _model():
    from bdm_b200 import BSDMConfig, HybridLanguageModel, LanguageModelConfig
    mem = BSDMConfig(dim=64, bank_count=64, bank_size=8, selected_banks=4, value_width=64, num_heads=2)
    return HybridLanguageModel(LanguageModelConfig(memory=mem, vocab_size=50, layers=2, seed=3), decay_layers=[0, 1]).to(DEV)


def test_training_and_steps_under_autocast():
    """Rounding to BF16 moves logits by a few 2^-8 of their size per layer; both runs round the same values."""
    m = _model()
    gen = torch.Generator().manual_seed(91)
    x = torch.randint(0, 50, (2, 70), generator=gen).to(DEV)
    with torch.autocast('cuda', dtype=torch.bfloat16):
        loss = m(x[:, :-1], x[:, 1:])
        loss.backward()
        assert all(torch.isfinite(p.grad).all() for p in m.parameters() if p.requires_grad)
        with torch.inference_mode():
            whole = m(x)
            _, states = m.prefill(x[:, :60])
            for t in range(60, 70):
                logits = m.step(x[:, t:t + 1], states)
                assert (logits[:, 0].float() - whole[:, t].float()).abs().max() <= 2.0 ** -4 * whole.float().abs().max()
    with torch.inference_mode():
        exact = m(x)
    assert (whole.float() - exact).abs().max() <= 2.0 ** -4 * exact.abs().max()
