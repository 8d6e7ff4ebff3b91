"""Decay attention's scale: its whole range works forwards and backwards, what lies outside is refused at once."""
import pytest
import torch

from test_decay_gpu import _check, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('scale', [2.0 ** -40, -2.0 ** 40])
def test_far_from_one(scale, dtype):
    _check(*_inputs(71, 2, 130, 2, 2, 64, 64, dtype), scale=scale)


@pytest.mark.parametrize('scale', [0.0, float('nan'), float('inf'), -float('inf'), 1e-40, -1e-46, 1e39, 1e300])
def test_refused(scale):
    """Past FP32's range, or where the backward pass's 1 / scale would be."""
    from bdm_b200 import decay_attention, decay_attention_step
    q, k, v, do, g, s0, _ = _inputs(72, 2, 10, 2, 2, 16, 16, torch.float32)
    q.requires_grad_(True)
    with pytest.raises(ValueError):
        torch.autograd.grad(decay_attention(q, k, v, g, scale=scale), q, do)
    with torch.no_grad(), pytest.raises(ValueError):
        decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g, s0, scale=scale)
