"""Tensors that the recurrent-decoder operators change in place say so to autograd."""
import pytest
import torch

from test_decay_gpu import _inputs

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def test_a_state_saved_for_backward_and_stepped():
    from bdm_b200 import decay_attention, decay_attention_step
    q, k, v, do, g, s0, _ = _inputs(52, 2, 20, 2, 2, 16, 16, torch.float32)
    q.requires_grad_(True)
    o = decay_attention(q, k, v, g, initial_state=s0)
    with torch.no_grad():
        decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g, s0)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        torch.autograd.grad(o, q, do)


def test_a_state_saved_for_backward_and_reordered():
    from bdm_b200 import decay_attention, reorder_states
    q, k, v, do, g, s0, _ = _inputs(53, 2, 20, 2, 2, 16, 16, torch.float32)
    q.requires_grad_(True)
    o = decay_attention(q, k, v, g, initial_state=s0)
    reorder_states([s0], torch.tensor([[1, 0]], device=DEV))
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        torch.autograd.grad(o, q, do)


def test_inference_tensors_are_changed_as_before():
    from bdm_b200 import decay_attention_step, reorder_states
    q, k, v, _, g, s0, _ = _inputs(54, 2, 1, 2, 2, 16, 16, torch.float32)
    want = s0.clone()
    decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g, want)
    with torch.inference_mode():
        s = s0.clone()
        decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g, s)
        assert torch.equal(s, want)
        reorder_states([s], torch.tensor([[1, 0]], device=DEV))
        assert torch.equal(s, want.flip(0))
