"""What autograd has to know of the recurrent-decoder operators: tangents and gradients that they have none of are
refused, not dropped, and tensors that they change say so."""
import pytest
import torch
from torch.autograd import forward_ad

from test_decay_gpu import _inputs

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def _some():
    q, k, v, _, g, s0, _ = _inputs(51, 2, 20, 2, 2, 16, 16, torch.float32)
    return q, k, v, g, s0


@pytest.mark.parametrize('grad', [True, False])
def test_forward_mode_is_refused(grad):
    from bdm_b200 import beam_select, decay_attention, decay_attention_step, reorder_states
    q, k, v, g, s0 = _some()
    logits, scores = torch.randn(2, 3, 10, device=DEV), torch.zeros(2, 3, device=DEV)
    parents = torch.zeros(1, 2, dtype=torch.long, device=DEV)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        dual = lambda x: forward_ad.make_dual(x, torch.ones_like(x))  # noqa: E731
        for call in (lambda: decay_attention(dual(q), k, v, g), lambda: decay_attention(q, dual(k), v, g),
                     lambda: decay_attention(q, k, dual(v), g), lambda: decay_attention(q, k, v, dual(g)),
                     lambda: decay_attention(q, k, v, g, initial_state=dual(s0)),
                     lambda: decay_attention_step(dual(q[:, 0]), k[:, 0], v[:, 0], g, s0),
                     lambda: decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g, dual(s0)),
                     lambda: beam_select(dual(logits), scores), lambda: beam_select(logits, dual(scores)),
                     lambda: reorder_states([dual(s0)], parents)):
            with pytest.raises(NotImplementedError):
                call()
        # what has no tangent goes on as it did
        assert torch.isfinite(decay_attention(q, k, v, g, initial_state=s0)).all()
        beam_select(logits, scores)


def test_a_layer_refuses_tangents():
    from bdm_b200 import DecayAttention
    m = DecayAttention(64, 2, seed=1).to(DEV)
    x = torch.randn(1, 10, 64, device=DEV)
    with torch.no_grad(), forward_ad.dual_level(), pytest.raises(NotImplementedError):
        m(forward_ad.make_dual(x, torch.ones_like(x)))


def test_selection_refuses_to_cut_a_graph():
    from bdm_b200 import beam_select
    logits, scores = torch.randn(2, 3, 10, device=DEV), torch.zeros(2, 3, device=DEV)
    for args in ((logits.clone().requires_grad_(True), scores), (logits, scores.clone().requires_grad_(True))):
        with pytest.raises(RuntimeError):
            beam_select(*args)
        with torch.no_grad():
            beam_select(*args)
