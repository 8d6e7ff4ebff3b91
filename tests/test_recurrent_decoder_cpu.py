"""Decay attention, beam selection and reordering without a GPU: host checks of the C ABI and of the modules."""
import ctypes

import pytest
import torch

from bdm_b200 import (BSDMConfig, DecayAttention, HybridLanguageModel, LanguageModelConfig, _lib, beam_search, beam_select,
                      decay_attention, decay_attention_step, reorder_states)

ONE = 1 << 20  # a pointer that is never read: every call below is refused on the host


def _walk_args(**over):
    w = _lib.DecayWalkArgs(ONE, ONE, ONE, ONE, ONE, None, None, None, None)
    for name, v in dict(batch=1, time=4, heads=4, a_heads=4, b_heads=2, c_heads=2, width_ab=16, width_c=16,
                        dtype=_lib.BDM_BF16, out_dtype=_lib.BDM_BF16, scale=1.0, state_in_mul=1.0,
                        state_out_mul=1.0).items():
        setattr(w, name, over.get(name, v))
    for name in ('reverse', 'log_decay'):
        if name in over:
            setattr(w, name, over[name])
    return w


@pytest.mark.parametrize('over,status', [
    (dict(batch=-1), _lib.BDM_ERR_INVALID), (dict(time=-1), _lib.BDM_ERR_INVALID), (dict(heads=0), _lib.BDM_ERR_INVALID),
    (dict(b_heads=3), _lib.BDM_ERR_INVALID), (dict(width_c=0), _lib.BDM_ERR_INVALID), (dict(reverse=2), _lib.BDM_ERR_INVALID),
    (dict(dtype=7), _lib.BDM_ERR_DTYPE), (dict(dtype=_lib.BDM_F32), _lib.BDM_ERR_DTYPE),
    (dict(width_ab=136), _lib.BDM_ERR_UNSUPPORTED), (dict(log_decay=None), _lib.BDM_ERR_INVALID),
])
def test_walk_refuses_on_the_host(over, status):
    assert _lib.load().bdm_decay_walk(ctypes.byref(_walk_args(**over)), None, 0, None) == status


def test_other_entry_points_refuse_on_the_host():
    lib = _lib.load()
    assert lib.bdm_decay_walk(None, None, 0, None) == _lib.BDM_ERR_INVALID
    assert lib.bdm_decay_walk_workspace_bytes(ctypes.byref(_walk_args(heads=0))) == -1
    assert lib.bdm_decay_step(None, None) == _lib.BDM_ERR_INVALID
    assert lib.bdm_decay_group_sum(None, 4, 2, 2, 8, 1, None, None) == _lib.BDM_ERR_INVALID
    select = lambda *a: lib.bdm_beam_select(*a)  # noqa: E731
    assert select(None, 10, 1, 2, 10, 0, None, None, -1, 0, None, None, None, None, None, 0, None) == _lib.BDM_ERR_INVALID
    assert select(ONE, 10, 1, 33, 10, 0, ONE, None, -1, 0, ONE, ONE, ONE, None, ONE, 1 << 30, None) == _lib.BDM_ERR_UNSUPPORTED
    assert select(ONE, 10, 1, 2, 10, 0, ONE, ONE, -1, 0, ONE, ONE, ONE, None, ONE, 1 << 30, None) == _lib.BDM_ERR_INVALID
    assert select(ONE, 10, 1, 2, 10, 0, ONE, None, -1, 0, ONE, ONE, ONE, None, None, 0, None) == _lib.BDM_ERR_WORKSPACE
    assert lib.bdm_beam_select_workspace_bytes(4, 33, 100) == -1
    assert lib.bdm_reorder_rows(None, None, None, 1, None, 1, 2, None, None) == _lib.BDM_ERR_INVALID
    assert lib.bdm_reorder_rows(None, None, None, 0, None, 1, 2, None, None) == _lib.BDM_OK


def test_cpu_tensors_are_refused():
    q, g, s = torch.zeros(1, 4, 2, 8), torch.zeros(2), torch.zeros(1, 2, 8, 8)
    for call in (lambda: decay_attention(q, q, q, g), lambda: decay_attention_step(q[:, 0], q[:, 0], q[:, 0], g, s),
                 lambda: beam_select(torch.zeros(1, 2, 5), torch.zeros(1, 2)),
                 lambda: reorder_states([s], torch.zeros(1, 1, dtype=torch.long))):
        with pytest.raises(ValueError):
            call()


def test_layer_and_model_construction():
    layer = DecayAttention(64, 4, kv_heads=2, seed=1)
    g = layer.log_decay(torch.device('cpu'))
    assert g.dtype == torch.float32 and g.shape == (4,) and (g < 0).all() and (g.diff() > 0).all()
    assert layer.bfloat16().log_decay(torch.device('cpu')).dtype == torch.float32
    assert layer.create_state(3).shape == (3, 4, 16, 16)
    before = torch.random.get_rng_state()
    again = DecayAttention(64, 4, kv_heads=2, seed=1).bfloat16()
    assert torch.equal(before, torch.random.get_rng_state())
    assert all(torch.equal(a, b) for a, b in zip(layer.state_dict().values(), again.state_dict().values()))
    for kind, bad in [(ValueError, dict(dim=64, num_heads=3)), (ValueError, dict(dim=64, num_heads=4, kv_heads=3)),
                      (NotImplementedError, dict(dim=512, num_heads=2))]:
        with pytest.raises(kind):
            DecayAttention(**bad)
    cfg = LanguageModelConfig(memory=BSDMConfig(dim=64, bank_count=64, bank_size=8, selected_banks=4, value_width=64,
                                                num_heads=2), vocab_size=50, layers=3)
    m = HybridLanguageModel(cfg, decay_layers=[2])
    assert [type(b.attention).__name__ for b in m.layers] == ['BankedDeltaMemory'] * 2 + ['DecayAttention']
    with pytest.raises(ValueError):
        HybridLanguageModel(cfg, decay_layers=[3])
    with pytest.raises(RuntimeError):
        beam_search(m, torch.zeros(1, 4, dtype=torch.long), beams=2, max_new_tokens=2)
    with torch.no_grad(), pytest.raises(ValueError):
        beam_search(m, torch.zeros(1, 4, dtype=torch.long), beams=0, max_new_tokens=2)
