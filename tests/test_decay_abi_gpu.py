"""Decay attention through its C entry points, with the argument blocks as a C caller fills them."""
import ctypes

import pytest
import torch

from test_decay_gpu import _inputs

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def _walk(q, k, v, g, s0, **over):
    from bdm_b200 import _lib
    B, T, H, dk = q.shape
    dv = v.shape[3]
    code = _lib.BDM_BF16 if q.dtype == torch.bfloat16 else _lib.BDM_F32
    out = torch.empty(B, T, H, dv, dtype=q.dtype, device=DEV)
    state = torch.empty(B, H, *((dv, dk) if over.get('state_out_transposed') else (dk, dv)), device=DEV)
    a = _lib.DecayWalkArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), g.data_ptr(), None, s0.data_ptr(),
                           state.data_ptr(), None)
    for name, x in (('a', q), ('b', k), ('c', v), ('out', out)):
        setattr(a, name + '_stride', (ctypes.c_int64 * 3)(*x.stride()[:3]))
    for name, value in dict(batch=B, time=T, heads=H, a_heads=H, b_heads=k.shape[2], c_heads=v.shape[2], width_ab=dk,
                            width_c=dv, dtype=code, out_dtype=code, scale=0.5, state_in_mul=1.0, state_out_mul=1.0,
                            **over).items():
        setattr(a, name, value)
    lib = _lib.load()
    n = lib.bdm_decay_walk_workspace_bytes(ctypes.byref(a))
    ws = torch.empty(max(n, 1), dtype=torch.uint8, device=DEV)
    _lib.check(lib.bdm_decay_walk(ctypes.byref(a), ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream), 'bdm_decay_walk')
    return out, state


@pytest.mark.parametrize('dtype,size', [(torch.float32, (2, 300, 4, 2, 40, 72)), (torch.bfloat16, (2, 300, 4, 2, 64, 128)),
                                        (torch.bfloat16, (2, 300, 4, 2, 33, 5)), (torch.bfloat16, (1, 2000, 2, 2, 128, 128))])
def test_walks_and_transposed_states(size, dtype):
    from bdm_b200 import decay_attention
    q, k, v, _, g, s0, _ = _inputs(81, *size, dtype)
    want = decay_attention(q, k, v, g, scale=0.5, initial_state=s0, return_state=True)
    given = s0.transpose(2, 3).contiguous()
    for turned_in in (0, 1):
        for turned_out in (0, 1):
            o, s = _walk(q, k, v, g, given if turned_in else s0, state_in_transposed=turned_in, state_out_transposed=turned_out)
            assert torch.equal(o, want[0])
            assert torch.equal(s.transpose(2, 3) if turned_out else s, want[1])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_a_step(dtype):
    from bdm_b200 import _lib, decay_attention_step
    q, k, v, _, g, s0, _ = _inputs(82, 3, 1, 4, 2, 40, 72, dtype)
    q, k, v = (x[:, 0] for x in (q, k, v))
    s = s0.clone()
    want = decay_attention_step(q, k, v, g, s, scale=0.5)
    state, out = s0.clone(), torch.empty_like(want)
    a = _lib.DecayStepArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), state.data_ptr(), out.data_ptr())
    for name, x in (('q', q), ('k', k), ('v', v)):
        setattr(a, name + '_stride', (ctypes.c_int64 * 2)(*x.stride()[:2]))
    a.batch, a.heads, a.kv_heads, a.key_width, a.value_width, a.scale = 3, 4, 2, 40, 72, 0.5
    a.dtype = _lib.BDM_BF16 if dtype == torch.bfloat16 else _lib.BDM_F32
    _lib.check(_lib.load().bdm_decay_step(ctypes.byref(a), torch.cuda.current_stream().cuda_stream), 'bdm_decay_step')
    assert torch.equal(out, want) and torch.equal(state, s)
