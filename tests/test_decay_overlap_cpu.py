"""The order of a backward pass's allocations and launches, with a library that launches nothing.

A walk that may start under the end of the launch before it must write to memory that nothing launched since the
first walk can still be using.  The launch before it need not be this pass's own: other threads use the same stream.
So every tensor that such a walk writes is taken from the allocator before the first walk is launched.
"""
from contextlib import nullcontext

import pytest
import torch

from bdm_b200 import _lib, decay, ops


class _Library:
    def __init__(self, log, workspace):
        self.log, self.workspace = log, workspace

    def bdm_decay_walk_workspace_bytes(self, w):
        return self.workspace

    def bdm_decay_walk(self, w, ws, nbytes, stream):
        a = _lib.DecayWalkArgs.from_buffer_copy(w)
        self.log.append(('walk', a.overlap, a.out, a.state_out))
        return 0

    def bdm_decay_group_sum(self, *a):
        self.log.append(('sum',))
        return 0


class _Status:
    mapped_ptr = 0

    def mapped_bits(self):
        return 0


@pytest.mark.parametrize('workspace', [0, 4096])
@pytest.mark.parametrize('kv_heads', [2, 1])
@pytest.mark.parametrize('state', [False, True])
def test_nothing_is_allocated_between_overlapping_walks(monkeypatch, state, kv_heads, workspace):
    log = []
    monkeypatch.setattr(_lib, 'load', lambda: _Library(log, workspace))
    monkeypatch.setattr(decay, '_on', lambda device: nullcontext())
    monkeypatch.setattr(decay, '_raw_stream', lambda device: 0)
    monkeypatch.setattr(ops, '_scan_status_of', lambda device: _Status())
    q = torch.randn(2, 9, 2, 8, requires_grad=True)
    k, v = (torch.randn(2, 9, kv_heads, 8, requires_grad=True) for _ in 'kv')
    s0 = torch.randn(2, 2, 8, 8, requires_grad=True) if state else None
    o, s = decay._DecayAttention.apply(q, k, v, torch.zeros(2), s0, None, 1.0, state)
    empty = torch.empty

    def allocate(*a, **kw):
        x = empty(*a, **kw)
        log.append(('empty', x.data_ptr()))
        return x

    del log[:]
    monkeypatch.setattr(torch, 'empty', allocate)
    outs = (o, s) if state else (o,)
    grads = torch.autograd.grad(outs, [x for x in (q, k, v, s0) if x is not None], [torch.ones_like(x) for x in outs])
    assert len(grads) == 3 + state
    walks = [i for i, e in enumerate(log) if e[0] == 'walk']
    assert len(walks) == 3
    assert (log[walks[1]][1], log[walks[2]][1]) == ((1, 1) if kv_heads == 2 and not workspace else (0, 0))
    assert log[walks[0]][1] == 0
    before = {e[1] for e in log[:walks[0]] if e[0] == 'empty'}
    for i in walks[1:]:
        if log[i][1]:
            assert {x for x in log[i][2:] if x} <= before
