"""Gradient walks that overlap: read at once by what follows, and beside another thread's walks on the same stream."""
import threading

import pytest
import torch

from test_decay_gpu import _inputs

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def test_gradients_in_poisoned_memory_are_whole_when_the_next_kernel_starts():
    """The gradients' memory holds NaN before every pass, so a read before a walk's end shows."""
    from bdm_b200 import decay_attention
    q, k, v, do, g, _, _ = _inputs(61, 24, 700, 8, 8, 64, 64, torch.bfloat16, state=False)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    o = decay_attention(q, k, v, g)
    want = [x.cpu() for x in torch.autograd.grad(o, leaves, do, retain_graph=True)]
    for _ in range(5):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        poison = [torch.full_like(q, float('nan')) for _ in range(8)]
        places = {x.data_ptr() for x in poison}
        torch.cuda.synchronize()
        del poison
        grads = torch.autograd.grad(o, leaves, do, retain_graph=True)
        copies = [x + 0 for x in grads]
        assert all(x.data_ptr() in places for x in grads)
        assert all(torch.equal(x.cpu(), y) for x, y in zip(copies, want))
        del grads, copies


def test_two_threads_on_one_stream():
    """Each thread's passes free their memory while the other's walks are still queued."""
    from bdm_b200 import decay_attention

    def problem(seed):
        q, k, v, do, g, _, _ = _inputs(seed, 8, 500, 8, 8, 64, 64, torch.bfloat16, state=False)
        return [q, k, v], g, do

    def once(x, g, do):
        leaves = [y.clone().requires_grad_(True) for y in x]
        o = decay_attention(*leaves, g)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]

    problems = [problem(s) for s in (62, 63)]
    want = [once(*p) for p in problems]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        for n in range(200):
            got = once(*problems[i])
            if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                wrong.append((i, n))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_overlapping_walks_in_a_graph():
    from bdm_b200 import decay_attention
    q, k, v, do, g, _, _ = _inputs(64, 4, 300, 4, 4, 64, 64, torch.bfloat16, state=False)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    want = [x + 0 for x in torch.autograd.grad(decay_attention(q, k, v, g), leaves, do)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [x + 0 for x in torch.autograd.grad(decay_attention(q, k, v, g), leaves, do)]
    for _ in range(3):
        for x in got:
            x.fill_(float('nan'))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
