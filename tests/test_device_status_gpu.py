"""Resetting the device status: in stream order, so what was launched before it cannot bring a bit back."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def test_reset_comes_after_what_is_still_running():
    from bdm_b200 import ops, reorder_states
    ops.reset_scan_status()
    s = torch.zeros(2, 4, device=DEV)
    parents = torch.tensor([[5, 0]], device=DEV)
    reorder_states([s], torch.tensor([[1, 0]], device=DEV))  # the kernel's first launch loads it, which waits for the GPU
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)  # a tenth of a second and more
    reorder_states([s], parents)
    ops.reset_scan_status()
    torch.cuda.synchronize()
    try:
        ops.check_scan_status(wait=True)
    finally:
        ops.reset_scan_status()


def test_reset_inside_a_graph():
    from bdm_b200 import ops, reorder_states
    from bdm_b200._lib import BDMError
    s = torch.zeros(2, 4, device=DEV)
    parents = torch.tensor([[5, 0]], device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.reset_scan_status()
    try:
        reorder_states([s], parents)
        with pytest.raises(BDMError):
            ops.check_scan_status(wait=True)
        graph.replay()
        ops.check_scan_status(wait=True)
    finally:
        ops.reset_scan_status()
