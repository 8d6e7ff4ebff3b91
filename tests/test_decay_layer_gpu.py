"""The decay-attention layer's constants: where the module is, in its checkpoints, and usable inside a capture."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def test_first_call_inside_a_capture():
    from bdm_b200 import DecayAttention
    with torch.no_grad():
        for first in ('prefill', 'step'):
            m, twin = (DecayAttention(64, 2, seed=2).bfloat16().to(DEV) for _ in range(2))
            x = torch.randn(2, 1, 64, device=DEV, dtype=torch.bfloat16)
            state = m.create_state(2)
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):  # the libraries' own first calls; another layer's constants
                getattr(twin, first)(x, twin.create_state(2))
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                got, _ = getattr(m, first)(x, state)
            graph.replay()
            want, _ = getattr(twin, first)(x, twin.create_state(2))
            assert torch.equal(got, want)
