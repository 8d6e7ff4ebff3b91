"""State reordering over views whose rows lie between one another's."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def test_interleaved_views_of_one_buffer():
    from bdm_b200 import reorder_states
    parents = torch.tensor([[1, 1, 0], [2, 0, 2]], device=DEV)
    flat = (parents + torch.tensor([[0], [3]], device=DEV)).reshape(-1)
    whole = torch.arange(6 * 4 * 16, device=DEV, dtype=torch.float32).reshape(6, 4, 16)  # [row, layer, ...]
    want = whole[flat]
    reorder_states(list(whole.unbind(1)), parents)
    assert torch.equal(whole, want)
    # two strides in one buffer, rows side by side: 6 of 16 bytes within the gaps of 6 others, then apart
    room = torch.arange(6 * 32 + 64, device=DEV, dtype=torch.float32)
    a, b = room.as_strided((6, 8), (32, 1)), room.as_strided((6, 2), (16, 1), 12)
    keep = room.clone()
    wa, wb = a[flat].clone(), b[flat].clone()
    reorder_states([a, b], parents)
    assert torch.equal(a, wa) and torch.equal(b, wb)
    keep.as_strided((6, 8), (32, 1)).copy_(wa)
    keep.as_strided((6, 2), (16, 1), 12).copy_(wb)
    assert torch.equal(room, keep)


def test_views_that_do_overlap_are_refused():
    from bdm_b200 import reorder_states
    parents = torch.tensor([[1, 0]], device=DEV)
    x = torch.zeros(2, 40, device=DEV)
    for states in ([x[:, :20], x[:, 19:]], [x[:, :20], x[:, 10:12]], [x, x[:, 39:]],
                   [x.flatten().as_strided((2, 4), (8, 1)), x.flatten().as_strided((2, 4), (12, 1))]):
        with pytest.raises(ValueError):
            reorder_states(states, parents)


def test_states_of_any_iterable_and_single_tensors():
    from bdm_b200 import reorder_states
    parents = torch.tensor([[1, 0]], device=DEV)
    x = torch.arange(8.0, device=DEV).reshape(2, 4)
    want = x.flip(0)
    reorder_states((s for s in [x]), parents)
    assert torch.equal(x, want)
    with pytest.raises(ValueError):
        reorder_states(torch.zeros(2, 2, device=DEV), parents)  # a tensor is not a list of states
