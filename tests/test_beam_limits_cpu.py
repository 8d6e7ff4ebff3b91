"""Beam selection's limits, refused on the host before anything is read or launched."""
import pytest

from bdm_b200 import _lib

ONE = 1 << 20  # a pointer that is never read
WORST = 2 ** 31 - 2 ** 16


@pytest.mark.parametrize('beams,vocab', [(1, WORST + 1), (1, 2 ** 31), (1, 3_000_000_000), (1, 2 ** 32 - 2), (2, 2 ** 31),
                                         (3, 2_000_000_000), (33, 10)])
def test_vocabularies_past_32_bit_indices_are_refused(beams, vocab):
    """A token's index, rounded up to a whole slice of its row, is a 32-bit signed integer in the kernels."""
    lib = _lib.load()
    assert lib.bdm_beam_select_workspace_bytes(1, beams, vocab) == -1
    assert lib.bdm_beam_select(ONE, vocab, 1, beams, vocab, _lib.BDM_BF16, ONE, None, -1, 0, ONE, ONE, ONE, None, None, 0,
                               None) == _lib.BDM_ERR_UNSUPPORTED


def test_the_largest_vocabulary_is_taken():
    lib = _lib.load()
    assert lib.bdm_beam_select_workspace_bytes(1, 1, WORST) > 0
    # as far as the check of the workspace
    assert lib.bdm_beam_select(ONE, WORST, 1, 1, WORST, _lib.BDM_BF16, ONE, None, -1, 0, ONE, ONE, ONE, None, None, 0,
                               None) == _lib.BDM_ERR_WORKSPACE
