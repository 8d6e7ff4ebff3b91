"""Beam selection where tokens are masked by large finite values, and the BF16 kernel of aligned rows.

Rows of a multiple of 8 BF16 logits start on 16-byte boundaries and take a kernel of their own, with 8, 32 or
64 logits per thread by the number of rows; a slice of a row is 256 threads' worth of them.  A slice may be masked
as a whole, so its own maximum is the mask's value.

Scores of the chosen tokens: the softmax's terms are off by 2^-22 each, so is the logarithm of their sum; it, the
differences and the sum round to FP32: 2^-22 + 4 2^-24 of the largest of |score|, |x - max| and the log-sum-exp.
Indices are compared exactly: candidates are equal in exact arithmetic and in FP32, or further apart.
"""
import pytest
import torch

from test_beam_gpu import _check, _reference, _spread

pytestmark = pytest.mark.gpu
DEV = 'cuda'
INF = float('inf')


def _check_masked(x, s, finished=None, eos=None):
    from bdm_b200 import beam_select
    top = x.float().amax(-1, keepdim=True)
    for stable in (False, True):
        got = beam_select(x, s, finished=finished, eos_token=eos, stable_slots=stable)
        best, parents, tokens, done = _reference(x, s, finished, eos, stable)
        assert torch.equal(got.parents.cpu(), parents)
        assert torch.equal(got.tokens.cpu(), tokens)
        assert torch.equal(got.finished.cpu(), done)
        below = (x.float() - top).flatten(1).gather(1, got.parents * x.shape[2] + got.tokens)
        big = max(float(below.abs().max()), float(s.abs().max())) + 12
        assert ((got.scores.cpu().double() - best).abs() <= (2.0 ** -22 + 4 * 2.0 ** -24) * big).all()


def _mask(x, value):
    """Row w of a request: 0 only its first 2048 tokens allowed, 1 only its last 5, 2 every seventh, 3 all, 4 none."""
    V = x.shape[2]
    t = torch.arange(V, device=DEV)
    allowed = [t < 2048, t >= V - 5, t % 7 == 3, t >= 0]
    for w, a in enumerate(allowed):
        x[:, w].masked_fill_(~a, value)
    x[:, 4] = value
    return x


@pytest.mark.parametrize('value', ['lowest', -1e30, -1e20, -1e10, -1e9, -1e4])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
# BF16: 8, 32 and 64 logits per thread; rows of 9001 take the kernel of unaligned rows
@pytest.mark.parametrize('B,V', [(2, 48), (2, 9000), (1, 32000), (9, 32000), (31, 32000), (2, 9001)])
def test_tokens_masked_by_finite_values(B, V, dtype, value):
    x, s = _spread(11, B, 5, V, dtype)
    _check_masked(_mask(x, torch.finfo(dtype).min if value == 'lowest' else value), s)


@pytest.mark.parametrize('level', ['highest', 1e30, 1e10, 1e4])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('B,V', [(2, 48), (9, 32000), (31, 32000)])
def test_rows_at_a_high_level(B, V, dtype, level):
    """One allowed level far above the others, in one slice of the row or all over it."""
    x, s = _spread(12, B, 5, V, dtype)
    level = torch.finfo(dtype).max if level == 'highest' else level
    x[:, 0, V // 2:V // 2 + 6] = level
    x[:, 1] = level
    x[:, 2, -6:] = level
    x[:, 3, :6] = level
    x[:, 4, ::6] = level
    _check_masked(x, s)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('B,V', [(2, 48), (2, 9000), (7, 32000), (25, 32000)])
def test_banned_tokens_and_broken_rows_of_aligned_sizes(B, V, dtype):
    x, s = _spread(13, B, 6, V, dtype)
    x[:, :, ::3] = -INF
    x[0, 1] = -INF
    x[0, 2, V // 2] = float('nan')
    x[0, 3, V - 1] = INF
    x[1, 4] = float('nan')
    x[1, 5, :V // 2] = -INF
    _check(x, s)
    gen = torch.Generator().manual_seed(14)
    _check(x, s, (torch.rand(B, 6, generator=gen) < 0.4).to(DEV), V // 2)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('B,V', [(2, 3000), (41, 32000)])
def test_rounding_that_merges_candidates_of_aligned_rows(B, V, dtype):
    """Scores so large that stretches of logits round to one candidate: the lowest index wins."""
    from bdm_b200 import beam_select
    W = 4
    gen = torch.Generator().manual_seed(15)
    x = torch.rand(B, W, V, generator=gen).to(dtype).to(DEV)
    for score in (-1e9, -2e6):
        s = torch.full((B, W), score, device=DEV)
        got = beam_select(x, s)
        low = x.float() - x.float().amax(-1, keepdim=True)
        cand = (s[..., None] + (low - low.exp().sum(-1, keepdim=True).log())).reshape(B, W * V)
        # rows' log-sum-exps differ by an ulp, which these scores' spacing (0.125 and more) absorbs
        best, at = cand.sort(dim=-1, descending=True, stable=True)
        assert torch.equal(got.parents * V + got.tokens, at[:, :W])
        assert torch.equal(got.scores, best[:, :W])
