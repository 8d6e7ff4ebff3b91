"""Infinities and NaN in decay attention: a token reaches what the recurrence lets it reach, and nothing else.

Every case is run twice, with and without the bad values; whatever the recurrence keeps apart from them has to be
the same bits, and what it lets them reach has to be infinite or NaN.
"""
import pytest
import torch

from test_decay_gpu import _inputs

pytestmark = pytest.mark.gpu
DEV = 'cuda'
BAD = [float('nan'), float('inf'), float('-inf')]
# unaligned BF16 (33 / 5), FP32 with 8 and with 16 warps
SIZES = [(torch.bfloat16, 33, 5), (torch.float32, 64, 64), (torch.float32, 128, 128), (torch.float32, 40, 72)]


def _run(x, g, s0, lengths=None):
    from bdm_b200 import decay_attention
    leaves = [x[name].clone().requires_grad_(True) for name in ('q', 'k', 'v')]
    o, s = decay_attention(*leaves, g, initial_state=s0, lengths=lengths, return_state=True)
    grads = torch.autograd.grad(o, leaves, x['do'])
    return dict(zip(('o', 'state', 'dq', 'dk', 'dv'), (o.detach(), s.detach(), *grads)))


def _same_outside(got, want, reached):
    """Where ``reached`` is false the bits agree; where it is true nothing is finite."""
    for name, r in reached.items():
        r = r.expand(got[name].shape)
        assert torch.equal(got[name][~r], want[name][~r]), name
        assert not torch.isfinite(got[name][r]).any(), name


@pytest.mark.parametrize('bad', BAD)
@pytest.mark.parametrize('what', ['q', 'k', 'v', 'do'])
@pytest.mark.parametrize('dtype,dk,dv', SIZES)
def test_one_bad_value_reaches_what_it_may(dtype, dk, dv, what, bad):
    B, T, H = 2, 300, 2
    q, k, v, do, g, s0, _ = _inputs(31, B, T, H, H, dk, dv, dtype)
    clean = dict(q=q, k=k, v=v, do=do)
    want = _run(clean, g, s0)
    t = torch.arange(T, device=DEV)
    for at in (0, 37, 63, 64, 150, 299):
        col = {'q': dk, 'k': dk, 'v': dv, 'do': dv}[what] // 2
        x = dict(clean, **{what: clean[what].clone()})
        x[what][1, at, 1, col] = bad
        here = torch.zeros(B, 1, H, 1, dtype=torch.bool, device=DEV)  # the row and head that hold it
        here[1, 0, 1] = True
        only, since, until = ((m[:, None, None]) & here for m in (t == at, t >= at, t <= at))
        none = torch.zeros_like(only)
        kcol, vcol = (torch.arange(w, device=DEV) == col for w in (dk, dv))
        state = here.transpose(1, 2)  # [B, H, 1, 1]
        off = dict(o=none, state=torch.zeros_like(state), dq=none, dk=none, dv=none)
        # o_t reads every k_s, v_s with s <= t; dq_t likewise, with do_t; dk_t and dv_t read q_s, do_s with s >= t
        if what == 'q':
            off.update(o=only, dk=until & kcol, dv=until)
        elif what == 'k':
            off.update(o=since, state=state & kcol[:, None], dq=since & kcol, dv=only)
        elif what == 'v':
            off.update(o=since & vcol, state=state & vcol, dq=since, dk=only)
        else:
            off.update(dq=only, dk=until, dv=until & vcol)
        _same_outside(_run(x, g, s0), want, off)


@pytest.mark.parametrize('dtype,dk,dv', SIZES)
def test_bad_values_in_many_columns_of_ragged_rows(dtype, dk, dv):
    """Several bad values to a column and a chunk, rows that end inside a chunk, and what lies past their ends."""
    B, T, H = 3, 200, 2
    q, k, v, do, g, s0, _ = _inputs(32, B, T, H, H, dk, dv, dtype)
    n = torch.tensor([200, 90, 130], device=DEV)
    t = torch.arange(T, device=DEV)[:, None, None]
    live = (t < n[:, None, None, None])
    clean = dict(q=q, k=k, v=v, do=do)
    want = _run(clean, g, s0, n)
    # column c of v is bad at tokens 20 + c and 60 + c of every head, and everywhere past the row's end
    at = 20 + torch.arange(dv, device=DEV)
    wrong = (t == at) | (t == at + 40)
    x = dict(clean, v=v.masked_fill(wrong, float('inf')).masked_fill(~live, float('nan')))
    got = _run(x, g, s0, n)
    # rows end before some columns turn bad
    reached = (t >= at) & live
    assert torch.equal(got['o'][~reached.expand_as(got['o'])], want['o'][~reached.expand_as(want['o'])])
    assert not torch.isfinite(got['o'][reached.expand_as(got['o'])]).any()
    over = (at < n[:, None])[:, None, None, :]
    assert torch.equal(got['state'][~over.expand_as(got['state'])], want['state'][~over.expand_as(want['state'])])
    assert not torch.isfinite(got['state'][over.expand_as(got['state'])]).any()
    # the same for the reverse walk: do
    x = dict(clean, do=do.masked_fill(wrong, float('inf')).masked_fill(~live, float('nan')))
    got = _run(x, g, s0, n)
    last = torch.where(at + 40 < n[:, None], at + 40, torch.where(at < n[:, None], at, -1))[:, None, None, :]
    reached = (t <= last) & live
    assert torch.equal(got['dv'][~reached.expand_as(got['dv'])], want['dv'][~reached.expand_as(want['dv'])])
    assert not torch.isfinite(got['dv'][reached.expand_as(got['dv'])]).any()


@pytest.mark.parametrize('dtype', [torch.float32])
def test_a_long_row_that_turns_bad_ends(dtype):
    """Every chunk after the first bad token takes the path for bad values."""
    from bdm_b200 import decay_attention
    q, k, v, _, g, s0, _ = _inputs(33, 1, 5000, 2, 2, 128, 128, dtype)
    want = decay_attention(q, k, v, g, initial_state=s0)
    for x in (q, k, v):
        x[:, 2500:] = float('nan')
    got = decay_attention(q, k, v, g, initial_state=s0)
    assert torch.equal(got[:, :2500], want[:, :2500]) and not torch.isfinite(got[:, 2500:]).any()
