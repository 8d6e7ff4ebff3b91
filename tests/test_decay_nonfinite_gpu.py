"""Infinities and NaN in decay attention: a token reaches what the recurrence lets it reach, and nothing else.

Every case is run twice, with and without the bad values.  What the recurrence lets them reach has to be infinite or
NaN.  What it keeps apart from them has to be the same bits; only in the BF16 kernel's 64-token chunks that hold a bad
value it is computed another way, and there it has to meet the bound of every BF16 output (2.1 u times the walk over
absolute values, test_decay_gpu.py).
"""
import functools

import pytest
import torch

from decay_reference import gradients, walk
from test_decay_gpu import _inputs, _near, _tol

pytestmark = pytest.mark.gpu
DEV = 'cuda'
BAD = [float('nan'), float('inf'), float('-inf')]
# BF16 at all four pairs of tile widths, unaligned BF16 (33 / 5), FP32 with 8 and with 16 warps
SIZES = [(torch.bfloat16, 64, 64), (torch.bfloat16, 64, 128), (torch.bfloat16, 128, 64), (torch.bfloat16, 128, 128),
         (torch.bfloat16, 40, 72), (torch.bfloat16, 33, 5), (torch.float32, 64, 64), (torch.float32, 128, 128),
         (torch.float32, 40, 72)]


def _run(x, g, s0, lengths=None):
    from bdm_b200 import decay_attention
    leaves = [x[name].clone().requires_grad_(True) for name in ('q', 'k', 'v')]
    o, s = decay_attention(*leaves, g, initial_state=s0, lengths=lengths, return_state=True)
    grads = torch.autograd.grad(o, leaves, x['do'])
    return dict(zip(('o', 'state', 'dq', 'dk', 'dv'), (o.detach(), s.detach(), *grads)))


def _truth(x, g, s0, lengths=None):
    """The clean case in FP64 and the walks over absolute values, as far as outputs have tokens."""
    q, k, v, do = (x[name] for name in ('q', 'k', 'v', 'do'))
    B, T, H, dk = q.shape
    n = torch.full((B,), T, device=DEV) if lengths is None else lengths
    out = []
    for absolute in (False, True):
        o = walk(q, k, v, g, n, H, dk ** -0.5, s0, absolute=absolute)[0]
        out.append(dict(zip(('o', 'dq', 'dk', 'dv'), (o, *gradients(q, k, v, do, g, n, dk ** -0.5, s0, absolute=absolute)))))
    return out


@functools.lru_cache(maxsize=1)
def _case(dtype, dk, dv):
    q, k, v, do, g, s0, _ = _inputs(31, 2, 300, 2, 2, dk, dv, dtype)
    clean = dict(q=q, k=k, v=v, do=do)
    return clean, g, s0, _run(clean, g, s0), _truth(clean, g, s0)


def _agree(got, want, truth, reached, chunk):
    """Where ``reached`` is true nothing is finite; elsewhere the bits agree, or inside ``chunk`` ([T] tokens) the bound
    holds."""
    for name, r in reached.items():
        x, y = got[name], want[name]
        r = r.expand(x.shape)
        assert not torch.isfinite(x[r]).any(), name
        same = ~r
        if name != 'state':
            same = same & ~chunk[:, None, None]
            near = (~r & chunk[:, None, None])
            _near(x[near], truth[0][name][near], _tol(x.dtype) * truth[1][name][near], name)
        assert torch.equal(x[same], y[same]), name


def _bad_chunks(at, T, dtype, dk, dv):
    """[T]: tokens in the chunk of a bad one, where the BF16 tensor-core kernel runs."""
    t = torch.arange(T, device=DEV)
    if dtype != torch.bfloat16 or dk % 8 or dv % 8:
        return torch.zeros_like(t, dtype=torch.bool)
    return (t[:, None] // 64 == torch.as_tensor(at, device=DEV).reshape(1, -1) // 64).any(-1)


@pytest.mark.parametrize('bad', BAD)
@pytest.mark.parametrize('what', ['q', 'k', 'v', 'do'])
@pytest.mark.parametrize('dtype,dk,dv', SIZES)
def test_one_bad_value_reaches_what_it_may(dtype, dk, dv, what, bad):
    B, T, H = 2, 300, 2
    clean, g, s0, want, truth = _case(dtype, dk, dv)
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
        _agree(_run(x, g, s0), want, truth, off, _bad_chunks(at, T, dtype, dk, dv))


@pytest.mark.parametrize('dtype,dk,dv', SIZES)
def test_bad_values_in_many_columns_of_ragged_rows(dtype, dk, dv):
    """Several bad values to a column and a chunk, rows that end inside a chunk, and what lies past their ends."""
    B, T, H = 3, 200, 2
    q, k, v, do, g, s0, _ = _inputs(32, B, T, H, H, dk, dv, dtype)
    n = torch.tensor([200, 90, 130], device=DEV)
    t = torch.arange(T, device=DEV)[:, None, None]
    live = (t < n[:, None, None, None])
    clean = dict(q=q, k=k, v=v, do=do)
    want, truth = _run(clean, g, s0, n), _truth(clean, g, s0, n)
    # column c of v is bad at tokens 20 + c and 60 + c of every head, and everywhere past the row's end
    at = 20 + torch.arange(dv, device=DEV)
    wrong = (t == at) | (t == at + 40)
    chunk = _bad_chunks(torch.cat([at, at + 40]), T, dtype, dk, dv)
    x = dict(clean, v=v.masked_fill(wrong, float('inf')).masked_fill(~live, float('nan')))
    over = (at < n[:, None])[:, None, None, :]  # rows end before some columns turn bad
    _agree(_run(x, g, s0, n), want, truth, dict(o=(t >= at) & live, state=over), chunk)
    # the same for the reverse walk: do
    x = dict(clean, do=do.masked_fill(wrong, float('inf')).masked_fill(~live, float('nan')))
    last = torch.where(at + 40 < n[:, None], at + 40, torch.where(at < n[:, None], at, -1))[:, None, None, :]
    _agree(_run(x, g, s0, n), want, truth, dict(dv=(t <= last) & live), chunk)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_a_long_row_that_turns_bad(dtype):
    from bdm_b200 import decay_attention
    q, k, v, _, g, s0, _ = _inputs(33, 1, 5000, 2, 2, 128, 128, dtype)
    n = torch.tensor([2500], device=DEV)
    truth = [dict(o=walk(q, k, v, g, n, 2, 128 ** -0.5, s0, absolute=a)[0]) for a in (False, True)]
    want = decay_attention(q, k, v, g, initial_state=s0)
    for x in (q, k, v):
        x[:, 2500:] = float('nan')
    got = decay_attention(q, k, v, g, initial_state=s0)
    t = torch.arange(5000, device=DEV)
    _agree(dict(o=got), dict(o=want), truth, dict(o=(t >= 2500)[:, None, None]), _bad_chunks(2500, 5000, dtype, 128, 128))


def test_rows_enough_for_whole_walks():
    """As many rows as SMs: one CTA has all columns of a row and no segments, unlike in the cases above."""
    from bdm_b200 import decay_attention
    q, k, v, _, g, _, _ = _inputs(34, 37, 330, 4, 4, 128, 128, torch.bfloat16, state=False)
    n = torch.full((37,), 330, device=DEV)
    truth = [dict(o=walk(q, k, v, g, n, 4, 128 ** -0.5, absolute=a)[0]) for a in (False, True)]
    want = decay_attention(q, k, v, g)
    col = torch.arange(128, device=DEV)
    at = torch.where(col % 3 == 0, 100 + col, 1 << 20)  # the first bad token of a column
    t = torch.arange(330, device=DEV)[:, None, None]
    got = decay_attention(q, k, v.masked_fill((t == at) | (t == at + 7), float('nan')), g)
    chunk = _bad_chunks(torch.cat([at, at + 7]), 330, torch.bfloat16, 128, 128)
    _agree(dict(o=got), dict(o=want), truth, dict(o=t >= at), chunk)


@pytest.mark.parametrize('dk,dv', [(64, 64), (128, 128)])
def test_shared_heads(dk, dv):
    """The gradients of shared heads leave the kernel in FP32."""
    q, k, v, do, g, s0, _ = _inputs(35, 2, 200, 4, 2, dk, dv, torch.bfloat16)
    clean = dict(q=q, k=k, v=v, do=do)
    want, truth = _run(clean, g, s0), _truth(clean, g, s0)
    t = torch.arange(200, device=DEV)
    for at in (70, 100):
        x = dict(clean, do=do.clone())
        x['do'][0, at, 2, 5] = float('inf')  # the first head of the second group
        here = torch.zeros(2, 1, 2, 1, dtype=torch.bool, device=DEV)
        here[0, 0, 1] = True
        until = (t <= at)[:, None, None] & here
        _agree(_run(x, g, s0), want, truth, dict(dk=until, dv=until & (torch.arange(dv, device=DEV) == 5)),
               _bad_chunks(at, 200, torch.bfloat16, dk, dv))
