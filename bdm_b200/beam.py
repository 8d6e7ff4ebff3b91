"""Beam search over a recurrent decoder: selection, in-place reordering of its states, and the search loop.

A recurrent decoder keeps one fixed-size state per row (bank caches, decay-attention states) where a
transformer keeps a growing cache, so a beam that changes parents takes the parent's whole state.
``beam_select`` with ``stable_slots`` leaves every surviving beam where its state already is, and
``reorder_states`` then moves only the rows of beams that died, without a second buffer.
There is no reference counterpart.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib, ops
from .decay import _on, _raw_stream

MAX_BEAMS = 32
MAX_VOCAB = 2 ** 31 - 2 ** 16


class BeamStep(NamedTuple):
    scores: torch.Tensor    # [B, W] float32: sums of log-probabilities
    parents: torch.Tensor   # [B, W] int64: the beam each one continues
    tokens: torch.Tensor    # [B, W] int64
    finished: torch.Tensor  # [B, W] bool


def beam_select(logits, scores, *, finished=None, eos_token=None, stable_slots=False) -> BeamStep:
    """The W best continuations of W beams per batch row.

    logits [B, W, V] (float32 or bfloat16, rows contiguous), scores [B, W] float32, finished [B, W] bool.
    Candidate (w, t) scores ``scores[w] + log_softmax(logits[w])[t]`` in FP32; a finished beam has one
    candidate, ``eos_token`` at its score.  Logits of -inf are banned tokens.  A row with NaN, +inf or no
    finite logit has no candidate above -inf.  Ties go to the lower w, then the lower t.  Beams come in
    descending order, or with ``stable_slots`` each parent's best child in the parent's place and the other
    children in the free places in turn.  W <= 32.  Not differentiable.
    """
    ops._cuda(logits, scores, finished)
    ops._no_tangents('beam_select', logits, scores)
    if torch.is_grad_enabled() and (logits.requires_grad or scores.requires_grad):
        raise RuntimeError('beam_select requires no_grad or inference_mode for logits and scores that need gradients')
    if logits.ndim != 3 or tuple(scores.shape) != tuple(logits.shape[:2]) or scores.dtype != torch.float32:
        raise ValueError('logits must be [batch, beams, vocab] and scores float32 [batch, beams]')
    batch, beams, vocab = logits.shape
    if beams < 1 or vocab < 1:
        raise ValueError('beams and vocab must be positive')
    dev = logits.device
    code = ops.dtype_code(logits.dtype)
    if finished is not None and (finished.dtype != torch.bool or finished.shape != scores.shape):
        raise ValueError('finished must be bool [batch, beams]')
    if finished is not None and eos_token is None:
        raise ValueError('finished beams need an eos_token')
    if eos_token is not None and not 0 <= eos_token < vocab:
        raise ValueError('eos_token is outside the vocabulary')
    if scores.device != dev or (finished is not None and finished.device != dev):
        raise ValueError('logits, scores and finished must be on one device')
    if beams > MAX_BEAMS or vocab > MAX_VOCAB or beams * vocab >= 2 ** 32 - 1:
        raise NotImplementedError(f'beam_select supports up to {MAX_BEAMS} beams, vocab <= {MAX_VOCAB} and '
                                  f'beams * vocab < 2^32 - 1')
    rows = logits.reshape(batch * beams, vocab)
    if rows.stride(1) != 1 and vocab > 1:
        rows = rows.contiguous()
    scores = scores.contiguous()
    finished = finished.contiguous() if finished is not None else None
    lib = _lib.load()
    with _on(dev):
        # one allocation: the workspace, then the outputs
        nbytes = lib.bdm_beam_select_workspace_bytes(batch, beams, vocab)
        if nbytes < 0:
            raise ValueError('invalid beam geometry')
        ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=dev)
        out_scores = torch.empty((batch, beams), dtype=torch.float32, device=dev)
        index = torch.empty((2, batch, beams), dtype=torch.int64, device=dev)
        done = torch.empty((batch, beams), dtype=torch.bool, device=dev)
        parents, tokens = index.unbind(0)
        ld = rows.stride(0) if batch * beams > 1 else vocab
        _lib.check(lib.bdm_beam_select(rows.data_ptr(), ld, batch, beams, vocab, code, scores.data_ptr(),
                                       ops._ptr(finished), -1 if eos_token is None else int(eos_token),
                                       int(stable_slots), out_scores.data_ptr(), parents.data_ptr(), tokens.data_ptr(),
                                       done.data_ptr(), ws.data_ptr(), nbytes, _raw_stream(dev)), 'bdm_beam_select')
    return BeamStep(out_scores, parents, tokens, done)


def _overlap(spans):
    spans.sort()
    return any(b[0] < a[1] for a, b in zip(spans, spans[1:]))


def reorder_states(states, parents):
    """In place, for every tensor of ``states`` ([B * W, ...]): row (b, w) becomes row (b, parents[b, w]).

    ``parents`` [B, W] int64 as ``beam_select`` returns them.  Rows must be contiguous (any stride between
    them) and the tensors must not overlap.  Rows that keep their own place are neither read nor written
    (unless another row takes them).  A parent outside [0, W) leaves its row as it is and sets the device
    status that ``ops.check_scan_status`` reports.  Returns ``states``.
    """
    if isinstance(states, torch.Tensor):
        raise ValueError('states must be a list of tensors')
    given, states = states, list(states)
    ops._cuda(parents, *states)
    ops._no_tangents('reorder_states', *states)
    if parents.ndim != 2 or parents.dtype != torch.int64 or parents.shape[1] < 1:
        raise ValueError('parents must be int64 [batch, beams]')
    batch, beams = parents.shape
    if beams > MAX_BEAMS:
        raise NotImplementedError(f'reorder_states supports up to {MAX_BEAMS} beams')
    dev = parents.device
    extents, bases, strides, sizes = [], [], [], []
    for s in states:
        if s.ndim < 1 or s.shape[0] != batch * beams or s.device != dev:
            raise ValueError(f'states must be [{batch * beams}, ...] tensors on {dev}')
        if torch.is_grad_enabled() and s.requires_grad:
            raise RuntimeError('reorder_states requires no_grad or inference_mode for states that need gradients')
        if s.numel() == 0:
            continue
        size = s.numel() // (batch * beams) * s.element_size()
        stride = size
        if not s.is_contiguous():
            if not s[0].is_contiguous():
                raise ValueError('the rows of a state must be contiguous')
            stride = s.stride(0) * s.element_size() if s.shape[0] > 1 else size
        if stride < size:
            raise ValueError('the rows of a state must not overlap')
        bases.append(s.data_ptr())
        strides.append(stride)
        sizes.append(size)
        extents.append((s.data_ptr(), s.data_ptr() + stride * (s.shape[0] - 1) + size))
    if _overlap(extents) and _overlap([(base + i * stride, base + i * stride + size)  # rows may lie between other rows
                                       for base, stride, size in zip(bases, strides, sizes)
                                       for i in range(batch * beams)]):
        raise ValueError('the states must not overlap')
    parents = parents.contiguous()
    n = len(bases)
    with _on(dev):
        _lib.check(_lib.load().bdm_reorder_rows((ctypes.c_void_p * n)(*bases), (ctypes.c_int64 * n)(*strides),
                                                (ctypes.c_int64 * n)(*sizes), n, parents.data_ptr(), batch, beams,
                                                ops._scan_status_of(dev).mapped_ptr + 4, _raw_stream(dev)),
                   'bdm_reorder_rows')
    ops._changed(*states)
    return given


def beam_search(model, prompt, *, beams, max_new_tokens, eos_token=None):
    """Beam search with a language model of recurrent layers (``prefill`` / ``capture_step``).

    prompt [B, T] int64 -> (tokens [B, beams, max_new_tokens], scores [B, beams]), best beam first; a beam
    that has produced ``eos_token`` repeats it.  The prompt is processed once per request; its states are
    then forked to the beams, and every step is the captured model step, one selection and one in-place
    reordering of all layers' states.  Requires no_grad / inference_mode.
    """
    if torch.is_grad_enabled():
        raise RuntimeError('beam_search requires no_grad or inference_mode')
    if beams < 1 or max_new_tokens < 1:
        raise ValueError('beams and max_new_tokens must be positive')
    batch = prompt.shape[0]
    dev = prompt.device
    logits, caches = model.prefill(prompt)
    caches = [c.repeat_interleave(beams, 0) for c in caches]
    # all beams of a request are alike: only the first one counts
    scores = torch.full((batch, beams), float('-inf'), device=dev)
    scores[:, 0] = 0.0
    finished = torch.zeros(batch, beams, dtype=torch.bool, device=dev) if eos_token is not None else None
    logits = logits[:, -1:].expand(batch, beams, -1)
    history = []
    run = None
    for i in range(max_new_tokens):
        step = beam_select(logits, scores, finished=finished, eos_token=eos_token, stable_slots=True)
        scores = step.scores
        finished = step.finished if eos_token is not None else None
        history.append((step.parents, step.tokens))
        if i + 1 == max_new_tokens:
            break
        if i:  # after the prompt every beam's states are the same
            reorder_states(caches, step.parents)
        if run is None:
            run = model.capture_step(caches)
        logits = run(step.tokens.reshape(batch * beams, 1)).reshape(batch, beams, -1)
    order = scores.argsort(dim=-1, descending=True, stable=True)
    at, out = order, []
    for parents, tokens in reversed(history):
        out.append(tokens.gather(1, at))
        at = parents.gather(1, at)
    ops.check_scan_status(dev, wait=True)
    return torch.stack(out[::-1], -1), scores.gather(1, order)
