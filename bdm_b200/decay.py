"""Decay attention: linear attention with a decay for each head, for prompts, training and single tokens.

Per batch row and head, with lam = exp(log_decay[h]):

    S_t = lam S_{t-1} + k_t v_t^T        o_t = scale * q_t S_t

``decay_attention`` runs whole sequences chunk by chunk (differentiable), ``decay_attention_step`` one
token against a resident state, and ``DecayAttention`` is the mixer layer around them, with the same
``forward`` / ``prefill`` / ``step`` / ``create_state`` calls as the bank memory layer, so a language
model can interleave the two (``HybridLanguageModel``).  There is no reference counterpart.
"""
from __future__ import annotations

import struct
from contextlib import nullcontext

import torch
from torch import nn
from torch.nn import functional as F

from . import _lib, ops


_HERE = nullcontext()


def _on(device):
    """The launches below go to the device of their tensors."""
    return _HERE if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)


def _raw_stream(device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def _rows(x):
    """Columns of a head contiguous; every other stride is free."""
    return x if x.stride(-1) == 1 else x.contiguous()


# bdm_decay_walk_args and bdm_decay_step_args (include/bdm_b200.h), packed in one go: filling a ctypes
# structure field by field costs several times as much
_WALK = struct.Struct('9P12q2q12i3f4x')
_STEP = struct.Struct('6P6qq5if')


def _walk(a, b, c, log_decay, lengths, st, *, heads, scale, reverse=0, out_dtype=None, state_in=None, state_in_mul=1.0,
          state_in_transposed=0, state_out=None, state_out_mul=1.0, out=None, after=None):
    """One bdm_decay_walk over [B, T, heads of the operand, width] tensors; returns out [B, T, heads, width of c].

    ``after``: list of the walks already launched for this backward, independent of this one; it may overlap
    the launch before it when the last of them had no workspace.  That launch may be another thread's on the same
    stream, and what it uses may have been freed since: a walk that may overlap writes only to an ``out`` and a
    ``state_out`` that were allocated before the backward's first walk, which waits for all earlier launches."""
    batch, time, a_heads, wab = a.shape
    c_heads, wc = c.shape[2:]
    dt = a.dtype
    if out is None:
        out = torch.empty((batch, time, heads, wc), dtype=out_dtype or dt, device=a.device)
    w = _WALK.pack(a.data_ptr(), b.data_ptr(), c.data_ptr(), out.data_ptr(), log_decay.data_ptr(),
                   0 if lengths is None else lengths.data_ptr(), 0 if state_in is None else state_in.data_ptr(),
                   0 if state_out is None else state_out.data_ptr(), st.mapped_ptr,
                   *a.stride()[:3], *b.stride()[:3], *c.stride()[:3], time * heads * wc, heads * wc, wc,
                   batch, time, heads, a_heads, b.shape[2], c_heads, wab, wc, ops._DT[dt], ops._DT[out.dtype],
                   reverse, state_in_transposed, 0, int(bool(after and after[-1])), scale, state_in_mul,
                   state_out_mul)
    lib = _lib.load()
    nbytes = lib.bdm_decay_walk_workspace_bytes(w)
    ws = None
    if nbytes > 0:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=a.device)
    elif nbytes < 0:
        raise ValueError('invalid decay-attention geometry')
    status = lib.bdm_decay_walk(w, ws.data_ptr() if nbytes else None, nbytes, _raw_stream(a.device))
    if status:
        _lib.check(status, 'bdm_decay_walk')
    if after is not None:
        after.append(ws is None)
    return out


def _group_sum(part, kv_heads, dtype):
    """[B, T, H, D] FP32 gradients per query head -> [B, T, kv_heads, D] in ``dtype``."""
    batch, time, heads, width = part.shape
    out = torch.empty((batch, time, kv_heads, width), dtype=dtype, device=part.device)
    _lib.check(_lib.load().bdm_decay_group_sum(part.data_ptr(), batch * time, kv_heads, heads // kv_heads, width,
                                               ops._DT[dtype], out.data_ptr(), _raw_stream(part.device)),
               'bdm_decay_group_sum')
    return out


def _forward(q, k, v, log_decay, initial_state, lengths, scale, want_state):
    heads = q.shape[2]
    state = torch.empty((q.shape[0], heads, q.shape[3], v.shape[3]), dtype=torch.float32,
                        device=q.device) if want_state else None
    with _on(q.device):
        out = _walk(q, k, v, log_decay, lengths, ops._scan_status_of(q.device), heads=heads, scale=scale,
                    state_in=initial_state, state_out=state)
    return out, state


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, initial_state, lengths, scale, want_state):
        ctx.save_for_backward(q, k, v, log_decay, initial_state, lengths)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return _forward(q, k, v, log_decay, initial_state, lengths, scale, want_state)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, dstate):
        q, k, v, log_decay, s0, lengths = ctx.saved_tensors
        scale, heads, kv_heads, dt = ctx.scale, q.shape[2], k.shape[2], q.dtype
        if do is None and dstate is None:
            return (None,) * 8
        do = _rows(do) if do is not None else torch.zeros_like(v[:, :, :1]).expand(-1, -1, heads, -1)
        dstate = dstate.contiguous() if dstate is not None else None
        need = ctx.needs_input_grad
        dq = dk = dv = ds0 = None
        shared = kv_heads != heads
        walk = dict(heads=heads, scale=scale, after=None if shared else [])
        back = dict(walk, reverse=1, state_in=dstate, state_in_mul=1.0 / scale,
                    out_dtype=torch.float32 if shared else dt)
        with _on(q.device):
            st = ops._scan_status_of(q.device)
            ops.check_mapped_status(st)
            # all that overlapping walks write is allocated before the first launch (see _walk)
            if need[4]:
                ds0 = torch.empty((q.shape[0], heads, q.shape[3], v.shape[3]), dtype=torch.float32, device=q.device)
            if not shared:
                dk = torch.empty(k.shape, dtype=dt, device=q.device) if need[1] else None
                dv = torch.empty(v.shape, dtype=dt, device=q.device) if need[2] or need[4] else None
            if need[0]:
                dq = _walk(do, v, k, log_decay, lengths, st, state_in=s0, state_in_transposed=1, **walk)
            if need[1]:
                dk = _walk(v, do, q, log_decay, lengths, st, state_in_transposed=1, out=dk, **back)
                dk = _group_sum(dk, kv_heads, dt) if shared else dk
            if need[2] or need[4]:
                dv = _walk(k, q, do, log_decay, lengths, st, state_out=ds0, state_out_mul=scale, out=dv, **back)
                dv = _group_sum(dv, kv_heads, dt) if shared else dv
        return dq, dk, dv if need[2] else None, None, ds0, None, None, None


def _check_heads(q, k, v, log_decay, scale):
    """Shapes [..., heads, width] with the same leading sizes (1 or 2); returns the scale."""
    dt, at = q.dtype, q.get_device()
    if at < 0 or k.get_device() != at or v.get_device() != at or log_decay.get_device() != at:
        ops._cuda(q, k, v, log_decay)
        raise ValueError('q, k, v and log_decay must be on one device')
    if k.dtype != dt or v.dtype != dt:
        raise ValueError('q, k and v must share one dtype')
    ops.dtype_code(dt)
    qs, ks, vs = q.shape, k.shape, v.shape
    heads, kv_heads, dk = qs[-2], ks[-2], qs[-1]
    if (ks[-1] != dk or vs[-2] != kv_heads or ks[0] != qs[0] or vs[0] != qs[0]
            or (len(qs) == 4 and (ks[1] != qs[1] or vs[1] != qs[1]))):
        raise ValueError('k must be [..., kv_heads, key width of q] and v [..., kv_heads, value width], '
                         'with the leading sizes of q')
    if heads < 1 or kv_heads < 1 or dk < 1 or vs[-1] < 1 or heads % kv_heads:
        raise ValueError('the heads of q must be a multiple of the heads of k and v')
    if log_decay.dtype != torch.float32 or log_decay.shape != (heads,) or not log_decay.is_contiguous():
        raise ValueError(f'log_decay must be a contiguous float32 [{heads}] tensor')
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise ValueError('log_decay is a constant: it gets no gradient')
    if scale is None:
        return dk ** -0.5
    scale = float(scale)
    if not 1e-38 <= abs(scale) <= 1e38:  # its reciprocal is an FP32 number too: the backward pass divides by it
        raise ValueError('scale must be between 1e-38 and 1e38 in magnitude')
    return scale


def _check_state(name, state, shape, device):
    if (state.dtype != torch.float32 or state.shape != shape or state.get_device() != device.index
            or not state.is_contiguous()):
        raise ValueError(f'{name} must be a contiguous float32 {list(shape)} tensor on {device}')


def decay_attention(q, k, v, log_decay, *, scale=None, initial_state=None, lengths=None, return_state=False):
    """Linear attention with a decay for each head over whole sequences.

    q [B, T, H, dk], k [B, T, G, dk], v [B, T, G, dv] in float32 or bfloat16 (any strides; head h of q uses
    head h // (H // G) of k and v); log_decay [H] float32, log of the decay per token, at most 0 in use;
    dk, dv <= 128.  ``lengths`` (int64 [B]): tokens of row b from lengths[b] on are padding: not read, their
    outputs and gradients 0, and the state stops before them.  ``scale`` defaults to dk ** -0.5.

    Returns o [B, T, H, dv] in q's dtype, and with ``return_state`` (o, state [B, H, dk, dv] float32), the
    state after each row's last valid token, starting from ``initial_state`` (zero if None).
    An infinity or NaN makes what the recurrence lets it reach infinite or NaN (an infinity may arrive as NaN) and
    leaves everything else, the tokens before it among it, as it is.
    Differentiable (in reverse mode, once) in q, k, v and initial_state, through o and the state.
    Sums and the state are FP32.  With bfloat16 inputs the decayed scores and the copy of the state that o reads are
    rounded to bfloat16 once each, as o is; without ``return_state``, and in gradients, the terms of the state that is
    not returned have 17 bits instead of 24, so that o may differ by a rounding.
    """
    if q.ndim != 4 or k.ndim != 4 or v.ndim != 4:
        raise ValueError('q, k and v must be [batch, time, heads, width]')
    scale = _check_heads(q, k, v, log_decay, scale)
    ops._no_tangents('decay_attention', q, k, v, log_decay, initial_state)
    batch = q.shape[0]
    if initial_state is not None:
        _check_state('initial_state', initial_state, (batch, q.shape[2], q.shape[3], v.shape[3]), q.device)
    if lengths is not None and (lengths.dtype != torch.int64 or lengths.shape != (batch,)
                                or lengths.device != q.device or not lengths.is_contiguous()):
        raise ValueError(f'lengths must be a contiguous int64 [{batch}] tensor on {q.device}')
    if q.shape[3] > 128 or v.shape[3] > 128:
        raise NotImplementedError('decay_attention supports head widths up to 128')
    ops.check_mapped_status(ops._scan_status_of(q.device))
    q, k, v = _rows(q), _rows(k), _rows(v)
    run = _forward
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or (initial_state is not None and initial_state.requires_grad)):
        run = _DecayAttention.apply
    out, state = run(q, k, v, log_decay, initial_state, lengths, scale, return_state)
    return (out, state) if return_state else out


def decay_attention_step(q, k, v, log_decay, state, *, scale=None):
    """One token per row: ``state`` [B, H, dk, dv] (float32) is advanced in place; returns o [B, H, dv].

    q [B, H, dk], k [B, G, dk], v [B, G, dv] as one token of ``decay_attention``; dk <= 1024, any dv.
    Not differentiable; requires no_grad or inference_mode where an input would need a gradient.
    """
    if q.ndim != 3 or k.ndim != 3 or v.ndim != 3:
        raise ValueError('q, k and v must be [batch, heads, width]')
    scale = _check_heads(q, k, v, log_decay, scale)
    ops._no_tangents('decay_attention_step', q, k, v, log_decay, state)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad):
        raise RuntimeError('decay_attention_step requires no_grad or inference_mode')
    batch, heads, dk = q.shape
    dv = v.shape[2]
    _check_state('state', state, (batch, heads, dk, dv), q.device)
    if dk > 1024:
        raise NotImplementedError('decay_attention_step supports key widths up to 1024')
    q, k, v = _rows(q), _rows(k), _rows(v)
    out = torch.empty((batch, heads, dv), dtype=q.dtype, device=q.device)
    a = _STEP.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), state.data_ptr(), out.data_ptr(),
                   q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1), batch, heads,
                   k.shape[1], dk, dv,
                   ops._DT[q.dtype], scale)
    with _on(q.device):
        status = _lib.load().bdm_decay_step(a, _raw_stream(q.device))
    if status:
        _lib.check(status, 'bdm_decay_step')
    ops._changed(state)
    return out


class DecayAttention(nn.Module):
    """Mixer layer of decay attention, a drop-in beside ``BankedDeltaMemory`` in a language-model block.

    One projection gives q, k (SiLU, unit norm per head), v and an output gate; the heads' outputs are
    RMS-normalised per head, gated by a sigmoid and projected back.  The decays are fixed: 1 - 2^-e with e
    spread evenly over [min_exponent, max_exponent] across the heads (buffer ``log_decays``).  ``forward`` /
    ``prefill`` / ``step`` / ``create_state`` mirror the bank memory layer's; the state is FP32 [B, H, key width,
    value width].
    """

    def __init__(self, dim, num_heads, *, key_width=None, value_width=None, kv_heads=None, min_exponent=3.0,
                 max_exponent=9.0, norm_eps=1e-5, seed=0):
        super().__init__()
        kv_heads = num_heads if kv_heads is None else kv_heads
        if min(dim, num_heads, kv_heads) < 1 or num_heads % kv_heads:
            raise ValueError('num_heads must be a positive multiple of kv_heads')
        if (key_width is None or value_width is None) and dim % num_heads:
            raise ValueError('dim must be divisible by num_heads')
        self.dim, self.num_heads, self.kv_heads = dim, num_heads, kv_heads
        self.key_width, self.value_width = key_width or dim // num_heads, value_width or dim // num_heads
        if self.key_width > 128 or self.value_width > 128:
            raise NotImplementedError('decay attention supports head widths up to 128')
        self.norm_eps = norm_eps
        self._splits = [num_heads * self.key_width, kv_heads * self.key_width, kv_heads * self.value_width,
                        num_heads * self.value_width]
        with torch.random.fork_rng(devices=[]):  # init_weights below seeds them: the caller's generator stays
            self.in_proj = nn.Linear(dim, sum(self._splits), bias=False)
            self.o_proj = nn.Linear(num_heads * self.value_width, dim, bias=False)
        self.norm_weight = nn.Parameter(torch.ones(num_heads * self.value_width))
        with torch.inference_mode(False):  # backward passes save them
            exponent = torch.linspace(float(min_exponent), float(max_exponent), num_heads, dtype=torch.float64, device='cpu')
            log_decays = torch.log1p(-torch.exp2(-exponent)).float()
            at = self.in_proj.weight.device
            self.register_buffer('log_decays', log_decays if at.type == 'meta' else log_decays.to(at))
        self.init_weights(initialization_seed=seed)

    def init_weights(self, *, initialization_seed=0):
        with torch.random.fork_rng(devices=[]):
            torch.manual_seed(initialization_seed)
            for w in (self.in_proj.weight, self.o_proj.weight):
                nn.init.trunc_normal_(w, std=w.shape[1] ** -0.5, a=-3 * w.shape[1] ** -0.5, b=3 * w.shape[1] ** -0.5)
        nn.init.ones_(self.norm_weight)

    def _apply(self, fn, recurse=True):
        # the decays follow the module's device, but are FP32 whatever its dtype
        log_decays = self.log_decays
        super()._apply(fn, recurse)
        with torch.inference_mode(False):
            self.log_decays = log_decays.to(self.log_decays.device)
        return self

    def _load_from_state_dict(self, state_dict, prefix, *args, **kwargs):
        # checkpoints of before the decays were part of them
        state_dict.setdefault(prefix + 'log_decays', self.log_decays)
        super()._load_from_state_dict(state_dict, prefix, *args, **kwargs)

    def log_decay(self, device):
        """The heads' log-decays [H] on ``device``."""
        return self.log_decays if self.log_decays.device == device else self.log_decays.to(device)

    def create_state(self, batch, *, device=None):
        """A zero state for ``batch`` rows."""
        device = self.in_proj.weight.device if device is None else device
        return torch.zeros(batch, self.num_heads, self.key_width, self.value_width, device=device)

    def _heads(self, hidden):
        q, k, v, gate = self.in_proj(hidden).split(self._splits, -1)
        lead = hidden.shape[:-1]
        unit = lambda x, n: F.normalize(F.silu(x.reshape(*lead, n, self.key_width)), dim=-1,  # noqa: E731
                                        eps=1e-6).to(v.dtype)  # autocast leaves norms in FP32
        return unit(q, self.num_heads), unit(k, self.kv_heads), v.reshape(*lead, self.kv_heads, self.value_width), gate

    def _output(self, o, gate):
        x = o.float()
        x = (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + self.norm_eps)).flatten(-2)
        return self.o_proj((x * self.norm_weight.float() * torch.sigmoid(gate.float())).to(gate.dtype))

    def forward(self, hidden, *, lengths=None):
        """[B, T, dim] -> [B, T, dim] from a zero state; differentiable."""
        q, k, v, gate = self._heads(hidden)
        return self._output(decay_attention(q, k, v, self.log_decay(hidden.device), lengths=lengths), gate)

    def prefill(self, hidden, state=None, *, lengths=None, state_dtype=None):
        """Process a prefix [B, T, dim] -> (output, state); continues from ``state`` if given.

        The state is always FP32: ``state_dtype`` (which picks the bank caches' storage) has no effect.
        """
        if torch.is_grad_enabled():
            raise RuntimeError('prefill requires no_grad or inference_mode')
        q, k, v, gate = self._heads(hidden)
        o, state = decay_attention(q, k, v, self.log_decay(hidden.device), initial_state=state, lengths=lengths,
                                   return_state=True)
        return self._output(o, gate), state

    def step(self, hidden, state):
        """One token per row [B, 1, dim] -> (output [B, 1, dim], state); ``state`` is advanced in place."""
        if torch.is_grad_enabled():
            raise RuntimeError('step requires no_grad or inference_mode')
        if hidden.ndim != 3 or hidden.shape[1] != 1:
            raise ValueError('step takes one token per row: [batch, 1, dim]')
        q, k, v, gate = self._heads(hidden[:, 0])
        o = decay_attention_step(q, k, v, self.log_decay(hidden.device), state)
        return self._output(o, gate)[:, None], state
