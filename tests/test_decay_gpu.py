"""Decay attention on the GPU against the token-by-token recurrence in FP64.

Bounds.  A is the same walk over absolute values, so every product that is summed is below it.
BF16 outputs: the chunk's decayed score matrix and the carried state are each rounded once to BF16
(unit roundoff u = 2^-8) where the tensor cores read them, and the output once more; a term is in the
score matrix or in the state, so |error| <= (2 u + u^2) A, plus the FP32 sums': 2.1 u A.
FP32 outputs, and every FP32 state: a sum's terms pass at most a few hundred FP32 roundings (chunk sums of
64, a carry per chunk, 128 columns) of 2^-24, nearly all of random sign; decays are exp of an FP32 product,
off by at most |log| 2^-24 relative.  1e-5 A leaves room for both.
"""
import pytest
import torch

from decay_reference import gradients, walk

pytestmark = pytest.mark.gpu
U = 2.0 ** -8
DEV = 'cuda'


def _inputs(seed, B, T, H, G, dk, dv, dtype, slow=9.0, state=True):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=DEV, generator=gen)  # noqa: E731
    q, k, v, do = r(B, T, H, dk), r(B, T, G, dk), r(B, T, G, dv), r(B, T, H, dv)
    g = torch.log1p(-torch.exp2(-torch.linspace(1.0, slow, H, device=DEV)))
    s0, ds = r(B, H, dk, dv), r(B, H, dk, dv)
    return [x.to(dtype) for x in (q, k, v, do)] + [g] + ([s0, ds] if state else [None, None])


def _near(got, ref, bound, what):
    assert got.shape == ref.shape, what
    off = (got.double() - ref).abs() - bound
    assert torch.isfinite(got).all(), what
    assert off.max() <= 1e-30 if off.numel() else True, f'{what}: {off.max().item():.3e} over the bound'


def _tol(dtype):
    return 2.1 * U if dtype == torch.bfloat16 else 1e-5


def _check(q, k, v, do, g, s0, ds, lengths=None, scale=None, grad=True):
    from bdm_b200 import decay_attention
    B, T, H, dk = q.shape
    n = lengths if lengths is not None else torch.full((B,), T, device=DEV)
    n = n.clamp(0, T)
    sc = dk ** -0.5 if scale is None else scale
    tol = _tol(q.dtype)
    leaves = [x.requires_grad_(True) for x in (q, k, v)] + ([s0.requires_grad_(True)] if s0 is not None else [])
    o, s = decay_attention(q, k, v, g, scale=scale, initial_state=s0, lengths=lengths, return_state=True)
    assert o.dtype == q.dtype and s.dtype == torch.float32
    ro, rs = walk(q, k, v, g, n, H, sc, s0)
    ao, as_ = walk(q, k, v, g, n, H, abs(sc), s0, absolute=True)
    _near(o.detach(), ro, tol * ao, 'o')
    _near(s.detach(), rs, 1e-5 * as_, 'state')
    if not grad:
        return
    if ds is not None:
        got = torch.autograd.grad((o, s), leaves, (do, ds))
    else:
        got = torch.autograd.grad(o, leaves, do)
    ref = gradients(q, k, v, do, g, n, sc, s0, ds)
    mag = gradients(q, k, v, do, g, n, abs(sc), s0, ds, absolute=True)
    for name, x, y, m, t in zip(('dq', 'dk', 'dv', 'ds0'), got, ref, mag, (tol, tol, tol, 1e-5)):
        _near(x, y, t * m, name)


# tokens around the chunk's edges, head widths around the tiles' and shared heads
SIZES = [(1, 1, 1, 1, 8, 8), (2, 2, 3, 3, 64, 64), (1, 63, 2, 1, 64, 128), (2, 64, 2, 2, 128, 128), (1, 65, 4, 2, 40, 72),
         (3, 127, 2, 2, 128, 64), (1, 128, 1, 1, 16, 24), (2, 200, 6, 2, 96, 120), (1, 1000, 2, 2, 64, 64),
         (1, 1536, 1, 1, 128, 128), (2, 777, 3, 1, 8, 128), (1, 70, 2, 2, 33, 5), (40, 130, 8, 8, 64, 64)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('size', SIZES)
def test_sequences_match_the_recurrence(size, dtype):
    _check(*_inputs(1, *size, dtype))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('size', [(4, 150, 4, 2, 64, 64), (5, 700, 2, 2, 128, 96), (4, 64, 2, 2, 64, 128)])
def test_ragged_rows_with_nan_padding(size, dtype):
    q, k, v, do, g, s0, ds = _inputs(2, *size, dtype)
    B, T = size[:2]
    n = torch.tensor([0, 1, T, T - 1, T // 2][:B], device=DEV)
    pad = (torch.arange(T, device=DEV) >= n[:, None])[:, :, None, None]
    for x in (q, k, v, do):
        x.masked_fill_(pad, float('nan'))
    _check(q, k, v, do, g, s0, ds, lengths=n)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_lengths_outside_the_tensor_are_clamped(dtype):
    q, k, v, do, g, s0, ds = _inputs(3, 3, 90, 2, 2, 64, 64, dtype)
    _check(q, k, v, do, g, s0, ds, lengths=torch.tensor([-5, 1 << 40, 33], device=DEV))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_no_state_and_scale(dtype):
    q, k, v, do, g, _, _ = _inputs(4, 2, 300, 4, 4, 64, 64, dtype, state=False)
    _check(q, k, v, do, g, None, None)
    _check(*_inputs(4, 2, 130, 2, 2, 64, 64, dtype), scale=-0.75)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('log_decay', [0.0, -1e-6, -0.7, -30.0, -200.0, float('-inf')])
def test_decays_from_none_to_total(log_decay, dtype):
    q, k, v, do, g, s0, ds = _inputs(5, 2, 260, 2, 2, 64, 64, dtype)
    _check(q, k, v, do, torch.full_like(g, log_decay), s0, ds)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_layouts(dtype):
    B, T, H, D = 2, 150, 4, 64
    q, k, v, do, g, s0, ds = _inputs(6, B, T, H, H, D, D, dtype)
    heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v, do)]
    _check(*heads_first, g, s0, ds)
    packed = torch.cat([x.flatten(2) for x in (q, k, v)], -1)  # as a fused projection leaves them
    a, b, c = (x.reshape(B, T, H, D) for x in packed.split(H * D, -1))
    _check(a.detach(), b.detach(), c.detach(), do, g, s0, ds)
    shifted = torch.empty(B * T * H * D + 1, dtype=dtype, device=DEV)[1:].reshape(B, T, H, D)  # no 16-byte alignment
    shifted.copy_(q)
    _check(shifted, k.detach(), v.detach(), do, g, s0, ds)
    columns = v.detach().transpose(-1, -2).contiguous().transpose(-1, -2)  # strided columns
    _check(q.detach(), k.detach(), columns, do, g, s0, ds)
    _check(q.detach(), k.detach()[:1].expand(B, -1, -1, -1).clone(), v.detach(), do.flip(1).flip(1), g, s0, ds)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_broadcast_inputs_and_their_gradients(dtype):
    from bdm_b200 import decay_attention
    q, k, v, do, g, _, _ = _inputs(7, 1, 100, 2, 2, 64, 64, dtype, state=False)
    do = torch.cat([do, do * 0.5])
    leaf = k.clone().requires_grad_(True)
    o = decay_attention(q.expand(2, -1, -1, -1), leaf.expand(2, -1, -1, -1), v.expand(2, -1, -1, -1), g)
    (got,) = torch.autograd.grad(o, leaf, do)
    n = torch.full((2,), 100, device=DEV)
    both = [x.expand(2, -1, -1, -1) for x in (q, k, v)]
    ref = gradients(*both, do, g, n, 64 ** -0.5)[1].sum(0, keepdim=True)
    mag = gradients(*both, do, g, n, 64 ** -0.5, absolute=True)[1].sum(0, keepdim=True)
    _near(got, ref, (_tol(dtype) + (U if dtype == torch.bfloat16 else 0)) * mag, 'dk')  # one more rounding: the sum over rows


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('size', [(2, 200, 4, 2, 64, 64), (1, 1100, 2, 2, 128, 128)])
def test_outputs_alone(size, dtype):
    """Without the state the BF16 walk rounds what it adds to the carried state to 17 bits, not 24: 2^-9 u A,
    far inside the bound of the outputs, which stays what it is."""
    from bdm_b200 import decay_attention
    q, k, v, do, g, s0, _ = _inputs(16, *size, dtype)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    o = decay_attention(q, k, v, g, initial_state=s0)
    got = torch.autograd.grad(o, leaves, do)
    H, sc, tol = size[2], size[4] ** -0.5, _tol(dtype)
    n = torch.full((size[0],), size[1], device=DEV)
    _near(o.detach(), walk(q, k, v, g, n, H, sc, s0)[0], tol * walk(q, k, v, g, n, H, sc, s0, absolute=True)[0], 'o')
    ref, mag = gradients(q, k, v, do, g, n, sc, s0), gradients(q, k, v, do, g, n, sc, s0, absolute=True)
    for name, x, y, m in zip(('dq', 'dk', 'dv'), got, ref, mag):
        _near(x, y, tol * m, name)


def test_gradient_through_the_state_alone():
    from bdm_b200 import decay_attention
    q, k, v, _, g, s0, ds = _inputs(17, 2, 90, 2, 1, 64, 64, torch.float32)
    leaves = [x.requires_grad_(True) for x in (k, v, s0)]
    _, s = decay_attention(q, k, v, g, initial_state=s0, return_state=True)
    got = torch.autograd.grad(s, leaves, ds)
    n, zero = torch.full((2,), 90, device=DEV), torch.zeros(2, 90, 2, 64, device=DEV)
    _, *ref = gradients(q, k, v, zero, g, n, 0.125, s0, ds)
    _, *mag = gradients(q, k, v, zero, g, n, 0.125, s0, ds, absolute=True)
    for x, y, m in zip(got, ref, mag):
        _near(x, y, 1e-5 * m, 'gradient')


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_many_ragged_rows(dtype):
    """More rows than fit one wave of CTAs, in every order of length."""
    B, T = 45, 150
    q, k, v, do, g, s0, ds = _inputs(18, B, T, 4, 4, 64, 64, dtype)
    gen = torch.Generator(device=DEV).manual_seed(19)
    n = torch.randint(0, T + 1, (B,), device=DEV, generator=gen)
    n[5] = n[6] = n[7]
    _check(q, k, v, do, g, s0, ds, lengths=n)


def test_no_tokens():
    from bdm_b200 import decay_attention
    for dtype in (torch.float32, torch.bfloat16):
        q, k, v, do, g, s0, ds = _inputs(8, 2, 0, 2, 2, 64, 64, dtype)
        o, s = decay_attention(q, k, v, g, initial_state=s0, return_state=True)
        assert o.shape == (2, 0, 2, 64) and torch.equal(s, s0)
        q, k, v, do, g, s0, ds = _inputs(8, 0, 5, 2, 2, 64, 64, dtype)
        assert decay_attention(q, k, v, g).shape == (0, 5, 2, 64)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_offsets_past_32_bits(dtype):
    """Rows further apart than 2^31 elements."""
    B, T, H, D = 2, 70, 2, 64
    q, k, v, do, g, s0, ds = _inputs(9, B, T, H, H, D, D, dtype)
    apart = (1 << 31) + 64
    far = torch.empty(apart + T * H * D, dtype=dtype, device=DEV).as_strided((B, T, H, D), (apart, H * D, D, 1))
    far.copy_(k)
    _check(q, far, v, do, g, s0, ds)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_gradient_against_differences(dtype):
    """o is linear in each of q, k, v and s0, so a central difference along a direction is exact up to the
    two evaluations' roundings (bounded as o is), whatever the step."""
    from bdm_b200 import decay_attention
    q, k, v, do, g, s0, _ = _inputs(10, 2, 140, 2, 1, 64, 64, dtype)
    leaves = [x.requires_grad_(True) for x in (q, k, v, s0)]
    o = decay_attention(q, k, v, g, initial_state=s0)
    grads = torch.autograd.grad(o, leaves, do)
    n = torch.full((2,), 140, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(11)
    for i, leaf in enumerate(leaves):
        d = (torch.randint(0, 2, leaf.shape, device=DEV, generator=gen) * 2 - 1).to(leaf.dtype)  # x +- d: d is what is added
        hi, lo = (leaf.detach() + d), (leaf.detach() - d)
        real = (hi.double() - lo.double())
        f, room = 0.0, 0.0
        for x, sign in ((hi, 1), (lo, -1)):
            args = [x if j == i else y.detach() for j, y in enumerate(leaves)]
            out = decay_attention(*args[:3], g, initial_state=args[3])
            f = f + sign * (out.double() * do.double()).sum()
            bound = _tol(dtype) * walk(*args[:3], g, n, 2, 64 ** -0.5, args[3], absolute=True)[0] * do.double().abs()
            room = room + bound.sum() / bound.numel() ** 0.5 * 4  # signs of single errors are independent
        mag = gradients(q, k, v, do, g, n, 64 ** -0.5, s0, torch.zeros_like(s0), absolute=True)[i]
        term = _tol(dtype) * mag * real.abs()
        room = room + term.sum() / term.numel() ** 0.5 * 4
        assert abs(f - (grads[i].double() * real).sum()) <= room, i


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('size', [(1, 1, 1, 8, 8), (3, 4, 2, 40, 72), (2, 3, 3, 33, 5), (64, 8, 8, 128, 128),
                                  (5, 2, 1, 200, 300), (4, 12, 12, 64, 64)])
def test_steps_match_the_recurrence(size, dtype):
    from bdm_b200 import decay_attention_step
    B, H, G, dk, dv = size
    T = 5
    q, k, v, _, g, s0, _ = _inputs(12, B, T, H, G, dk, dv, dtype)
    n = torch.full((B,), T, device=DEV)
    ro, rs = walk(q, k, v, g, n, H, dk ** -0.5, s0)
    ao, as_ = walk(q, k, v, g, n, H, dk ** -0.5, s0, absolute=True)
    s = s0.clone()
    o = torch.stack([decay_attention_step(q[:, t], k[:, t], v[:, t], g, s) for t in range(T)], 1)
    _near(o, ro, (1e-5 + (U if dtype == torch.bfloat16 else 0)) * ao, 'o')
    _near(s, rs, 1e-5 * as_, 'state')


def test_step_with_unaligned_state():
    from bdm_b200 import decay_attention_step
    q, k, v, _, g, s0, _ = _inputs(13, 2, 1, 2, 2, 16, 32, torch.float32)
    s = torch.empty(s0.numel() + 1, device=DEV)[1:].reshape(s0.shape).copy_(s0)
    o = decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g, s)
    n = torch.full((2,), 1, device=DEV)
    ro, rs = walk(q, k, v, g, n, 2, 0.25, s0)
    ao, as_ = walk(q, k, v, g, n, 2, 0.25, s0, absolute=True)
    _near(o[:, None], ro, 1e-5 * ao, 'o')
    _near(s, rs, 1e-5 * as_, 'state')


def test_side_stream_and_repeated_calls_agree():
    from bdm_b200 import decay_attention
    q, k, v, _, g, s0, _ = _inputs(14, 4, 513, 4, 4, 128, 128, torch.bfloat16)
    first = decay_attention(q, k, v, g, initial_state=s0, return_state=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = decay_attention(q, k, v, g, initial_state=s0, return_state=True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(first, second))


def test_first_call_of_a_thread():
    """A new thread (an autograd worker, say) has no current context until something makes it one."""
    import threading
    from bdm_b200 import decay_attention
    q, k, v, _, g, s0, _ = _inputs(20, 2, 200, 2, 2, 64, 64, torch.bfloat16)
    want = decay_attention(q, k, v, g, initial_state=s0)
    spare = torch.empty_like(want)
    del spare  # the allocator has a block for the output: the thread's first driver call is the walk's
    got = []
    worker = threading.Thread(target=lambda: got.append(decay_attention(q, k, v, g, initial_state=s0)))
    worker.start()
    worker.join()
    torch.cuda.synchronize()
    assert got and torch.equal(got[0], want)


def test_training_step_in_a_graph():
    from bdm_b200 import decay_attention
    q, k, v, do, g, _, _ = _inputs(21, 2, 300, 2, 1, 64, 64, torch.bfloat16, state=False)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    want = torch.autograd.grad(decay_attention(q, k, v, g), leaves, do)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(decay_attention(q, k, v, g), leaves, do)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_gradients_are_whole_when_the_next_kernel_starts():
    """dk and dv may start under dq's end; what follows in the stream must still see all three."""
    from bdm_b200 import decay_attention
    q, k, v, do, g, _, _ = _inputs(22, 24, 700, 8, 8, 64, 64, torch.bfloat16, state=False)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    o = decay_attention(q, k, v, g)
    torch.cuda.synchronize()
    want = [x.clone() for x in torch.autograd.grad(o, leaves, do, retain_graph=True)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = [x + 0 for x in torch.autograd.grad(o, leaves, do, retain_graph=True)]
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_refusals():
    from bdm_b200 import decay_attention, decay_attention_step
    q, k, v, _, g, s0, _ = _inputs(15, 2, 8, 4, 2, 16, 16, torch.float32)
    bad = [
        (ValueError, lambda: decay_attention(q.cpu(), k, v, g)),
        (ValueError, lambda: decay_attention(q.half(), k.half(), v.half(), g)),
        (ValueError, lambda: decay_attention(q.bfloat16(), k, v, g)),
        (ValueError, lambda: decay_attention(q[:, :, :3], k, v, g[:3])),
        (ValueError, lambda: decay_attention(q, k[:, :5], v, g)),
        (ValueError, lambda: decay_attention(q, k, v, g.double())),
        (ValueError, lambda: decay_attention(q, k, v, g[:2])),
        (ValueError, lambda: decay_attention(q, k, v, g.clone().requires_grad_(True))),
        (ValueError, lambda: decay_attention(q, k, v, g, scale=0.0)),
        (ValueError, lambda: decay_attention(q, k, v, g, initial_state=s0.bfloat16())),
        (ValueError, lambda: decay_attention(q, k, v, g, initial_state=s0[:1])),
        (ValueError, lambda: decay_attention(q, k, v, g, lengths=torch.tensor([1, 2, 3], device=DEV))),
        (ValueError, lambda: decay_attention(q, k, v, g, lengths=torch.tensor([1.0, 2.0], device=DEV))),
        (ValueError, lambda: decay_attention(q[0], k[0], v[0], g)),
        (NotImplementedError, lambda: decay_attention(*(torch.zeros(1, 2, 2, 136, device=DEV),) * 3, g[:2])),
        (ValueError, lambda: decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g, s0.transpose(2, 3))),
        (ValueError, lambda: decay_attention_step(q, k, v, g, s0)),
        (RuntimeError, lambda: decay_attention_step(q[:, 0].clone().requires_grad_(True), k[:, 0], v[:, 0], g, s0)),
    ]
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            pytest.fail(f'call {i} was accepted')
