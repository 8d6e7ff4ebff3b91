"""Workloads of the recurrent-decoder operators: linear attention with a decay for each head (prompt,
training and single-token forms), beam selection and the in-place reordering of the decoder's states.

``run`` computes an operator in its plain form (elementary torch operations, FP32) or, with ``own``,
through the framework's entry points; ``exact`` restates its definition token by token in FP64.
"""
import math

import torch

own = False

DTYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16}
DEV = 'cuda'


def listed():
    return [
        # A chat-sized prompt of one request through one 12-head layer: launch latency counts.
        dict(name='prompt_short', op='prefill', batch=1, time=37, heads=12, kv_heads=12, dk=64, dv=64,
             dtype='bfloat16', ragged=False, state=False),
        # The layer benchmark's prefill: batch 8 x 4096 tokens, 8 heads of 128.
        dict(name='prompt_layer', op='prefill', batch=8, time=4096, heads=8, kv_heads=8, dk=128, dv=128,
             dtype='bfloat16', ragged=False, state=False),
        # One long document: few sequences, so the time axis itself has to be split.
        dict(name='prompt_long', op='prefill', batch=1, time=65536, heads=8, kv_heads=8, dk=128, dv=128,
             dtype='bfloat16', ragged=False, state=True),
        # A served batch of prompts of unequal length (one of them empty), continued from states,
        # with keys and values shared by groups of heads and head widths that fill no tile.
        dict(name='prompt_ragged', op='prefill', batch=24, time=1333, heads=8, kv_heads=2, dk=96, dv=120,
             dtype='bfloat16', ragged=True, state=True),
        # Gradients in FP32 at odd sizes: ragged rows, shared heads, states in and out.
        dict(name='train_fp32', op='train', batch=3, time=777, heads=6, kv_heads=2, dk=40, dv=72,
             dtype='float32', ragged=True, state=True),
        # One layer of the 12-layer language model's training step: batch 32 x 2048, 12 heads of 64.
        dict(name='train_lm', op='train', batch=32, time=2048, heads=12, kv_heads=12, dk=64, dv=64,
             dtype='bfloat16', ragged=False, state=False),
        # One token of one request.
        dict(name='step_one', op='step', batch=1, heads=12, kv_heads=12, dk=64, dv=64, dtype='bfloat16'),
        # One token of 64 requests with 4 beams each.
        dict(name='step_beams', op='step', batch=256, heads=8, kv_heads=8, dk=128, dv=128, dtype='bfloat16'),
        # Beam step of one request over the language model's vocabulary, FP32 logits.
        dict(name='beam_one', op='beam', batch=1, beams=4, vocab=32000, dtype='float32', stable=False),
        # Beam step of a served batch; survivors keep their cache slots.
        dict(name='beam_batch', op='beam', batch=64, beams=8, vocab=32000, dtype='bfloat16', stable=True),
        # Reordering of one request's 4 beams by rank: one layer's bank cache and one FP32 state.
        dict(name='reorder_one', op='reorder', batch=1, beams=4, layers=1, banks=512, heads=12, bank_size=8,
             width=64, moved=2, stable=False),
        # Reordering of 16 requests with 4 beams over two layers' bank caches and FP32 states.
        dict(name='reorder_batch', op='reorder', batch=16, beams=4, layers=2, banks=512, heads=12, bank_size=8,
             width=64, moved=2, stable=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['prefill', 'prefill', 'train', 'train', 'step', 'beam', 'reorder'])
    dtype = rng.choice(['bfloat16', 'bfloat16', 'float32'])
    groups, kv = rng.choice([1, 1, 1, 2, 4]), rng.randint(1, 6)
    dk, dv = rng.choice([(64, 64), (128, 128), (8 * rng.randint(2, 16), 8 * rng.randint(2, 16))])
    heads = kv * groups
    if op in ('prefill', 'train'):
        time = _log(rng, 1, 20000)
        # at most the largest listed case's tokens times heads for its direction
        most = (2 ** 19 if op == 'prefill' else 2 ** 18) // (4 if dtype == 'float32' else 1)
        batch = _log(rng, 1, max(1, min(48, most // (time * heads))))
        time = max(1, min(time, most // (batch * heads)))
        return dict(op=op, batch=batch, time=time, heads=heads, kv_heads=kv, dk=dk, dv=dv, dtype=dtype,
                    ragged=rng.random() < 0.5, state=rng.random() < 0.5)
    if op == 'step':
        return dict(op=op, batch=_log(rng, 1, 256 * 8 // heads // 2), heads=heads, kv_heads=kv, dk=dk, dv=dv, dtype=dtype)
    beams = rng.randint(2, 16)
    if op == 'beam':
        return dict(op=op, batch=_log(rng, 1, 512 // beams), beams=beams, vocab=_log(rng, 100, 32000), dtype=dtype,
                    stable=rng.random() < 0.5)
    return dict(op=op, batch=_log(rng, 1, 96 // beams), beams=beams, layers=rng.randint(1, 2), banks=_log(rng, 64, 256),
                heads=rng.choice([1, 4, 8]), bank_size=rng.choice([4, 8, 16]), width=64,
                moved=rng.randint(1, beams - 1), stable=rng.random() < 0.5)


# ------------------------------------------------------------------ inputs

def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) % (2 ** 62))


def _unit(gen, *shape, dtype):
    """Queries and keys as the layer makes them: SiLU, then a unit norm over the head."""
    x = torch.nn.functional.silu(torch.randn(*shape, device=DEV, generator=gen))
    return (x / x.square().sum(-1, keepdim=True).sqrt().clamp_min(1e-6)).to(dtype)


def _decays(gen, heads):
    """log(1 - 2^-e) with e spread over 3 .. 9, the slopes from short to long memory, jittered by the seed."""
    e = torch.linspace(3, 9, heads, device=DEV) + torch.rand(heads, device=DEV, generator=gen) * 0.5
    return torch.log1p(-torch.exp2(-e))


def _parents(gen, batch, beams, moved, stable):
    """Parents as a beam step gives them: ``moved`` beams of each request die, and survivors take their places."""
    order = torch.rand(batch, beams, device=DEV, generator=gen).argsort(-1)
    dead, alive = order[:, :moved], order[:, moved:]
    source = alive[:, torch.arange(moved, device=DEV) % (beams - moved)]
    p = torch.arange(beams, device=DEV).repeat(batch, 1).scatter(1, dead, source)
    return p if stable else p.gather(1, torch.rand(batch, beams, device=DEV, generator=gen).argsort(-1))


def prepare(case, seed):
    gen = _generator(seed)
    c = dict(case)
    rand = lambda *s, dtype=torch.float32: torch.randn(*s, device=DEV, generator=gen, dtype=dtype)  # noqa: E731
    if c['op'] in ('prefill', 'train', 'step'):
        dt = DTYPES[c['dtype']]
        B, H, G, dk, dv = c['batch'], c['heads'], c['kv_heads'], c['dk'], c['dv']
        lead = (B, c['time']) if c['op'] != 'step' else (B,)
        c['g'] = _decays(gen, H)
        c['q'], c['k'] = _unit(gen, *lead, H, dk, dtype=dt), _unit(gen, *lead, G, dk, dtype=dt)
        c['v'] = rand(*lead, G, dv, dtype=dt)
        c['s0'] = rand(B, H, dk, dv) * 0.3 if c['op'] == 'step' or c['state'] else None
        c['lengths'] = None
        if c.get('ragged'):
            # uniform over 0 .. T, one row empty where there are several, and one full
            n = torch.randint(0, c['time'] + 1, (B,), device=DEV, generator=gen)
            n[-1] = c['time']
            n[:-1][:1] = 0
            c['lengths'] = n
        if c['op'] == 'train':
            c['do'] = rand(*lead, H, dv, dtype=dt)
            c['ds'] = rand(B, H, dk, dv) * 0.3 if c['state'] else None
            c['q'], c['k'], c['v'] = (x.requires_grad_(True) for x in (c['q'], c['k'], c['v']))
            if c['state']:
                c['s0'].requires_grad_(True)
    elif c['op'] == 'beam':
        B, W, V = c['batch'], c['beams'], c['vocab']
        c['logits'] = (rand(B, W, V) * 2.5).to(DTYPES[c['dtype']])
        banned = torch.rand(V, device=DEV, generator=gen) < 0.02
        c['logits'].masked_fill_(banned, float('-inf'))
        c['scores'] = -(torch.rand(B, W, device=DEV, generator=gen) * 8).cumsum(-1)
        c['finished'] = torch.rand(B, W, device=DEV, generator=gen) < 0.15
        c['eos'] = V // 2
    else:
        rows = c['batch'] * c['beams']
        c['parents'] = _parents(gen, c['batch'], c['beams'], c['moved'], c['stable'])
        c['states'] = [rand(rows, c['banks'], c['heads'], c['bank_size'], c['width'], dtype=torch.bfloat16)
                       for _ in range(c['layers'])]
        c['states'] += [rand(rows, c['heads'], c['width'], c['width']) for _ in range(c['layers'])]
    return c


# -------------------------------------------------------------- plain forms

CHUNK = 128


def _walk(a, b, c, g):
    """out[t] = sum over s <= t of exp(g (t - s)) (a[t] . b[s]) c[s], chunk by chunk: FP32 [B, H, T, *]."""
    B, H, T, _ = a.shape
    n = -(-T // CHUNK)
    a, b, c = (torch.nn.functional.pad(x, (0, 0, 0, n * CHUNK - T)).reshape(B, H, n, CHUNK, -1) for x in (a, b, c))
    g = g.reshape(1, H, 1, 1, 1)
    i = torch.arange(CHUNK, device=a.device, dtype=torch.float32)
    inner = torch.where(i[:, None] >= i, torch.exp(g * (i[:, None] - i).clamp_min(0)), 0.0)
    out = ((a @ b.transpose(-1, -2)) * inner) @ c
    if n > 1:
        # state before every chunk: the chunks' own sums, mixed by a triangular matrix of decays
        z = (b * torch.exp(g * (CHUNK - 1 - i)[:, None])).transpose(-1, -2) @ c
        m = torch.arange(n, device=a.device, dtype=torch.float32)
        mix = torch.where(m[:, None] > m, torch.exp(g[:, :, 0] * CHUNK * (m[:, None] - 1 - m).clamp_min(0)), 0.0)
        s = (mix @ z.reshape(B, H, n, -1)).reshape(z.shape)
        out = out + torch.exp(g * (i + 1)[:, None]) * (a @ s)
    return out.reshape(B, H, n * CHUNK, -1)[:, :, :T]


def _per_head(x, heads):
    """[B, T, G, D] -> FP32 [B, H, T, D], shared heads repeated."""
    return x.detach().float().repeat_interleave(heads // x.shape[2], 2).transpose(1, 2)


def _plain_attention(c):
    B, T, H, dk = c['q'].shape
    scale, g = dk ** -0.5, c['g']
    t = torch.arange(T, device=g.device)
    n = c['lengths'] if c['lengths'] is not None else torch.full((B,), T, device=g.device)
    valid = (t < n[:, None])[:, None, :, None]
    q, k, v = (torch.where(valid, _per_head(c[x], H), 0.0) for x in 'qkv')
    since = torch.exp(g[:, None] * (t + 1)).reshape(1, H, T, 1)                # from the given state to token t
    left = torch.exp(g[:, None] * (n[:, None, None] - 1 - t).clamp_min(0))[..., None]  # from token t to the end
    whole = torch.exp(g * n[:, None])[..., None, None]                         # over the row's valid tokens
    s0 = c['s0'].detach() if c['s0'] is not None else None
    o = _walk(q, k, v, g)
    if s0 is not None:
        o = o + since * (q @ s0)
    state = (k * left).transpose(-1, -2) @ v
    if s0 is not None:
        state = state + whole * s0
    dt = c['q'].dtype
    out = {'o': torch.where(valid, scale * o, 0.0).transpose(1, 2).to(dt), 'state': state}
    if c['op'] == 'prefill':
        return out
    do, ds = torch.where(valid, _per_head(c['do'], H), 0.0), c['ds']
    flip = lambda x: x.flip(2)  # noqa: E731
    dq = _walk(do, v, k, g)
    dk_ = flip(_walk(flip(v), flip(do), flip(q), g)) * scale
    dv_ = flip(_walk(flip(k), flip(q), flip(do), g)) * scale
    if s0 is not None:
        dq = dq + since * (do @ s0.transpose(-1, -2))
        dk_ = dk_ + left * (v @ ds.transpose(-1, -2))
        dv_ = dv_ + left * (k @ ds)
        out['ds0'] = scale * ((q * since).transpose(-1, -2) @ do) + whole * ds
    G = c['k'].shape[2]
    group = lambda x: torch.where(valid, x, 0.0).reshape(B, G, H // G, T, -1).sum(2).transpose(1, 2).to(dt)  # noqa: E731
    out.update(dq=torch.where(valid, scale * dq, 0.0).transpose(1, 2).to(dt), dk=group(dk_), dv=group(dv_))
    return out


def _plain_step(c):
    H = c['q'].shape[1]
    k, v = (c[x].float().repeat_interleave(H // c[x].shape[1], 1) for x in 'kv')
    s = c['s0'].mul_(torch.exp(c['g'])[None, :, None, None]).add_(k[..., None] * v[..., None, :])
    o = (c['q'].float()[..., None] * s).sum(-2) * c['q'].shape[-1] ** -0.5
    return {'o': o.to(c['q'].dtype), 'state': s}


def _plain_beam(c):
    x, scores, eos = c['logits'].float(), c['scores'], c['eos']
    B, W, V = x.shape
    top = x.amax(-1, keepdim=True)
    cand = scores[..., None] + ((x - top) - torch.exp(x - top).sum(-1, keepdim=True).log())
    done = torch.full_like(cand, float('-inf'))
    done[..., eos] = scores
    cand = torch.where(c['finished'][..., None], done, cand)
    best, at = torch.where(cand.isnan(), float('-inf'), cand).reshape(B, W * V).sort(dim=-1, descending=True, stable=True)
    best, at = best[:, :W], at[:, :W]
    parents, tokens = at // V, at % V
    if c['stable']:
        # the first child of a parent takes the parent's slot, the others the free slots in turn
        same = parents[:, :, None] == parents[:, None, :]
        first = ~torch.tril(same, -1).any(-1)
        taken = torch.zeros(B, W, dtype=torch.bool, device=x.device).scatter(1, parents, True)
        free = taken.to(torch.int8).sort(dim=-1, stable=True).indices
        slot = torch.where(first, parents, free.gather(1, ((~first).long().cumsum(-1) - 1).clamp_min(0)))
        rank = slot.argsort(-1)
        best, parents, tokens = (y.gather(1, rank) for y in (best, parents, tokens))
    return {'scores': best, 'parents': parents, 'tokens': tokens,
            'finished': c['finished'].gather(1, parents) | (tokens == eos)}


def _plain_reorder(c):
    B, W = c['parents'].shape
    rows = (c['parents'] + W * torch.arange(B, device=c['parents'].device)[:, None]).reshape(-1)
    return [s.copy_(s.index_select(0, rows)) for s in c['states']]


def run(state):
    c = state
    if not own:
        plain = {'prefill': _plain_attention, 'train': _plain_attention, 'step': _plain_step, 'beam': _plain_beam,
                 'reorder': _plain_reorder}
        return plain[c['op']](c)
    import bdm_b200
    if c['op'] == 'prefill':
        o, s = bdm_b200.decay_attention(c['q'], c['k'], c['v'], c['g'], initial_state=c['s0'], lengths=c['lengths'],
                                        return_state=True)
        return {'o': o, 'state': s}
    if c['op'] == 'train':
        o, s = bdm_b200.decay_attention(c['q'], c['k'], c['v'], c['g'], initial_state=c['s0'], lengths=c['lengths'],
                                        return_state=True)
        out = {'o': o.detach(), 'state': s.detach()}
        if c['s0'] is None:
            grads = torch.autograd.grad(o, (c['q'], c['k'], c['v']), c['do'])
        else:
            grads = torch.autograd.grad((o, s), (c['q'], c['k'], c['v'], c['s0']), (c['do'], c['ds']))
            out['ds0'] = grads[3]
        out.update(dq=grads[0], dk=grads[1], dv=grads[2])
        return out
    if c['op'] == 'step':
        o = bdm_b200.decay_attention_step(c['q'], c['k'], c['v'], c['g'], c['s0'])
        return {'o': o, 'state': c['s0']}
    if c['op'] == 'beam':
        b = bdm_b200.beam_select(c['logits'], c['scores'], finished=c['finished'], eos_token=c['eos'],
                                 stable_slots=c['stable'])
        return {'scores': b.scores, 'parents': b.parents, 'tokens': b.tokens, 'finished': b.finished}
    bdm_b200.reorder_states(c['states'], c['parents'])
    return c['states']


# ------------------------------------------------------------------- work

def work(case):
    c = case
    if c['op'] in ('prefill', 'train', 'step'):
        size, tokens = (4 if c['dtype'] == 'float32' else 2), c['batch'] * c.get('time', 1)
        qo, kv = tokens * c['heads'] * size, tokens * c['kv_heads'] * size
        state = c['batch'] * c['heads'] * c['dk'] * c['dv'] * 4
        given = c['op'] == 'step' or c['state']
        flops = tokens * c['heads'] * c['dk'] * c['dv']
        nbytes = (qo + kv) * (c['dk'] + c['dv']) + state * (2 if given else 1)
        if c['op'] != 'train':
            return {'bytes': nbytes, 'flops': 4 * flops}
        # the gradient of o read, those of q, k and v written; state recomputed, its adjoint, three products
        nbytes += qo * (c['dv'] + c['dk']) + kv * (c['dk'] + c['dv']) + (2 * state if given else 0)
        return {'bytes': nbytes, 'flops': 14 * flops}
    if c['op'] == 'beam':
        n = c['batch'] * c['beams']
        return {'bytes': n * c['vocab'] * (4 if c['dtype'] == 'float32' else 2) + n * 26, 'flops': n * c['vocab'] * 3}
    row = c['layers'] * (c['banks'] * c['heads'] * c['bank_size'] * c['width'] * 2 + c['heads'] * c['width'] ** 2 * 4)
    w, m = c['beams'], c['moved']
    # stable: the dead rows are written from as many survivors; by rank: every row is written from the survivors
    rows = m + min(m, w - m) if c['stable'] else w + (w - m)
    return {'bytes': c['batch'] * rows * row, 'flops': 0}


# -------------------------------------------- definitions in 64 bits, token by token

def _exact_attention(c):
    B, T, H, dk = c['q'].shape
    dv, G = c['v'].shape[-1], c['k'].shape[2]
    D = torch.float64
    lam = torch.exp(c['g'].to(D)).reshape(1, H, 1, 1)
    n = c['lengths'] if c['lengths'] is not None else torch.full((B,), T, device=DEV)
    n = n.reshape(B, 1, 1, 1)
    train = c['op'] == 'train'
    up = lambda x, t: x[:, t].detach().to(D).repeat_interleave(H // x.shape[2], 1)  # noqa: E731
    S = c['s0'].detach().to(D) if c['s0'] is not None else torch.zeros(B, H, dk, dv, dtype=D, device=DEV)
    o, dq = (torch.zeros(B, T, H, w, dtype=D, device=DEV) for w in (dv, dk))
    scale = dk ** -0.5
    for t in range(T):
        live = t < n
        S = torch.where(live, lam * S + up(c['k'], t)[..., None] * up(c['v'], t)[..., None, :], S)
        o[:, t] = torch.where(live[..., 0], (up(c['q'], t)[..., None, :] @ S)[..., 0, :] * scale, 0.0)
        if train:
            dq[:, t] = torch.where(live[..., 0], (S @ up(c['do'], t)[..., None])[..., 0] * scale, 0.0)
    out = {'o': o, 'state': S}
    if not train:
        return out
    R = c['ds'].to(D) if c['ds'] is not None else torch.zeros(B, H, dk, dv, dtype=D, device=DEV)
    dk_, dv_ = (torch.zeros(B, T, G, w, dtype=D, device=DEV) for w in (dk, dv))
    for t in reversed(range(T)):
        live = t < n
        # R: gradient of the state after token t
        A = R + scale * up(c['q'], t)[..., None] * up(c['do'], t)[..., None, :]
        gk, gv = (A @ up(c['v'], t)[..., None])[..., 0], (up(c['k'], t)[..., None, :] @ A)[..., 0, :]
        dk_[:, t] = torch.where(live[..., 0], gk, 0.0).reshape(B, G, H // G, dk).sum(2)
        dv_[:, t] = torch.where(live[..., 0], gv, 0.0).reshape(B, G, H // G, dv).sum(2)
        R = torch.where(live, lam * A, R)
    out.update(dq=dq, dk=dk_, dv=dv_)
    if c['s0'] is not None:
        out['ds0'] = R
    return out


def exact(case, seed):
    c = prepare(case, seed)
    D = torch.float64
    if c['op'] in ('prefill', 'train'):
        return _exact_attention(c)
    if c['op'] == 'step':
        H = c['heads']
        q, k, v = (c[x].to(D) for x in 'qkv')
        k, v = (x.repeat_interleave(H // x.shape[1], 1) for x in (k, v))
        S = torch.exp(c['g'].to(D)).reshape(1, H, 1, 1) * c['s0'].to(D) + torch.einsum('bhk,bhv->bhkv', k, v)
        return {'o': torch.einsum('bhk,bhkv->bhv', q, S) / math.sqrt(c['dk']), 'state': S}
    if c['op'] == 'beam':
        W, V = c['beams'], c['vocab']
        logp = torch.log_softmax(c['logits'].to(D), -1) + c['scores'].to(D)[..., None]
        keep = torch.zeros(V, dtype=torch.bool, device=DEV)
        keep[c['eos']] = True
        held = torch.where(keep, c['scores'].to(D)[..., None], float('-inf'))
        best = torch.where(c['finished'][..., None], held, logp).flatten(1).topk(W, -1)
        if not c['stable']:
            return {'scores': best.values, 'parents': None, 'tokens': None, 'finished': None}
        scores = torch.zeros(c['batch'], W, dtype=D)
        values, parents = best.values.cpu(), (best.indices // V).cpu().tolist()
        for b in range(c['batch']):
            slots = [None] * W
            later = []
            for r, p in enumerate(parents[b]):
                if slots[p] is None:
                    slots[p] = r
                else:
                    later.append(r)
            for r in later:
                slots[slots.index(None)] = r
            scores[b] = values[b, slots]
        return {'scores': scores, 'parents': None, 'tokens': None, 'finished': None}
    return None  # a reordering copies: nothing is computed
