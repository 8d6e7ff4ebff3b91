"""Beam selection and state reordering on the GPU against plain implementations on the CPU.

Scores are compared with the FP64 log-softmax at 4 roundings of 2^-24 of the largest magnitude in the sum
(log-sum-exp, the difference, the score's addition; the softmax sum's own error is below one of them).
Indices are compared exactly, on inputs whose candidates are either equal in exact arithmetic and in FP32,
or further apart than twice that error.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def _reference(logits, scores, finished, eos, stable):
    """Candidates in FP64, stable order; returns scores, parents, tokens, finished as lists of lists."""
    B, W, V = logits.shape
    x = logits.double().cpu()
    ok = torch.isfinite(x).any(-1) & ~(x.isnan() | (x == float('inf'))).any(-1)
    logp = torch.log_softmax(torch.where(ok[..., None], x, 0.0), -1)
    cand = torch.where(ok[..., None], scores.double().cpu()[..., None] + logp, float('-inf'))
    if finished is not None:
        held = torch.full_like(cand, float('-inf'))
        held[..., eos] = scores.double().cpu()
        cand = torch.where(finished.cpu()[..., None], held, cand)
    best, at = cand.reshape(B, W * V).sort(dim=-1, descending=True, stable=True)
    best, parents, tokens = best[:, :W], at[:, :W] // V, at[:, :W] % V
    if stable:
        for b in range(B):
            slots = [None] * W
            rest = []
            for r in range(W):
                p = int(parents[b, r])
                if slots[p] is None:
                    slots[p] = r
                else:
                    rest.append(r)
            for r in rest:
                slots[slots.index(None)] = r
            best[b], parents[b], tokens[b] = best[b, slots], parents[b, slots], tokens[b, slots]
    done = tokens == eos if eos is not None else torch.zeros_like(tokens, dtype=torch.bool)
    if finished is not None:
        done = done | finished.cpu().gather(1, parents)
    return best, parents, tokens, done


def _check(logits, scores, finished=None, eos=None):
    from bdm_b200 import beam_select
    for stable in (False, True):
        got = beam_select(logits, scores, finished=finished, eos_token=eos, stable_slots=stable)
        best, parents, tokens, done = _reference(logits, scores, finished, eos, stable)
        assert torch.equal(got.parents.cpu(), parents)
        assert torch.equal(got.tokens.cpu(), tokens)
        assert torch.equal(got.finished.cpu(), done)
        s = got.scores.cpu().double()
        assert torch.equal(torch.isfinite(s), torch.isfinite(best))
        fine = torch.isfinite(best)
        big = max(1.0, float(logits.float()[torch.isfinite(logits)].abs().max()) if torch.isfinite(logits).any() else 1.0,
                  float(scores[torch.isfinite(scores)].abs().max()) if torch.isfinite(scores).any() else 1.0) + 12
        assert ((s - best)[fine].abs() <= 4 * 2.0 ** -24 * 2 * big).all()


def _spread(seed, B, W, V, dtype):
    """Logits whose candidates are well apart: distinct multiples of a step, shuffled, offset by row."""
    gen = torch.Generator().manual_seed(seed)
    if dtype == torch.bfloat16:
        x = torch.randn(B, W, V, generator=gen).mul(3).to(dtype)
    else:
        x = torch.stack([torch.randperm(V, generator=gen) for _ in range(B * W)]).reshape(B, W, V) * (12.0 / V) - 6
    scores = -torch.rand(B, W, generator=gen).mul(9)
    return x.to(dtype).to(DEV), scores.to(DEV)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('B,W,V', [(1, 1, 1), (2, 1, 100), (3, 4, 192), (1, 4, 32000), (2, 8, 32000), (5, 32, 7), (2, 32, 4099),
                                   (1, 3, 70001), (70, 4, 9000), (3, 2, 1)])
def test_selection(B, W, V, dtype):
    x, s = _spread(B + W + V, B, W, V, dtype)
    _check(x, s)
    gen = torch.Generator().manual_seed(1)
    finished = (torch.rand(B, W, generator=gen) < 0.4).to(DEV)
    _check(x, s, finished, V // 2)
    _check(x, s, torch.ones_like(finished), 0)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('V', [5, 1000, 20011])
def test_ties_go_to_the_lowest_index(V, dtype):
    W = 4
    _check(torch.zeros(2, W, V, dtype=dtype, device=DEV), torch.zeros(2, W, device=DEV))
    gen = torch.Generator().manual_seed(2)
    x = torch.randint(0, 3, (1, 1, V), generator=gen).to(dtype).to(DEV).expand(3, W, V)
    _check(x, torch.zeros(3, W, device=DEV))
    _check(x, torch.tensor([[0.0, -1.0, 0.0, -64.0]], device=DEV).expand(3, W))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('V', [50, 9001])
def test_banned_tokens_and_broken_rows(V, dtype):
    inf = float('inf')
    x, s = _spread(3, 2, 6, V, dtype)
    x[:, :, ::3] = -inf
    x[0, 1] = -inf                                  # nothing allowed
    x[0, 2, V // 2] = float('nan')
    x[0, 3, V - 1] = inf
    x[1, 4] = torch.finfo(dtype).min                # the type's lowest value everywhere: uniform
    _check(x, s)
    s[0, 4] = -inf
    s[1, 0] = float('nan')
    _check_nan_score(x, s)
    x[0] = -inf                                     # a request without any candidate
    _check_nan_score(x, s)


def _check_nan_score(x, s):
    from bdm_b200 import beam_select
    clean = torch.where(s.isnan(), float('-inf'), s)
    for stable in (False, True):
        got, ref = beam_select(x, s, stable_slots=stable), beam_select(x, clean, stable_slots=stable)
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
    _check(x, clean)


def test_first_step_takes_all_beams_from_one():
    x, _ = _spread(4, 3, 5, 32000, torch.float32)
    s = torch.full((3, 5), float('-inf'), device=DEV)
    s[:, 0] = 0
    _check(x[:, :1].expand(-1, 5, -1), s)


def test_rounding_that_merges_candidates():
    """A score so large that whole stretches of logits round to one candidate: the lowest index wins, though
    its logit is not among the row's largest."""
    from bdm_b200 import beam_select
    V, W = 3000, 4
    gen = torch.Generator().manual_seed(5)
    x = torch.rand(2, W, V, generator=gen).to(DEV)
    for score in (-1e9, -3e4, -2e6):
        s = torch.full((2, W), score, device=DEV)
        got = beam_select(x, s)
        low = x - x.amax(-1, keepdim=True)
        cand = (s[..., None] + (low - low.exp().sum(-1, keepdim=True).log())).reshape(2, W * V)
        # a candidate's own rounding is the same everywhere: only rows' log-sum-exps could differ by an ulp,
        # which these scores absorb (their spacing is 2e-3 or more)
        best, at = cand.sort(dim=-1, descending=True, stable=True)
        if score != -3e4:
            assert torch.equal(got.parents * V + got.tokens, at[:, :W])
        assert torch.equal(got.scores, best[:, :W])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_concentrated_candidates(dtype):
    """The largest logits all in a few threads' hands."""
    V, W = 32000, 32
    x, s = _spread(6, 2, W, V, dtype)
    x[:, :, 512:512 + 24 * 8] = (torch.arange(24 * 8, device=DEV) * 0.125 + 8).to(dtype)
    x[:, 3, 4096:4096 + 2000] = 40.0
    _check(x, s)


def test_strided_logits():
    x, s = _spread(7, 3, 4, 1001, torch.float32)
    wide = torch.full((3, 4, 1100), 99.0, device=DEV)
    wide[..., 3:1004] = x
    _check(wide[..., 3:1004], s)
    _check(x.transpose(1, 2).contiguous().transpose(1, 2), s)


def test_selection_refusals():
    from bdm_b200 import beam_select
    x, s = torch.zeros(2, 3, 10, device=DEV), torch.zeros(2, 3, device=DEV)
    done = torch.zeros(2, 3, dtype=torch.bool, device=DEV)
    for kind, call in [
        (ValueError, lambda: beam_select(x.cpu(), s)),
        (ValueError, lambda: beam_select(x.half(), s)),
        (ValueError, lambda: beam_select(x, s[:1])),
        (ValueError, lambda: beam_select(x, s.double())),
        (ValueError, lambda: beam_select(x, s, finished=done)),
        (ValueError, lambda: beam_select(x, s, finished=done.long(), eos_token=1)),
        (ValueError, lambda: beam_select(x, s, eos_token=10)),
        (ValueError, lambda: beam_select(x[:, :, :0], s)),
        (NotImplementedError, lambda: beam_select(torch.zeros(1, 33, 4, device=DEV), torch.zeros(1, 33, device=DEV))),
    ]:
        with pytest.raises(kind):
            call()


# ------------------------------------------------------------------- reordering

@pytest.mark.parametrize('W', [1, 2, 4, 5, 8, 13, 32])
@pytest.mark.parametrize('B', [1, 3])
def test_reordering(B, W):
    from bdm_b200 import reorder_states
    gen = torch.Generator().manual_seed(W)
    rows = B * W
    states = [torch.randn(rows, 16, 1, 8, 64, generator=gen).bfloat16().to(DEV), torch.randn(rows, 3, 40, 72, generator=gen).to(DEV),
              torch.randint(0, 255, (rows, 7), generator=gen, dtype=torch.uint8).to(DEV), torch.arange(rows, device=DEV),
              torch.randn(rows, 20000, generator=gen).to(DEV), torch.randn(rows, 33, generator=gen).bfloat16().to(DEV),
              torch.zeros(rows, 0, device=DEV), torch.randn(rows, 9, generator=gen).to(DEV)[:, :5]]
    for parents in (torch.randint(0, W, (B, W), generator=gen), torch.arange(W).repeat(B, 1), torch.zeros(B, W, dtype=torch.long),
                    torch.arange(W).flip(0).repeat(B, 1), torch.arange(W).roll(1).repeat(B, 1)):
        flat = (parents + W * torch.arange(B)[:, None]).reshape(-1).to(DEV)
        want = [s.clone().index_select(0, flat) for s in states]
        assert reorder_states(states, parents.to(DEV)) is states
        assert all(torch.equal(a, b) for a, b in zip(states, want))


def test_reordering_many_tensors_and_rows_past_32_bits():
    from bdm_b200 import reorder_states
    parents = torch.tensor([[1, 0]], device=DEV)
    many = [torch.full((2, 5), float(i), device=DEV) + torch.arange(2, device=DEV)[:, None] for i in range(70)]
    want = [m.flip(0) for m in many]
    reorder_states(many, parents)
    assert all(torch.equal(a, b) for a, b in zip(many, want))
    wide = torch.empty((2, (1 << 31) + 40), dtype=torch.uint8, device=DEV)
    wide[0].fill_(3)
    wide[1].fill_(9)
    wide[1, -1] = 77
    reorder_states([wide], parents)
    assert int(wide[0, -1]) == 77 and int(wide[0, -2]) == 9 and int(wide[1].max()) == 3 and int(wide[1].min()) == 3


def test_parents_out_of_range_keep_the_row_and_set_the_status():
    from bdm_b200 import ops, reorder_states
    from bdm_b200._lib import BDMError
    s = torch.arange(6.0, device=DEV).reshape(3, 2)
    want = s.clone()[[0, 1, 1]]
    reorder_states([s], torch.tensor([[-1, 3, 1]], device=DEV))
    assert torch.equal(s, want)
    with pytest.raises(BDMError):
        ops.check_scan_status(wait=True)
    ops.reset_scan_status()
    ops.check_scan_status(wait=True)


def test_reordering_refusals():
    from bdm_b200 import reorder_states
    p = torch.zeros(2, 2, dtype=torch.long, device=DEV)
    s = torch.zeros(4, 6, device=DEV)
    for kind, call in [
        (ValueError, lambda: reorder_states([s.cpu()], p)),
        (ValueError, lambda: reorder_states([s[:3]], p)),
        (ValueError, lambda: reorder_states([s], p.int())),
        (ValueError, lambda: reorder_states([s], p[0])),
        (ValueError, lambda: reorder_states([s, s], p)),
        (ValueError, lambda: reorder_states([s[:, ::2]], p)),
        (ValueError, lambda: reorder_states([torch.zeros(6, device=DEV).expand(4, 6)], p)),
        (RuntimeError, lambda: reorder_states([s.clone().requires_grad_(True)], p)),
        (NotImplementedError, lambda: reorder_states([torch.zeros(33, 2, device=DEV)], torch.zeros(1, 33, dtype=torch.long, device=DEV))),
    ]:
        with pytest.raises(kind):
            call()


# ---------------------------------------------------------------- the whole search

def _model(dtype=torch.float32):
    from bdm_b200 import BSDMConfig, HybridLanguageModel, LanguageModelConfig
    mem = BSDMConfig(dim=64, bank_count=64, bank_size=8, selected_banks=4, value_width=64, num_heads=2,
                     training_state_dtype='float32')
    return HybridLanguageModel(LanguageModelConfig(memory=mem, vocab_size=50, layers=2, seed=3)).to(dtype).to(DEV)


def test_hybrid_model_trains_and_steps_like_its_prompt():
    m = _model()
    gen = torch.Generator().manual_seed(8)
    tokens = torch.randint(0, 50, (2, 70), generator=gen).to(DEV)
    loss = m(tokens[:, :-1], tokens[:, 1:])
    loss.backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters() if p.requires_grad)
    with torch.inference_mode():
        whole = m(tokens)
        _, caches = m.prefill(tokens[:, :60], state_dtype=torch.float32)
        for t in range(60, 70):
            logits = m.step(tokens[:, t:t + 1], caches)
            # two FP32 evaluations of one function: the LM shell's own bound
            assert (logits[:, 0] - whole[:, t]).abs().max() <= 1e-4 * whole.abs().max()


def test_beam_search_equals_a_plain_search():
    """Against a search that re-evaluates every prefix with the full forward and keeps plain lists."""
    from bdm_b200 import beam_search
    m = _model()
    gen = torch.Generator().manual_seed(9)
    prompt = torch.randint(0, 50, (2, 12), generator=gen).to(DEV)
    W, N, eos = 3, 5, 7
    with torch.inference_mode():
        got, scores = beam_search(m, prompt, beams=W, max_new_tokens=N, eos_token=eos)
        assert got.shape == (2, W, N)
        for b in range(2):
            live = [([], 0.0, False)]
            for _ in range(N):
                cand = []
                for seq, sc, done in live:
                    if done:
                        cand.append((sc, seq + [eos], True))
                        continue
                    ids = torch.cat([prompt[b], torch.tensor(seq, dtype=torch.long, device=DEV)])[None]
                    logp = torch.log_softmax(m(ids)[0, -1].double(), -1).cpu()
                    cand += [(sc + float(logp[t]), seq + [t], t == eos) for t in range(50)]
                cand.sort(key=lambda c: -c[0])
                live = [(seq, sc, done) for sc, seq, done in cand[:W]]
            for w in range(W):
                assert got[b, w].tolist() == live[w][0]
                assert abs(float(scores[b, w]) - live[w][1]) <= 1e-2  # BF16 caches of the bank layers
