"""States of long rows whose terms all have one sign and hardly decay: whatever a long sum loses adds up here.

The state is a sum of positive terms, so the absolute sum that bounds its roundings is itself.  The bound is the one
of every FP32 state, 1e-5 of it, where nothing decays (lam = 1, the first head).  Where lam^64 is not an FP32 number, a
chunk's carry is off by up to 2^-24 of it, the same way every time: 2^-24 more for every chunk of 64 tokens.  The
reference is the closed form sum_t lam^(n-1-t) k_t v_t^T in FP64.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'


# one long row (many segments), a few, as many as the GPU has SMs, and one row per SM and more (no segments)
@pytest.mark.parametrize('dtype,B,T,H,dk,dv', [
    (dtype, *size) for dtype in (torch.bfloat16, torch.float32)
    for size in [(1, 65536, 8, 128, 128), (1, 200000, 2, 64, 64), (8, 20000, 8, 64, 64), (1, 20000, 40, 64, 128),
                 (1, 9000, 148, 64, 64), (4, 30000, 4, 40, 72), (1, 65536, 74, 64, 64)]] + [(torch.bfloat16, 1, 400000, 8, 128, 128)])
def test_states_of_one_sign(B, T, H, dk, dv, dtype):
    from bdm_b200 import decay_attention
    gen = torch.Generator(device=DEV).manual_seed(41)
    r = lambda w: (torch.rand(B, T, H, w, device=DEV, generator=gen) + 0.5).to(dtype)  # noqa: E731
    q, k, v = r(dk), r(dk), r(dv)
    g = -torch.logspace(-7, -4, H, device=DEV)
    g[0] = 0.0
    _, s = decay_attention(q, k, v, g, return_state=True)
    w = torch.exp(g.double()[:, None] * (T - 1 - torch.arange(T, device=DEV)))  # [H, T]
    for b in range(B):
        for h in range(H):
            want = (k[b, :, h].double() * w[h][:, None]).T @ v[b, :, h].double()
            off = ((s[b, h].double() - want).abs() / want).max().item()
            assert off <= 1e-5 + (T / 64 * 2.0 ** -24 if h else 0), (b, h, off)


def test_gradient_of_the_initial_state_of_one_sign():
    from bdm_b200 import decay_attention
    gen = torch.Generator(device=DEV).manual_seed(42)
    B, T, H, D = 1, 40000, 4, 64
    q, k, v, do = ((torch.rand(B, T, H, D, device=DEV, generator=gen) + 0.5).bfloat16() for _ in range(4))
    g = -torch.logspace(-7, -4, H, device=DEV)
    g[0] = 0.0
    s0 = torch.zeros(B, H, D, D, device=DEV, requires_grad=True)
    (ds0,) = torch.autograd.grad(decay_attention(q, k, v, g, initial_state=s0), s0, do)
    w = torch.exp(g.double()[:, None] * (1 + torch.arange(T, device=DEV)))
    for h in range(H):
        want = (q[0, :, h].double() * w[h][:, None]).T @ do[0, :, h].double() * D ** -0.5
        assert ((ds0[0, h].double() - want).abs() / want).max().item() <= 1e-5 + (T / 64 * 2.0 ** -24 if h else 0), h
