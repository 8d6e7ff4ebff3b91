"""Decay attention token by token in FP64 (the tests' plain implementation), and error bounds for it."""
import torch


def _up(x, heads):
    return x.detach().double().repeat_interleave(heads // x.shape[2], 2)


def walk(a, b, c, g, n, heads, scale, s0=None, reverse=False, absolute=False):
    """out [B, T, H, wc] and the final state [B, H, wab, wc] of one walk.  a, b, c [B, T, *, width], g [H],
    n [B] valid tokens.  ``absolute``: the same sums over absolute values, which bound every rounding."""
    a, b, c = (_up(x, heads) for x in (a, b, c))
    B, T = a.shape[:2]
    mag = (lambda x: x.abs()) if absolute else (lambda x: x)
    a, b, c = (torch.where((torch.arange(T, device=x.device) < n[:, None])[:, :, None, None], mag(x), 0.0)
               for x in (a, b, c))
    lam = torch.exp(g.double()).reshape(1, heads, 1, 1)
    S = torch.zeros(B, heads, a.shape[3], c.shape[3], dtype=torch.float64, device=a.device)
    if s0 is not None:
        S = mag(s0.detach().double())
    out = torch.zeros(B, T, heads, c.shape[3], dtype=torch.float64, device=a.device)
    for t in (reversed(range(T)) if reverse else range(T)):
        live = (t < n).reshape(B, 1, 1, 1)
        w = b[:, t, :, :, None] * c[:, t, :, None, :]
        if not reverse:
            S = torch.where(live, lam * S + w, S)
            out[:, t] = torch.where(live[..., 0], (a[:, t, :, None, :] @ S)[..., 0, :] * scale, 0.0)
        else:
            A = S + w
            out[:, t] = torch.where(live[..., 0], (a[:, t, :, None, :] @ A)[..., 0, :] * scale, 0.0)
            S = torch.where(live, lam * A, S)
    return out, S


def gradients(q, k, v, do, g, n, scale, s0=None, ds=None, absolute=False):
    """dq, dk, dv, ds0 of sum(o * do) + sum(state * ds), by the formulas of the reverse recurrence."""
    H, G = q.shape[2], k.shape[2]
    t = lambda s: None if s is None else s.transpose(-1, -2)  # noqa: E731
    dq, _ = walk(do, v, k, g, n, H, scale, t(s0), absolute=absolute)
    over = None if ds is None else ds.double() / scale
    dk, _ = walk(v, do, q, g, n, H, scale, t(over), reverse=True, absolute=absolute)
    dv, r = walk(k, q, do, g, n, H, scale, over, reverse=True, absolute=absolute)
    group = lambda x: x.reshape(*x.shape[:2], G, H // G, -1).sum(3)  # noqa: E731
    return dq, group(dk), group(dv), r * scale
