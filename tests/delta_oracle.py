"""The gated delta rule and the RMS norm in 64 bits, from their formulas, token by token."""

import torch


def rule(q, k, v, g, beta, scale, state=None):
    """q, k [T,Hk,128], v [T,Hv,128], g, beta [T,Hv], state [Hv,128,128], all float64 -> (o, state)."""
    T, Hv, d = v.shape
    share = Hv // q.shape[1]
    q, k = q.repeat_interleave(share, 1), k.repeat_interleave(share, 1)
    S = torch.zeros(Hv, d, d, dtype=v.dtype) if state is None else state
    out = []
    for t in range(T):
        S = S * g[t].exp()[:, None, None]
        u = beta[t][:, None] * (v[t] - (S.transpose(1, 2) @ k[t][:, :, None])[..., 0])
        S = S + k[t][:, :, None] * u[:, None, :]
        out.append(scale * (S.transpose(1, 2) @ q[t][:, :, None])[..., 0])
    return (torch.stack(out) if out else v), S


def norm(x, w, res, eps, dtype):
    """(y, h) in float64; h rounded to dtype, as the stream is kept (its gradient passes the rounding)."""
    h = x if res is None else x + res
    h = h + (h.detach().to(dtype).double() - h.detach())
    return h * (h.square().mean(-1, keepdim=True) + eps) ** -0.5 * w, h
