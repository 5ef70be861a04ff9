"""Linear attention with decays in 64 bits, from its recurrence, token by token."""

import torch


def rule(q, k, v, g, scale, state=None):
    """q, k [T,Hk,128], v [T,Hv,128], g [Hv], state [Hv,128,128], all float64 -> (o, state)."""
    T, Hv, d = v.shape
    share = Hv // q.shape[1]
    q, k = q.repeat_interleave(share, 1), k.repeat_interleave(share, 1)
    S = torch.zeros(Hv, d, d, dtype=v.dtype) if state is None else state
    a = g.exp()[:, None, None]
    out = []
    for t in range(T):
        S = S * a + k[t][:, :, None] * v[t][:, None, :]
        out.append(scale * (S.transpose(1, 2) @ q[t][:, :, None])[..., 0])
    return (torch.stack(out) if out else v), S
