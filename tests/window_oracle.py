"""Attention in a sliding window with first tokens, in 64 bits, from its definition, and the sizes of its terms."""

import torch


def visible(T, window, sinks):
    i, j = torch.arange(T)[:, None], torch.arange(T)
    return (j <= i) & ((j > i - window) | (j < sinks))


def attention(q, k, v, window, sinks, scale, do=None):
    """One sequence: q [T,H,128], k, v [T,Hkv,128] -> {o, dq, dk, dv} in float64, and of each result the sum of its terms'
    sizes: o: P |v|;  dv: P^T |do|;  dq, dk: of P (|do| |v| + |do| |o|) times |k| or |q|; `score`: the largest sum of a
    score's terms."""
    q, k, v = (t.double().transpose(0, 1) for t in (q, k, v))
    share, Hkv = q.shape[0] // k.shape[0], k.shape[0]
    kk, vv = (t.repeat_interleave(share, 0) for t in (k, v))
    s = (q @ kk.transpose(1, 2) * scale).masked_fill(~visible(q.shape[1], window, sinks), -float("inf"))
    p = torch.softmax(s, -1)
    ref, size = {"o": p @ vv}, {"o": p @ vv.abs()}
    if not v.isfinite().all():                   # 0 * NaN: each query over what it sees alone
        see = visible(q.shape[1], window, sinks)
        ref["o"] = torch.stack([(p[:, i:i + 1, row] @ vv[:, row])[:, 0] for i, row in enumerate(see)], 1)
    score = (q.abs() @ kk.abs().transpose(1, 2)).max() * abs(scale)
    if do is not None:
        do = do.double().transpose(0, 1)
        dp = do @ vv.transpose(1, 2)
        ds = p * (dp - (do * ref["o"]).sum(-1, keepdim=True)) * scale
        big = p * (do.abs() @ vv.abs().transpose(1, 2) + (do * ref["o"]).abs().sum(-1, keepdim=True)) * abs(scale)
        group = lambda t: t.unflatten(0, (Hkv, share)).sum(1)  # noqa: E731
        ref |= {"dq": ds @ kk, "dk": group(ds.transpose(1, 2) @ q), "dv": group(p.transpose(1, 2) @ do)}
        size |= {"dq": big @ kk.abs(), "dk": group(big.transpose(1, 2) @ q.abs()), "dv": group(p.transpose(1, 2) @ do.abs())}
    return {n: t.transpose(0, 1) for n, t in ref.items()}, {n: t.transpose(0, 1) for n, t in size.items()}, float(score)
