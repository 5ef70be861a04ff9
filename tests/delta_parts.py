"""The chunked gated delta rule in fp32 on the CPU with the operands of its products cut to bf16 parts,
and the measure of error that tells three parts (24 bits) from two (16).

``check`` holds the root mean square error of an fp32 result to 16 roundings of 2**-24 of the
result's root mean square.  A result is a sum in which roundings of at most 2**-24 of a partial sum add up
like a walk, sqrt(M) of them for M.  On the way to an output or a state lie the products K S0 and Q S0
(128 elements: 4 steps of up to 6 matrix instructions), Tm R, P U and K^T U (up to 64 tokens: 2 steps
of 6): 84 accumulations, and what a state carried in from the chunk before has decayed by then; a
gradient goes that way twice and through the products with E and F (24 more): M below 256 = 16**2.
An operand of two parts errs by 2**-17 to 2**-18, 64 to 128 of these units, in every term.
"""

import math

import torch

D = 128
NAMES = ("q", "k", "v", "g", "beta")
PRODUCTS = ("KK", "QK", "KS", "TR", "QS", "PU", "KU")
UNITS = 16


def units(got, ref):
    """Root mean square of the error, in 2**-24 of the reference's."""
    return float((got.double().cpu() - ref).square().mean().sqrt() / ref.square().mean().sqrt()) * 2 ** 24


def check(got, ref, name):
    assert tuple(got.shape) == tuple(ref.shape) and got.dtype == torch.float32, name
    u = units(got, ref)
    assert u <= UNITS, f"{name}: {u:.1f} roundings of 2^-24, {UNITS} allowed"


def inputs(B, T, Hk, Hv, dtype, seed, slow):
    """q, k of unit length; gates that forget within some ten tokens, or (slow) within hundreds."""
    gen = torch.Generator().manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, generator=gen)

    q, k = (torch.nn.functional.normalize(rn(B, T, Hk, D), dim=-1).to(dtype) for _ in range(2))
    x = dict(q=q, k=k, v=rn(B, T, Hv, D).to(dtype), g=-torch.exp(rn(B, T, Hv) - (6 if slow else 2)), beta=torch.sigmoid(rn(B, T, Hv)))
    return x, rn(B, Hv, D, D), (rn(B, T, Hv, D).to(dtype), rn(B, Hv, D, D))


def _cut(x, parts):
    if parts >= 3:
        return x
    rest, total = x, torch.zeros_like(x)
    for _ in range(parts):
        p = rest.to(torch.bfloat16).float()
        total, rest = total + p, rest - p
    return total


class _Product(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, b, parts):
        ctx.parts = parts
        ctx.save_for_backward(a, b)
        return _cut(a, parts) @ _cut(b, parts)

    @staticmethod
    def backward(ctx, g):
        a, b = ctx.saved_tensors
        g, a, b = (_cut(t, ctx.parts) for t in (g, a, b))
        return g @ b.transpose(-1, -2), a.transpose(-1, -2) @ g, None


def chunked(x, state, grads, C, two=()):
    """(o, state, gradients); two: the products whose operands are cut to two parts."""
    leaf = {n: t.float().requires_grad_(True) for n, t in x.items()}
    st = state.clone().requires_grad_(True)
    share = x["v"].shape[2] // x["q"].shape[2]
    q, k, v, g, beta = ((leaf[n].repeat_interleave(share, 2) if n in "qk" else leaf[n]).transpose(1, 2) for n in NAMES)
    T, scale = q.shape[2], D ** -0.5
    pad = -T % C
    q, k, v = (torch.nn.functional.pad(t, (0, 0, 0, pad)).unflatten(2, (-1, C)) for t in (q, k, v))
    g, beta = (torch.nn.functional.pad(t, (0, pad)).unflatten(2, (-1, C)) for t in (g, beta))

    def mm(name, a, b):
        return _Product.apply(a, b, 2 if name in two else 3)

    G = g.double().cumsum(-1)
    low = torch.ones(C, C, dtype=torch.bool).tril()
    decay = torch.where(low, G[..., :, None] - G[..., None, :], -math.inf).exp().float()
    e, rest, whole = G.exp().float(), (G[..., -1:] - G).exp().float(), G[..., -1].exp().float()
    kt = k.transpose(-1, -2)
    A = (mm("KK", k, kt) * decay * beta[..., None]).tril(-1)
    eye = torch.eye(C)
    Tm = torch.linalg.solve_triangular(A + eye, eye.expand_as(A), upper=False, unitriangular=True)
    P = scale * mm("QK", q, kt) * decay
    S, outs = st, []
    for c in range(q.shape[2]):
        R = beta[:, :, c, :, None] * (v[:, :, c] - e[:, :, c, :, None] * mm("KS", k[:, :, c], S))
        U = mm("TR", Tm[:, :, c], R)
        outs.append(scale * e[:, :, c, :, None] * mm("QS", q[:, :, c], S) + mm("PU", P[:, :, c], U))
        S = whole[:, :, c, None, None] * S + mm("KU", kt[:, :, c], rest[:, :, c, :, None] * U)
    o = torch.cat(outs, 2)[:, :, :T].transpose(1, 2)
    d = torch.autograd.grad([o, S], [leaf[n] for n in NAMES] + [st], [grads[0].float(), grads[1]])
    return o.detach(), S.detach(), dict(zip(NAMES + ("state",), d))


def fp32_results(got, ref, inputs_dtype):
    """(name, result, reference) of what the operator gives in fp32."""
    both = {"o": (got[0], ref[0]), "state": (got[1], ref[1])} | {"d" + n: (got[2][n], ref[2][n]) for n in got[2]}
    keep = both if inputs_dtype == torch.float32 else ("state", "dg", "dbeta", "dstate")
    return [(n, *both[n]) for n in keep]
