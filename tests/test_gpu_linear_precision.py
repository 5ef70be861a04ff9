"""Linear attention over long sequences with slow decays: how its error grows with the chunks that a term passes.

In the norm, against the sums over pairs of tokens in 64 bits, with A the same sums of the terms' sizes, in roundings of fp32
(2^-24).  A decay is an exp2 (2) and, across chunks, factors whose product is off by one.  A chunk's products: 8 steps of 32
that the matrix cores add up, cut downwards (half a step of the last bit each in the mean, 16 for the two products in a row).
Each chunk's addition to the state, and its decay, round to nearest, one way as often as the other: the square root of twice the
chunks over that of 3 (37 for 2048 chunks of 32).  60 in all; a factor that is off by half a rounding would give 1024 for a term that
passes 2048 chunks.  bf16 inputs: the same for what is fp32 (states, their gradients, dg); o and dq, dk, dv round to bf16.
"""

import pytest
import torch

from gsa_gdn_benchmarkstudy_amd import linear_attention

pytestmark = pytest.mark.gpu

D, SCALE = 128, 128 ** -0.5


def _inputs(dev, T, Hk, H, dtype, seed):
    """Values and their gradients with a mean, q and k behind a SiLU: sums that grow, whose errors would add up."""
    gen = torch.Generator(device=dev).manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, generator=gen, device=dev)

    x = {n: torch.nn.functional.silu(rn(1, T, Hk, D)).to(dtype) for n in ("q", "k")}
    x |= {"v": (rn(1, T, H, D) + 1).to(dtype), "state": rn(1, H, D, D)}
    return x, (rn(1, T, H, D) + 1).to(dtype), rn(1, H, D, D)


def _close(got, ref, size, name):
    """got in bf16 rounds the result besides: 1.1 of what rounding the exact one gives."""
    one = (ref.to(got.dtype).double() - ref).norm()
    err = (got.double() - ref).norm()
    assert err <= 1.1 * one + 60 * 2.0 ** -24 * size.norm(), f"{name}: {err / (2.0 ** -24 * size.norm()):.1f} roundings"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_states_of_many_chunks_in_a_row(dev, dtype):
    """So many heads that no head is cut into segments, with memories of 200 to 100000 tokens: the final state and the gradient of
    the initial one."""
    T, H = 65536 + 37, 176
    print(f"states {dtype}", flush=True)
    x, do, ds = _inputs(dev, T, 1, H, dtype, seed=3)
    decay = -1e-5 * 2 ** (torch.arange(H, device=dev) / 20)
    st = x["state"].clone().requires_grad_()
    o, final = linear_attention(x["q"], x["k"], x["v"], decay, initial_state=st, output_final_state=True)
    dst, = torch.autograd.grad([o, final], [st], [do, ds])
    at = torch.arange(T, device=dev, dtype=torch.float64)
    for h in range(0, H, 7):
        e = decay[h].double()
        q, k, v, w = (t[0, :, h % t.shape[2]].double() for t in (x["q"], x["k"], x["v"], do))
        out = []
        for f in (lambda t: t, torch.abs):
            out.append((((e * T).exp() * f(x["state"][0, h].double()) + (f(k) * (e * (T - 1 - at)).exp()[:, None]).T @ f(v)),
                        (e * T).exp() * f(ds[0, h].double()) + SCALE * (f(q) * (e * (at + 1)).exp()[:, None]).T @ f(w)))
        _close(final[0, h].detach(), out[0][0], out[1][0], f"final, g {decay[h]}")
        _close(dst[0, h], out[0][1], out[1][1], f"dstate, g {decay[h]}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("g", [-1e-5, -1e-4, -1e-3, -1e-2, -0.2])
def test_everything_under_slow_decays(dev, g, dtype):
    T = 8192 + 5
    print(f"everything {dtype} g={g}", flush=True)
    x, do, ds = _inputs(dev, T, 1, 1, dtype, seed=4)
    leaf = [t.clone().requires_grad_() for t in (x["q"], x["k"], x["v"], torch.tensor([g], device=dev), x["state"])]
    o, final = linear_attention(*leaf[:4], initial_state=leaf[4], output_final_state=True)
    got = dict(zip(("o", "final", "dq", "dk", "dv", "dg", "dstate"),
                   [o.detach(), final.detach(), *torch.autograd.grad([o, final], leaf, [do, ds])]))
    e, at = torch.tensor(g, device=dev).double(), torch.arange(T, device=dev, dtype=torch.float64)
    gap = at[:, None] - at
    decay = torch.where(gap >= 0, (e * gap.clamp_min(0)).exp(), 0.0)
    up, down, whole = (e * (at + 1)).exp()[:, None], (e * (T - 1 - at)).exp()[:, None], (e * T).exp()
    out = []
    for f in (lambda t: t, torch.abs):
        q, k, v, w = (f(t[0, :, 0].double()) for t in (x["q"], x["k"], x["v"], do))
        S, dS = f(x["state"][0, 0].double()), f(ds[0, 0].double())
        P, R = SCALE * (q @ k.T) * decay, SCALE * (w @ v.T) * decay
        r = {"o": SCALE * up * (q @ S) + P @ v, "final": whole * S + (k * down).T @ v, "dq": SCALE * up * (w @ S.T) + R @ k,
             "dk": down * (v @ dS.T) + R.T @ q, "dv": down * (k @ dS) + P.T @ w, "dstate": whole * dS + SCALE * (q * up).T @ w}
        r["dg"] = (P * (w @ v.T) * gap).sum() + T * whole * (S * dS).sum() + ((T - 1 - at) * ((down * k) @ dS * v).sum(1)).sum() \
            + SCALE * ((at + 1) * ((up * q) @ S * w).sum(1)).sum()
        out.append(r)
    for n, ref in out[0].items():
        _close(got[n].reshape(ref.shape), ref, out[1][n], n)
