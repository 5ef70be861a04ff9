"""How near window attention's results are to the definition's in 64 bits.

bf16, in the norm.  A result that carries its own rounding alone is off by what rounding the exact one gives (`one`).  Where a
query sees at most 128 keys P and dS enter the second products in two parts, off by at most 2^-16 of a term (half a step of
bf16, 2^-8, twice), under a tenth of `one` in the norm: 1.1.  Elsewhere P's and dS's own rounding is as large as the result's: the
square root of 2, and 1.47 with what a norm over these many elements scatters.  2^-20 of the terms' sizes is left for results
that cancel (one visible key: dq and dk are 0).

bf16, each element, where at most 128 keys are visible: half a step of the result, 2^-16 of the terms' sizes for o and dv,
2^-15 for dq and dk (dS, and D = do . o from o in two parts), and fp32's part as tests/test_gpu_window.py counts it.
"""

import pytest
import torch

from gsa_gdn_benchmarkstudy_amd import window_attention
from tests import test_gpu_window as tw

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _spans(B, T, lens):
    if lens is None:
        return [(b, 0, T) for b in range(B)]
    ends = torch.tensor([0] + lens).cumsum(0).tolist()
    return [(0, a, b) for a, b in zip(ends, ends[1:])]


def _both(dev, B, T, H, Hkv, lens, W, S, dtype=BF16):
    print(f"{dtype} B={B} T={T} H={H} Hkv={Hkv} W={W} S={S} sequences={lens and len(lens)}", flush=True)
    x, do = tw._inputs(B, T, H, Hkv, dtype, seed=T + W), tw._grad(B, T, H, dtype, 7)
    spans = _spans(B, T, lens)
    cu = None if lens is None else torch.tensor([0] + lens).cumsum(0).to(dev)
    got = {n: t.cpu() for n, t in tw._run(x, dev, W, S, cu=cu, do=do).items()}
    return got, *tw._oracle(x, spans, W, S, 128 ** -0.5, do), spans


def _in_the_norm(got, ref, size, times, name):
    one = (ref.to(got.dtype).double() - ref).norm()
    err = (got.double() - ref).norm()
    assert err <= times * one + 2.0 ** -20 * size.norm(), f"{name}: {err / one:.3f} roundings"


def _elements(got, ref, size, score, T, name):
    few = 2.0 ** -16 if name in ("o", "dv") else 2.0 ** -15
    tol = torch.finfo(BF16).eps / 2 * ref.abs() + (few + (80 * score + 128 + T / 8) * 2.0 ** -24) * size + 2.0 ** -126
    err = (got.double() - ref).abs()
    assert bool((err <= tol).all()), f"{name}: {(err / tol).max():.2f} of the tolerance"


@pytest.mark.parametrize("H,Hkv,lens,W,S", [(4, 2, [20] * 300, 512, 0), (8, 8, [20] * 300, 512, 4), (4, 1, [1, 2, 5, 128, 100, 17, 64, 127] * 4, 1000, 4),
                                            (2, 2, [6, 7, 5] * 10, 1 << 20, 0)])
def test_short_sequences_under_a_long_window(dev, H, Hkv, lens, W, S):
    """Packed sequences of at most 128 tokens see few keys, whatever the window."""
    got, ref, size, score, _ = _both(dev, 1, sum(lens), H, Hkv, lens, W, S)
    for n in got:
        _in_the_norm(got[n], ref[n], size[n], 1.1, n)
        _elements(got[n], ref[n], size[n], score, max(lens), n)


@pytest.mark.parametrize("B,T,H,Hkv,lens,W,S", [(2, 700, 4, 2, None, 1000, 0), (8, 1100, 8, 8, None, 200, 35), (1, 1480, 4, 4, [300, 129, 1, 1050], 500, 3),
                                                (2, 700, 4, 1, None, 20, 300)])
def test_first_queries_under_a_long_window(dev, B, T, H, Hkv, lens, W, S):
    """The first 128 queries of longer sequences see few keys; the others' results are off by P's and dS's rounding too."""
    got, ref, size, score, spans = _both(dev, B, T, H, Hkv, lens, W, S)
    first = torch.zeros(B, T, dtype=torch.bool)
    for b, s, e in spans:
        first[b, s:min(e, s + 128)] = True
    for n in got:
        _in_the_norm(got[n], ref[n], size[n], 1.47, n)
        if n in ("o", "dq"):
            _in_the_norm(got[n][first], ref[n][first], size[n][first], 1.1, n)
            _elements(got[n][first], ref[n][first], size[n][first], score, T, n)


@pytest.mark.parametrize("B,T,H,Hkv,lens,W,S", [(8, 600, 16, 8, None, 50, 5), (5, 1000, 16, 16, None, 60, 65), (1, 5849, 12, 12, [700, 0, 1500, 65, 2300, 1, 1283], 100, 4),
                                                (1, 900, 2, 1, None, 28, 100)])
def test_short_windows(dev, B, T, H, Hkv, lens, W, S):
    """Blocks of 128 queries and keys and of 64, first tokens with far queries: all see few keys."""
    got, ref, size, score, _ = _both(dev, B, T, H, Hkv, lens, W, S)
    for n in got:
        _in_the_norm(got[n], ref[n], size[n], 1.1, n)
        _elements(got[n], ref[n], size[n], score, T, n)


def _in_full(q, k, v, do, W):
    """The definition's results in the inputs' type by whole matrices: [1, T, H, 128], keys of one head."""
    T = q.shape[1]
    q, do, k, v = (t[0].transpose(0, 1) for t in (q, do, k, v))
    at = torch.arange(T, device=q.device)
    seen = (at[:, None] >= at) & (at[:, None] - at < W)
    p = torch.softmax((q @ k.transpose(1, 2) * 128 ** -0.5).masked_fill(~seen, -float("inf")), -1)
    o = p @ v
    ds = p * (do @ v.transpose(1, 2) - (do * o).sum(-1, keepdim=True)) * 128 ** -0.5
    dk, dv = ((a.transpose(1, 2) @ b).sum(0, keepdim=True) for a, b in ((ds, q), (p, do)))
    return {n: t.transpose(0, 1)[None] for n, t in (("o", o), ("dq", ds @ k), ("dk", dk), ("dv", dv))}


@pytest.mark.parametrize("T,W", [(8192, 8192), (4096, 4096), (4096, 300)])
def test_fp32_errors_of_long_sums(dev, T, W):
    """Four query heads on a key head and values and gradients with a mean: sums that grow over thousands of keys and queries.  Their errors
    are those of plain fp32 sums in torch or less: either side rounds a score and a do . v over 128 products, and the sums over
    keys once a tile here; 1.25 for what such errors scatter by."""
    gen = torch.Generator(device=dev).manual_seed(T)
    q, k, v, do = (torch.randn(1, T, h, 128, generator=gen, device=dev) + mean for h, mean in ((4, 0), (1, 0), (1, 1), (4, 1)))
    ref, plain = _in_full(*(t.double() for t in (q, k, v, do)), W), _in_full(q, k, v, do, W)
    leaf = [t.requires_grad_() for t in (q, k, v)]
    o = window_attention(*leaf, W)
    got = {"o": o.detach(), **dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaf, do)))}
    for n in got:
        own, other = ((t[n].double() - ref[n]).norm() / ref[n].norm() for t in (got, plain))
        print(f"{n}: {own:.2e}, plain {other:.2e}", flush=True)
        assert own <= 1.25 * other, n
