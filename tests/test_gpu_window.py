"""Attention in a sliding window, its cache and its single-token step on the GPU against the definition in 64 bits.

Tolerances.  The oracle gives with each result the sum A of its terms' sizes.  A result of type t carries one rounding, at
most eps(t) / 2 of its value.  In bf16 P enters the second product rounded (2^-8 of a term) and the gradients' dS too: 2^-8 A for o
and dv, and 2^-7 A for dq and dk, which is enough for D = do . o from o rounded to bf16 as well (the kernels use o in two parts, and
two parts of P and dS where few keys are visible: tests/test_gpu_window_precision.py holds them to that).  Scores are sums of 128 products in
fp32: at most 32 + 6 roundings of 2^-24 of the sum of their terms' sizes (8 steps of 16 summed by the matrix cores, up to 6
products each), which moves P by as much, numerator and denominator; so do the exponent's rounding, exp2 and the
running sums: (2 * 40 * score + 128 + T / 8) roundings of A in all.
"""

import pytest
import torch

from gsa_gdn_benchmarkstudy_amd import add_rms_norm, window_attention, window_attention_step, window_cache_write
from tests import window_oracle as orc

pytestmark = pytest.mark.gpu

D = 128
TYPES = [torch.bfloat16, torch.float32]


def _inputs(B, T, H, Hkv, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    return {n: torch.randn(B, T, h, D, generator=gen).to(dtype) for n, h in (("q", H), ("k", Hkv), ("v", Hkv))}


def _grad(B, T, H, dtype, seed):
    return torch.randn(B, T, H, D, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _oracle(x, spans, window, sinks, scale, do):
    ref, size, score = {}, {}, 0.0
    for b, s, e in spans:
        if e == s:
            continue
        r, z, y = orc.attention(*(x[n][b, s:e] for n in "qkv"), window, sinks, scale, None if do is None else do[b, s:e])
        score = max(score, y)
        for n in r:
            if n not in ref:
                like = x["q" if n == "o" else n[1]]
                ref[n], size[n] = (torch.zeros(like.shape, dtype=torch.float64) for _ in range(2))
            ref[n][b, s:e], size[n][b, s:e] = r[n], z[n]
    return ref, size, score


def _check(got, ref, size, score, T, name):
    assert tuple(got.shape) == tuple(ref.shape), name
    bf16 = got.dtype == torch.bfloat16
    few = (2.0 ** -8 if name in ("o", "dv") else 2.0 ** -7) if bf16 else 0.0
    tol = torch.finfo(got.dtype).eps / 2 * ref.abs() + (few + (80 * score + 128 + T / 8) * 2.0 ** -24) * size + 2.0 ** -126
    err = (got.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), f"{name}: {(err / tol).max():.2f} of the tolerance (|err| {err.max():.2e})"


def _run(x, dev, window, sinks, cu=None, do=None, scale=None):
    leaf = {n: t.to(dev).requires_grad_(do is not None) for n, t in x.items()}
    o = window_attention(leaf["q"], leaf["k"], leaf["v"], window, sinks=sinks, scale=scale, cu_seqlens=cu)
    out = {"o": o.detach()}
    if do is not None:
        out |= dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, [leaf[n] for n in "qkv"], do.to(dev))))
    return out


def _compare(got, x, spans, window, sinks, do=None, scale=D ** -0.5):
    ref, size, score = _oracle(x, spans, window, sinks, scale, do)
    T = max(e - s for _, s, e in spans)
    for n in got:
        if n in ref:
            _check(got[n], ref[n], size[n], score, T, n)


CASES = [(1, 1, 1, 1, 1, 0), (2, 2, 2, 1, 1, 1), (1, 31, 1, 1, 5, 0), (1, 33, 3, 1, 100, 0), (2, 64, 2, 2, 32, 3), (1, 65, 4, 2, 64, 64),
         (1, 127, 1, 1, 63, 200), (1, 128, 2, 1, 65, 0), (3, 129, 2, 2, 128, 4), (1, 200, 4, 1, 1, 0), (2, 200, 2, 1, 2, 33),
         (1, 300, 2, 2, 150, 70), (1, 513, 1, 1, 64, 130), (1, 700, 2, 1, 1000000, 0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,T,H,Hkv,W,S", CASES)
def test_forward(dev, B, T, H, Hkv, W, S, dtype):
    print(f"forward {dtype} B={B} T={T} H={H} Hkv={Hkv} W={W} S={S}", flush=True)
    x = _inputs(B, T, H, Hkv, dtype, seed=T)
    _compare(_run(x, dev, W, S), x, [(b, 0, T) for b in range(B)], W, S)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,T,H,Hkv,W,S", CASES)
def test_backward(dev, B, T, H, Hkv, W, S, dtype):
    print(f"backward {dtype} B={B} T={T} H={H} Hkv={Hkv} W={W} S={S}", flush=True)
    x, do = _inputs(B, T, H, Hkv, dtype, seed=T + 1), _grad(B, T, H, dtype, 7)
    _compare(_run(x, dev, W, S, do=do), x, [(b, 0, T) for b in range(B)], W, S, do)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,T,H,Hkv,W,S", [(1, 2300, 2, 1, 40, 70), (2, 1400, 1, 1, 300, 1), (1, 2049, 1, 1, 897, 150), (1, 1153, 1, 1, 1, 1)])
def test_far_queries_of_first_tokens(dev, B, T, H, Hkv, W, S, dtype):
    """First tokens whose queries come in several parts."""
    print(f"far {dtype} B={B} T={T} H={H} Hkv={Hkv} W={W} S={S}", flush=True)
    x, do = _inputs(B, T, H, Hkv, dtype, seed=T + 1), _grad(B, T, H, dtype, 7)
    _compare(_run(x, dev, W, S, do=do), x, [(b, 0, T) for b in range(B)], W, S, do)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,T,H,Hkv,W,S", [(1, 700, 2, 1, 650, 50), (1, 700, 2, 1, 650, 49), (2, 300, 2, 2, 10, 299), (4, 1100, 24, 2, 50, 1000)])
def test_many_first_tokens(dev, B, T, H, Hkv, W, S, dtype):
    """First tokens that are all that the window leaves out, all but one, and so many that their queries' parts grow."""
    print(f"first tokens {dtype} B={B} T={T} H={H} Hkv={Hkv} W={W} S={S}", flush=True)
    x, do = _inputs(B, T, H, Hkv, dtype, seed=T + S), _grad(B, T, H, dtype, 7)
    _compare(_run(x, dev, W, S, do=do), x, [(b, 0, T) for b in range(B)], W, S, do)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,T,H,Hkv,W,S", [(8, 600, 16, 8, 50, 5), (8, 1100, 8, 8, 200, 35), (9, 897, 8, 8, 897, 0), (5, 1000, 32, 16, 128, 200)])
def test_many_blocks(dev, B, T, H, Hkv, W, S, dtype):
    """Enough blocks of keys and queries for the larger ones, none of them in parts; first tokens with and without far queries."""
    print(f"many {dtype} B={B} T={T} H={H} Hkv={Hkv} W={W} S={S}", flush=True)
    x, do = _inputs(B, T, H, Hkv, dtype, seed=T + S), _grad(B, T, H, dtype, 7)
    _compare(_run(x, dev, W, S, do=do), x, [(b, 0, T) for b in range(B)], W, S, do)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_blocks_packed(dev, dtype):
    lens = [700, 0, 1500, 65, 2300, 1, 1283]
    T, H = sum(lens), 12
    x, do = _inputs(1, T, H, H, dtype, seed=T), _grad(1, T, H, dtype, 7)
    cu = torch.tensor([0] + lens).cumsum(0)
    _compare(_run(x, dev, 150, 4, cu=cu.to(dev), do=do), x, [(0, int(cu[i]), int(cu[i + 1])) for i in range(len(lens))], 150, 4, do)


@pytest.mark.parametrize("W,S,few", [(1, 0, True), (2, 0, True), (4, 0, True), (16, 3, True), (100, 28, True), (129, 0, False), (1000, 0, False)])
def test_bf16_errors_in_the_norm(dev, W, S, few):
    """Where few keys are visible P and dS take two parts: results are off by their own rounding, the rest is 2^-17 of terms, under
    a tenth of it in the norm.  Elsewhere by P's or dS's as well, which does not depend on theirs: the square root of 2 of one
    rounding's error (1.41; sums over more than 128 terms and 1400 rows: within 1.47)."""
    x, do = _inputs(2, 700, 4, 2, torch.bfloat16, seed=W), _grad(2, 700, 4, torch.bfloat16, 7)
    got = _run(x, dev, W, S, do=do)
    ref, size, _ = _oracle(x, [(0, 0, 700), (1, 0, 700)], W, S, D ** -0.5, do)
    for n in got:
        one = (ref[n].to(torch.bfloat16).double() - ref[n]).norm()
        least = 2.0 ** -20 * size[n].norm()      # (one visible key: dq and dk are 0)
        assert (got[n].double().cpu() - ref[n]).norm() <= (1.1 if few else 1.47) * one + least, n


PACKS = [[1], [5, 0, 64, 1, 65, 63], [0, 0, 3], [130, 32, 33], [128, 64, 256], [0], [1300, 1, 0, 333]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", PACKS)
@pytest.mark.parametrize("lead,trail,idx,W,S", [(0, 0, torch.int32, 40, 3), (3, 37, torch.int64, 100, 0), (1, 0, torch.int64, 7, 140)])
def test_packed(dev, lens, lead, trail, idx, W, S, dtype):
    """Packed sequences, empty ones among them; rows before the first and behind the last become 0, whatever they hold."""
    print(f"packed {dtype} {lens} lead={lead} trail={trail} W={W} S={S}", flush=True)
    T, N, H, Hkv = lead + sum(lens) + trail, len(lens), 2, 1
    if T == 0:
        return
    cu = torch.tensor([lead] + lens).cumsum(0).to(idx)
    x, do = _inputs(1, T, H, Hkv, dtype, seed=N), _grad(1, T, H, dtype, 8)
    outside = torch.ones(T, dtype=torch.bool)
    outside[lead:T - trail] = False
    for t in (*x.values(), do):
        t[0, outside] = float("nan")
    got = _run(x, dev, W, S, cu=cu.to(dev), do=do)
    _compare(got, x, [(0, int(cu[i]), int(cu[i + 1])) for i in range(N)], W, S, do)
    for t in got.values():
        assert not t[0, outside.to(dev)].any()


def test_offsets_outside_the_tokens_touch_nothing(dev):
    """Offsets past T or descending: held within the tokens, other sequences are right."""
    x = _inputs(1, 100, 1, 1, torch.bfloat16, seed=3)
    _compare(_run(x, dev, 9, 2, cu=torch.tensor([0, 40, 1 << 30], dtype=torch.int64, device=dev)), x, [(0, 0, 40), (0, 40, 100)], 9, 2)
    got = _run(x, dev, 9, 2, cu=torch.tensor([-5, 40, 20], dtype=torch.int32, device=dev))["o"]
    ref, size, score = _oracle(x, [(0, 0, 40)], 9, 2, D ** -0.5, None)
    _check(got[:, :40], ref["o"][:, :40], size["o"][:, :40], score, 40, "o")
    assert not got[:, 40:].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [0.0, -0.09, 0.3, 1e-30])
def test_scale(dev, scale, dtype):
    x, do = _inputs(1, 150, 2, 1, dtype, seed=12), _grad(1, 150, 2, dtype, 9)
    _compare(_run(x, dev, 70, 5, do=do, scale=scale), x, [(0, 0, 150)], 70, 5, do, scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_large_scores(dev, dtype):
    """Scores that rise and fall by hundreds along the keys: the running maximum moves in most tiles."""
    x = _inputs(1, 400, 1, 1, dtype, seed=13)
    x["k"] = (x["k"].float() * torch.linspace(0.1, 30, 400)[:, None, None] * torch.where(torch.arange(400) % 130 < 90, 1, -1)[:, None, None]).to(dtype)
    _compare(_run(x, dev, 333, 4), x, [(0, 0, 400)], 333, 4)


def test_gradient_against_differences(dev):
    """The kernels' gradient along random directions against differences of the definition in 64 bits."""
    T, W, S = 140, 50, 3
    x, do = _inputs(1, T, 2, 1, torch.float32, seed=21), _grad(1, T, 2, torch.float32, 10)
    got = _run(x, dev, W, S, do=do)
    _, size, score = _oracle(x, [(0, 0, T)], W, S, D ** -0.5, do)
    gen = torch.Generator().manual_seed(9)
    for n in "qkv":
        r, h = torch.randn(x[n].shape, generator=gen).double(), 1e-5
        up, dn = ((_oracle({m: t.double() for m, t in x.items()} | {n: x[n].double() + e * r}, [(0, 0, T)], W, S, D ** -0.5, None)[0]["o"]
                   * do.double()).sum() for e in (h, -h))
        want = (up - dn) / (2 * h)
        # differences: h^2 of a third derivative and 2^-52 / h of the loss (1e-6); the gradient's elements as in _check
        tol = ((80 * score + 146) * 2.0 ** -24 * size["d" + n] * r.abs()).sum() + 1e-6 * (abs(want) + abs(up))
        assert abs(want - (got["d" + n].double().cpu() * r).sum()) <= tol, n


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("name", ["q", "k", "v"])
def test_what_a_query_does_not_see_does_not_reach_it(dev, name, bad, dtype):
    """One element of one token that is not finite: the queries that do not see it are right, those that do have what the
    definition gives."""
    T, W, S, at = 300, 70, 3, 150
    x = _inputs(2, T, 2, 2, dtype, seed=5)
    clean = _run(x, dev, W, S)["o"]
    x[name][1, at, 1, 33] = bad
    got = _run(x, dev, W, S)["o"]
    ref, _, _ = _oracle(x, [(b, 0, T) for b in range(2)], W, S, D ** -0.5, None)
    fine = ref["o"].isfinite()
    assert torch.equal(got.isfinite().cpu(), fine) and torch.equal(got.isnan().cpu(), ref["o"].isnan())
    assert torch.equal(got[0], clean[0]) and torch.equal(got[:, :, 0], clean[:, :, 0])
    other = _oracle({n: t.nan_to_num(0, 0, 0) for n, t in x.items()}, [(b, 0, T) for b in range(2)], W, S, D ** -0.5, None)
    where = orc.visible(T, W, S)[:, at] if name != "q" else torch.arange(T) == at
    for b, h in ((1, 1),):
        rows = ~where
        _check(got[b, rows.to(dev), h], ref["o"][b, rows, h], other[1]["o"][b, rows, h], other[2], T, "o")


@pytest.mark.parametrize("dtype", TYPES)
def test_garbage_behind_a_padded_batch(dev, dtype):
    """Padding of NaN behind each row's tokens: the tokens' outputs are those without it."""
    T, lens, W, S = 260, [260, 131, 7], 100, 2
    x = _inputs(3, T, 2, 1, dtype, seed=15)
    for b, n in enumerate(lens):
        for t in x.values():
            t[b, n:] = float("nan")
    got = _run(x, dev, W, S)["o"]
    for b, n in enumerate(lens):
        ref, size, score = _oracle(x, [(b, 0, n)], W, S, D ** -0.5, None)
        _check(got[b, :n], ref["o"][b, :n], size["o"][b, :n], score, T, "o")


def test_a_packed_neighbour_that_is_not_finite(dev):
    x, do = _inputs(1, 150, 2, 1, torch.bfloat16, seed=6), _grad(1, 150, 2, torch.bfloat16, 11)
    cu = torch.tensor([0, 70, 75, 150], device=dev)
    want = _run(x, dev, 20, 3, cu=cu, do=do)
    for t in (*x.values(), do):
        t[0, 70:75] = float("nan")
    got = _run(x, dev, 20, 3, cu=cu, do=do)
    for n in got:
        assert torch.equal(got[n][:, :70], want[n][:, :70]) and torch.equal(got[n][:, 75:], want[n][:, 75:]), n


def test_strided_views_and_broadcasts(dev):
    """Views of one projection output, heads broadcast with stride 0, transposed layouts: the same bits as copies."""
    gen = torch.Generator().manual_seed(31)
    B, T, H = 2, 190, 2
    big = torch.randn(B, T, 3 * H * D + 64, generator=gen).to(torch.bfloat16).to(dev)
    q, k, v = (big[..., i * H * D:(i + 1) * H * D].view(B, T, H, D) for i in range(3))
    k = k.transpose(1, 2).contiguous().transpose(1, 2)
    a = window_attention(q, k, v, 60, 3)
    b = window_attention(*(t.contiguous() for t in (q, k, v)), 60, 3)
    assert torch.equal(a, b)
    odd = torch.empty(B * T * H * D + 1, device=dev, dtype=torch.bfloat16)[1:].view(B, T, H, D)
    odd.copy_(q)                                 # 2-byte aligned: copied
    assert torch.equal(window_attention(odd, k, v, 60, 3), b)
    one = k[:, :, :1].detach().requires_grad_(True)
    do = torch.randn(q.shape, generator=gen).to(torch.bfloat16).to(dev)
    (d1,) = torch.autograd.grad(window_attention(q, one.expand(B, T, H, D), v, 60, 3), one, do)
    full = k[:, :, :1].expand(B, T, H, D).contiguous().requires_grad_(True)
    (d2,) = torch.autograd.grad(window_attention(q, full, v, 60, 3), full, do)
    assert torch.equal(d1, d2.sum(2, keepdim=True))
    (d3,) = torch.autograd.grad(window_attention(q, full, v, 60, 3).sum(), full)           # an expanded gradient
    (d4,) = torch.autograd.grad(window_attention(q, full, v, 60, 3), full, torch.ones_like(q))
    assert torch.equal(d3, d4)


def test_same_bits_and_other_stream(dev):
    x, do = _inputs(1, 1700, 4, 2, torch.bfloat16, seed=51), _grad(1, 1700, 4, torch.bfloat16, 12)
    a = _run(x, dev, 200, 4, do=do)
    s = torch.cuda.Stream(device=dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        b = _run(x, dev, 200, 4, do=do)
    torch.cuda.current_stream(dev).wait_stream(s)
    for y in (b, _run(x, dev, 200, 4, do=do)):
        for n in a:
            assert torch.equal(a[n], y[n]), n


def test_parts_of_the_graph(dev):
    x = {n: t.to(dev) for n, t in _inputs(1, 64, 1, 1, torch.bfloat16, seed=71).items()}
    assert not window_attention(*x.values(), 5).requires_grad
    x["v"].requires_grad_(True)
    with torch.no_grad():
        assert not window_attention(*x.values(), 5).requires_grad
    (dv,) = torch.autograd.grad(window_attention(*x.values(), 5).float().sum(), x["v"], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dv.sum(), x["v"])                    # once differentiable
    with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError):
        q = torch.autograd.forward_ad.make_dual(x["q"], torch.ones_like(x["q"]))
        window_attention(q, x["k"], x["v"], 5)
    e = torch.zeros(2, 0, 1, D, device=dev, requires_grad=True)
    o = window_attention(e, e, e, 3, 1)
    assert o.shape == e.shape and torch.autograd.grad(o, e, torch.zeros_like(o))[0].shape == e.shape


# ---------------------------------------------------------------------------
# The cache and the step
# ---------------------------------------------------------------------------

def _row(p, sinks, rows):
    return p if p < sinks else sinks + (p - sinks) % (rows - sinks)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S,rows", [(0, 1), (0, 7), (3, 4), (4, 40), (5, 300)])
@pytest.mark.parametrize("packed", [False, True])
def test_cache_write(dev, S, rows, packed, dtype):
    """Prompts of several lengths, from several positions, in two pieces: the cache holds what comes last; nothing else changes."""
    Hkv, slots, idx = 2, 6, [4, -1, 0, 9, 2]
    gen = torch.Generator().manual_seed(rows)
    caches = [torch.randn(slots, rows, Hkv, D, generator=gen).to(dtype) for _ in range(2)]
    mine, want = [c.to(dev) for c in caches], [c.clone() for c in caches]
    start = [0, 0, 3, 1, 1000]
    for piece in range(2):
        lens = ([70, 3, 1, 5, 131] if piece == 0 else [1, 2, 300, 1, 2]) if packed else [66 + piece] * 5
        n = sum(lens) if packed else lens[0]
        k, v = (torch.randn(1 if packed else 5, n, Hkv, D, generator=gen).to(dtype) for _ in range(2))
        cu = torch.tensor([0] + lens, device=dev).cumsum(0) if packed else None
        pos = None if start == [0] * 5 else torch.tensor(start, device=dev)
        window_cache_write(k.to(dev), v.to(dev), *mine, S, pos, torch.tensor(idx, dtype=torch.int32, device=dev), cu)
        at = 0
        for i, L in enumerate(lens):
            for t in range(L):
                if 0 <= idx[i] < slots:
                    for c, x in zip(want, (k, v)):
                        c[idx[i], _row(start[i] + t, S, rows)] = x[0, at + t] if packed else x[i, t]
            at += L
            start[i] += L
    for a, b in zip(mine, want):
        assert torch.equal(a.cpu(), b)


def _step_oracle(x, caches, pos, at, W, S, scale=D ** -0.5):
    """Caches after the call, o, sizes of its terms, the largest score's: all rows are written first."""
    slots, rows, Hkv, _ = caches[0].shape
    after = [c.clone() for c in caches]
    on = [0 <= s < slots and p >= 0 for s, p in zip(at, pos)]
    for i, (s, p) in enumerate(zip(at, pos)):
        if on[i] and "k" in x:
            for c, n in zip(after, "kv"):
                c[s, _row(p, S, rows)] = x[n][i]
    o, size, score = torch.zeros(x["q"].shape, dtype=torch.float64), torch.zeros(x["q"].shape, dtype=torch.float64), 0.0
    for i, (s, p) in enumerate(zip(at, pos)):
        if on[i]:
            seen = [_row(j, S, rows) for j in range(max(0, p - W + 1) if p < 2 * W + S else p - W + 1, p + 1) if j >= S or j > p - W]
            seen = sorted({*range(min(S, p + 1))} | set(seen))
            k, v = (c[s, seen].double().transpose(0, 1) for c in after)
            q = x["q"][i].double().unflatten(0, (Hkv, -1))
            prob = torch.softmax(q @ k.transpose(1, 2) * scale, -1)
            o[i], size[i] = (prob @ v).flatten(0, 1), (prob @ v.abs()).flatten(0, 1)
            score = max(score, float((q.abs() @ k.abs().transpose(1, 2)).max()) * abs(scale))
    return after, o, size, score


def _step_case(dev, dtype, N, H, Hkv, slots, rows, W, S, pos, at, idx=torch.int32, with_kv=True, scale=None):
    gen = torch.Generator().manual_seed(N + W)
    x = {n: torch.randn(N, h, D, generator=gen).to(dtype) for n, h in (("q", H), ("k", Hkv), ("v", Hkv))}
    if not with_kv:
        x = {"q": x["q"]}
    caches = [torch.randn(slots, rows, Hkv, D, generator=gen).to(dtype) for _ in range(2)]
    mine = [c.to(dev) for c in caches]
    o = window_attention_step(x["q"].to(dev), *(x[n].to(dev) if n in x else None for n in "kv"), *mine, torch.tensor(pos, dtype=idx, device=dev), W,
                              S, None if at is None else torch.tensor(at, dtype=idx, device=dev), scale)
    after, ref, size, score = _step_oracle(x, caches, pos, list(range(N)) if at is None else at, W, S, D ** -0.5 if scale is None else scale)
    for a, b in zip(mine, after):
        assert torch.equal(a.cpu(), b)
    few = 0.0                                    # P stays fp32
    tol = torch.finfo(dtype).eps / 2 * ref.abs() + (few + (80 * score + 128 + W / 8) * 2.0 ** -24) * size + 2.0 ** -126
    err = (o.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), f"{(err / tol).max():.2f} of the tolerance (|err| {err.max():.2e})"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,H,Hkv,slots,rows,W,S,pos,at", [
    (1, 1, 1, 1, 1, 1, 0, [0], None), (1, 2, 1, 1, 9, 5, 4, [123456789], None), (3, 3, 1, 5, 64, 60, 4, [0, 3, 4], None),
    (4, 8, 2, 9, 70, 64, 3, [5, 63, 64, 1000], [8, 0, 3, 5]), (5, 4, 4, 4, 300, 257, 40, [41, 10, 700, 3, -1], [3, -1, 0, 4, 1]),
    (2, 5, 1, 2, 1200, 1100, 2, [5000, 1101], [1, 0]), (2, 16, 1, 3, 200, 190, 0, [189, 190], [2, 1]), (3, 2, 2, 3, 40, 7, 33, [0, 32, 40], None)])
@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
def test_step(dev, N, H, Hkv, slots, rows, W, S, pos, at, idx, dtype):
    """Short sequences, full rings, rows of padding, keys split over blocks, odd numbers of heads."""
    print(f"step {dtype} N={N} H={H} Hkv={Hkv} rows={rows} W={W} S={S} pos={pos} at={at}", flush=True)
    _step_case(dev, dtype, N, H, Hkv, slots, rows, W, S, pos, at, idx)
    _step_case(dev, dtype, N, H, Hkv, slots, rows, W, S, pos, at, idx, with_kv=False, scale=-0.2)


@pytest.mark.parametrize("dtype", TYPES)
def test_step_tokens_of_one_sequence(dev, dtype):
    """Consecutive tokens of one sequence in one call, as many as the ring has room for: each sees those before it."""
    W, S, n = 50, 4, 9
    for first in (0, 2, 47, 333):
        _step_case(dev, dtype, n + 1, 4, 2, 3, S + W + n - 1, W, S, [first + i for i in range(n)] + [20], [1] * n + [2])


def test_step_many_rows(dev):
    N = 300
    _step_case(dev, torch.bfloat16, N, 2, 1, N + 3, 40, 30, 3, [(7 * i) % 101 for i in range(N)], [(i * 7) % (N + 3) if i % 5 else -1 for i in range(N)])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [70, 512, 513])
def test_step_rows_of_the_same_sequences(dev, N, dtype):
    """Tokens of some sequences scattered over the batch, among padding: written by the blocks that read them, or before."""
    W, S, slots = 40, 3, N // 2
    gen = torch.Generator().manual_seed(N)
    at = torch.randint(-1, slots, (N,), generator=gen).tolist()
    seen, pos = {}, []
    for s in at:                                 # consecutive tokens of each sequence, in the batch's order
        seen[s] = seen.get(s, 20 + 7 * s) + 1
        pos.append(seen[s] if s % 11 else -5)
    most = max(seen[s] - (20 + 7 * s) for s in seen if s >= 0)
    _step_case(dev, dtype, N, 4, 2, slots, S + W + most - 1, W, S, pos, at)


def test_step_positions_past_every_sequence(dev):
    """Positions whose sums would pass 64 bits are padding, in the step and in the write."""
    k = torch.randn(3, 2, 1, D, dtype=torch.bfloat16, device=dev)
    for far in (1 << 62, 2 ** 63 - 1, -2 ** 63):
        at = torch.tensor([7, far, far - 1 if far > 0 else far], device=dev)
        kc, vc = (torch.zeros(3, 12, 1, D, dtype=torch.bfloat16, device=dev) for _ in range(2))
        window_cache_write(k, k, kc, vc, 4, at)
        assert kc[0].any() and vc[0].any()
        if far == 1 << 62:                       # 2**62 - 1 is a position
            assert kc[2].any() and not kc[1].any() and not vc[1].any()
        else:
            assert not kc[1:].any() and not vc[1:].any()
        kc, vc = (torch.zeros(3, 12, 1, D, dtype=torch.bfloat16, device=dev) for _ in range(2))
        o = window_attention_step(k[:, 0], k[:, 0], k[:, 0], kc, vc, at, 6, 4)
        assert o[0].any() and not o[1].any() and not kc[1].any() and not vc[1].any()
        if far != 1 << 62:
            assert not o[2].any() and not kc[2].any() and not vc[2].any()


def test_step_far_position(dev):
    """A position past 2^32."""
    _step_case(dev, torch.bfloat16, 2, 2, 1, 2, 90, 60, 4, [(1 << 40) + 12345, 1 << 33], None, torch.int64)


@pytest.mark.parametrize("dtype", TYPES)
def test_step_reads_only_what_it_sees(dev, dtype):
    """Rows of the caches that the tokens do not see hold NaN."""
    W, S, rows, pos = 40, 3, 60, [0, 2, 3, 30, 43, 200]
    gen = torch.Generator().manual_seed(1)
    caches = [torch.full((len(pos), rows, 1, D), float("nan")).to(dtype) for _ in range(2)]
    for n, p in enumerate(pos):
        for j in range(p):
            if j < S or j > p - W:
                for c in caches:
                    c[n, _row(j, S, rows)] = torch.randn(1, D, generator=gen).to(dtype)
    x = {n: torch.randn(len(pos), h, D, generator=gen).to(dtype) for n, h in (("q", 2), ("k", 1), ("v", 1))}
    mine = [c.to(dev) for c in caches]
    o = window_attention_step(*(x[n].to(dev) for n in "qkv"), *mine, torch.tensor(pos, device=dev), W, S)
    _, ref, size, score = _step_oracle(x, caches, pos, list(range(len(pos))), W, S)
    assert o.isfinite().all() and bool(((o.double().cpu() - ref).abs() <= torch.finfo(dtype).eps / 2 * ref.abs()
                                        + (80 * score + 133) * 2.0 ** -24 * size).all())
    v = mine[1].clone()
    v[5, _row(180, S, rows), 0, 7] = float("inf")                # one that is seen: that element, and no other
    o2 = window_attention_step(x["q"].to(dev), None, None, mine[0], v, torch.tensor(pos, device=dev), W, S)
    assert torch.equal(o2[:5], o[:5]) and (o2[5, :, 7] == float("inf")).all() and torch.equal(o2[5, :, 8:], o[5, :, 8:])


def test_step_strided_caches_and_inputs(dev):
    """Keys and values in one tensor, heads outside rows, a slice of a wider pool."""
    gen = torch.Generator().manual_seed(2)
    both = torch.randn(4, 2, 2, 50, D, generator=gen).to(torch.bfloat16).to(dev)       # [slots, k or v, heads, rows, 128]
    kc, vc = (both[:, i].transpose(1, 2) for i in range(2))
    flat = [t.contiguous() for t in (kc, vc)]
    pos = torch.tensor([3, 60, 49, 200], device=dev)
    qkv = torch.randn(4, 6, D, generator=gen).to(torch.bfloat16).to(dev)
    q, k, v = qkv[:, :2], qkv[:, 2:4], qkv[:, 4:]
    a = window_attention_step(q, k, v, kc, vc, pos, 40, 3)
    b = window_attention_step(q.contiguous(), k.contiguous(), v.contiguous(), *flat, pos, 40, 3)
    assert torch.equal(a, b) and torch.equal(kc, flat[0]) and torch.equal(vc, flat[1])


def test_step_captured_beside_another(dev):
    """Two captured steps on their own caches, replayed in turn and at once on two streams: each as if alone."""
    gen = torch.Generator().manual_seed(3)
    sides = []
    for i in range(2):
        x = [torch.randn(3, h, D, generator=gen).to(torch.bfloat16).to(dev) for h in (4, 1, 1)]
        caches = [torch.randn(4, 900, 1, D, generator=gen).to(torch.bfloat16).to(dev) for _ in range(2)]
        pos = torch.tensor([5, 850, 3000], device=dev)
        run = lambda x=x, c=caches, p=pos: window_attention_step(*x, *c, p, 800, 4)  # noqa: E731
        s = torch.cuda.Stream(device=dev)
        s.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(s):
            run()
        torch.cuda.current_stream(dev).wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = run()
        sides.append((graph, o, x, caches, pos, s))
    for i in range(4):
        for _, _, x, _, pos, _ in sides:
            for t in x:
                t.copy_(torch.randn(t.shape, generator=gen).to(torch.bfloat16))
            pos += 7
        want = [window_attention_step(*x, *[c.clone() for c in caches], pos, 800, 4) for _, _, x, caches, pos, _ in sides]
        torch.cuda.synchronize()
        for graph, _, _, _, _, s in sides:
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (_, o, *_), w in zip(sides, want):
            assert torch.equal(o, w)


def test_captured_training(dev):
    """Forward and backward in one graph, replayed on new inputs with eager work in between."""
    x = {n: t.to(dev).requires_grad_(True) for n, t in _inputs(1, 1300, 2, 1, torch.bfloat16, seed=61).items()}
    do = _grad(1, 1300, 2, torch.bfloat16, 13).to(dev)

    def both(x):
        o = window_attention(x["q"], x["k"], x["v"], 100, 3)
        return [o.detach(), *torch.autograd.grad(o, [x[n] for n in "qkv"], do)]

    s = torch.cuda.Stream(device=dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        both(x)
    torch.cuda.current_stream(dev).wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both(x)
    for i in range(4):
        with torch.no_grad():
            for n, t in _inputs(1, 1300, 2, 1, torch.bfloat16, seed=70 + i).items():
                x[n].copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, both({n: t.detach().clone().requires_grad_(True) for n, t in x.items()})):
            assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
def test_prefill_then_decode(dev, dtype):
    """A layer as it is used: norm, projections, a packed prefill, its keys to a pool of caches, steps from there; the
    same as whole sequences in 64 bits."""
    torch.manual_seed(0)
    lens, new, H, Hkv, width, W, S = [75, 1, 130], 4, 4, 2, 256, 40, 3
    N = len(lens)
    x = torch.randn(N, max(lens) + new, width).to(dtype)
    w = (torch.randn((H + 2 * Hkv) * D, width) * 0.05).to(dtype).to(dev)
    wn = torch.ones(width, dtype=dtype, device=dev)
    with torch.no_grad():
        q, k, v = torch.nn.functional.linear(add_rms_norm(x.to(dev), wn)[0], w).unflatten(-1, (-1, D)).split([H, Hkv, Hkv], -2)
        pack = lambda t: torch.cat([t[i, :n] for i, n in enumerate(lens)])[None]  # noqa: E731
        cu = torch.tensor([0] + lens, device=dev).cumsum(0)
        o = window_attention(pack(q), pack(k), pack(v), W, S, cu_seqlens=cu)
        caches = [torch.full((8, S + W, Hkv, D), float("nan"), dtype=dtype, device=dev) for _ in range(2)]
        slots = torch.tensor([5, 0, 3], device=dev)
        window_cache_write(pack(k), pack(v), *caches, S, cache_indices=slots, cu_seqlens=cu)
        pos, outs = torch.tensor(lens, device=dev), []
        for t in range(new):
            outs.append(window_attention_step(*(torch.stack([a[i, n + t] for i, n in enumerate(lens)]) for a in (q, k, v)), *caches, pos + t, W, S, slots))
    for i, n in enumerate(lens):
        xi = {m: t[i:i + 1, :n + new].cpu() for m, t in (("q", q), ("k", k), ("v", v))}
        ref, size, score = _oracle(xi, [(0, 0, n + new)], W, S, D ** -0.5, None)
        _check(torch.cat([o[0, int(cu[i]):int(cu[i + 1])], *(y[i:i + 1] for y in outs)]), ref["o"][0], size["o"][0], score, n + new, "o")


def test_offsets_past_32_bits(dev):
    """Tokens 512 KiB apart, the last of them past 2^32 bytes and 2^31 elements; caches of more."""
    T, H, Hkv, apart = 8300, 4, 2, 1 << 18
    big = torch.empty(T * apart, dtype=torch.bfloat16, device=dev)
    gen = torch.Generator(device=dev).manual_seed(3)
    near, far = [], []
    for i, h in enumerate((H, Hkv, Hkv, H)):
        near.append(torch.randn(1, T, h, D, generator=gen, device=dev).to(torch.bfloat16))
        far.append(big.as_strided((1, T, h, D), (0, apart, D, 1), 4096 * i).copy_(near[-1]))
    out = []
    for q, k, v, do in (near, far):
        leaf = [t.detach().requires_grad_() for t in (q, k, v)]
        o = window_attention(*leaf, 300, 3)
        out.append([o.detach(), *torch.autograd.grad(o, leaf, do)])
    for a, b in zip(*out):
        assert torch.equal(a, b)
    slots = 305
    wide = [big.as_strided((slots, 64, 1, D), (apart * 27, apart // 64, D, 1), 128 * i) for i in range(2)]
    assert apart * 27 * (slots - 1) > 1 << 31
    small = [torch.empty(2, 64, 1, D, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    at, pos = torch.tensor([slots - 1, 0], device=dev), torch.tensor([0, 0], device=dev)
    tokens = [near[1][:, :80, :1].expand(2, -1, -1, -1), near[2][:, :80, :1].expand(2, -1, -1, -1)]
    with torch.no_grad():
        window_cache_write(*tokens, *small, 2, pos, None)
        window_cache_write(*tokens, *wide, 2, pos, at)
        for a, b in zip(small, wide):
            assert torch.equal(a[0], b[slots - 1]) and torch.equal(a[1], b[0])
        args = [t[0, :2] for t in (near[0], near[1][:, :, :1], near[2][:, :, :1])]
        x = window_attention_step(*args, *small, pos + 80, 50, 2)
        y = window_attention_step(*args, *wide, pos + 80, 50, 2, at)
    assert torch.equal(x, y)
