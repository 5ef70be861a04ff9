"""The gated delta rule and its single-token step on the GPU against the recurrence in 64 bits.

Tolerances.  A result of type t carries one rounding, at most eps(t) / 2 of its value.  Under
it lie fp32 sums: with keys of unit length and beta <= 1 no token's update lengthens an earlier
error, so after T tokens the states hold at most T times the roundings of one update, and a
result adds a sum over 128 elements, over a chunk's tokens at most 64 and, for the gradients of
g, over 128 x 128 products: ROUNDS (16 for outputs, 64 for gradients) roundings of 2^-24 of the
largest value for each of T + 128 terms.  Gradients that are sums over the v heads of a q/k
head add their number of such terms, and for bf16 the largest of the heads' values counts.  Under
2^-126, fp32's smallest normal number, a factor e^g keeps fewer bits or is flushed: 2^-126 more
(e^-90 = 2^-129.8 in front of a gradient of order 1 leaves nothing of it).
"""

import pytest
import torch

from gsa_gdn_benchmarkstudy_amd import add_rms_norm, gated_delta_rule, gated_delta_step
from tests import delta_oracle as orc

pytestmark = pytest.mark.gpu

D = 128
NAMES = ("q", "k", "v", "g", "beta")


def _inputs(B, T, Hk, Hv, dtype, seed, strong=False):
    gen = torch.Generator().manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, generator=gen)

    q, k = (torch.nn.functional.normalize(rn(B, T, Hk, D), dim=-1).to(dtype) for _ in range(2))
    if strong:                                   # keys that hardly differ: the largest entries of the inverse
        k = torch.nn.functional.normalize(k[:, :1].float() + 0.02 * rn(B, T, Hk, D), dim=-1).to(dtype)
    v = rn(B, T, Hv, D).to(dtype)
    g = -torch.exp(rn(B, T, Hv) - 2)
    beta = torch.sigmoid(rn(B, T, Hv) + (6 if strong else 0))
    return dict(q=q, k=k, v=v, g=g, beta=beta)


def _check(got, ref, T, rounds, name):
    assert tuple(got.shape) == tuple(ref.shape), name
    if not got.numel():
        return
    half = torch.finfo(got.dtype).eps / 2
    tol = half * ref.abs() + rounds * (T + 128) * 2.0 ** -24 * ref.abs().max() + 2.0 ** -126
    err = (got.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), f"{name}: {(err / tol).max():.2f} of the tolerance (|err| {err.max():.2e})"


def _run(x, dev, state=None, want=True, cu=None, grads=None, scale=None):
    """gated_delta_rule on the device; with grads (do, dS) the gradients too."""
    leaf = {n: t.to(dev).requires_grad_(grads is not None) for n, t in x.items()}
    st = None if state is None else state.to(dev).requires_grad_(grads is not None)
    o, S = gated_delta_rule(*(leaf[n] for n in NAMES), scale=scale, initial_state=st, output_final_state=want, cu_seqlens=cu)
    if grads is None:
        return o, S, None
    ins = [leaf[n] for n in NAMES] + ([st] if st is not None else [])
    outs, gr = [o], [grads[0].to(dev)]
    if want:
        outs.append(S)
        gr.append(grads[1].to(dev))
    d = torch.autograd.grad(outs, ins, gr)
    return o.detach(), None if S is None else S.detach(), dict(zip(NAMES + ("state",), d))


def _oracle(x, spans, state=None, grads=None, scale=D ** -0.5, want=True):
    """The recurrence over spans [(row, start, end)]; outputs and gradients laid out as the op's."""
    leaf = {n: t.double().requires_grad_(grads is not None) for n, t in x.items()}
    st = None if state is None else state.double().requires_grad_(grads is not None)
    o = torch.zeros(x["v"].shape, dtype=torch.float64)
    finals = []
    for i, (b, s, e) in enumerate(spans):
        oi, S = orc.rule(*(leaf[n][b, s:e] for n in NAMES), scale, None if st is None else st[i])
        finals.append(S)
        if e > s:
            mask = torch.zeros(o.shape[0], o.shape[1], 1, 1, dtype=torch.float64)
            mask[b, s:e] = 1
            o = o + mask * torch.nn.functional.pad(oi, (0, 0, 0, 0, s, o.shape[1] - e))[None]
    S = torch.stack(finals)
    if grads is None:
        return o, S, None
    ins = [leaf[n] for n in NAMES] + ([st] if st is not None else [])
    outs, gr = ([o, S], [grads[0].double(), grads[1].double()]) if want else ([o], [grads[0].double()])
    d = torch.autograd.grad(outs, ins, gr, allow_unused=True)
    d = [torch.zeros_like(i) if t is None else t for i, t in zip(ins, d)]
    return o.detach(), S.detach(), dict(zip(NAMES + ("state",), d))


def _compare(got, ref, T, share=1, want=True):
    _check(got[0], ref[0], T, 16, "o")
    if want:
        _check(got[1], ref[1], T, 16, "state")
    if got[2] is not None:
        for n, d in got[2].items():
            _check(d, ref[2][n], T, 64 * share, "d" + n)


CASES = [(1, 1, 1, 1), (2, 2, 1, 2), (1, 31, 2, 2), (1, 32, 1, 1), (2, 33, 1, 3), (1, 63, 1, 2), (1, 64, 2, 2), (3, 65, 1, 1),
         (1, 129, 2, 4), (2, 200, 2, 2)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,T,Hk,Hv", CASES)
def test_forward(dev, B, T, Hk, Hv, dtype):
    print(f"forward {dtype} B={B} T={T} Hk={Hk} Hv={Hv}", flush=True)
    x = _inputs(B, T, Hk, Hv, dtype, seed=T)
    spans = [(b, 0, T) for b in range(B)]
    _compare(_run(x, dev), _oracle(x, spans), T)
    state = torch.randn(B, Hv, D, D, generator=torch.Generator().manual_seed(5))
    _compare(_run(x, dev, state), _oracle(x, spans, state), T)
    assert _run(x, dev, want=False)[1] is None


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,T,Hk,Hv", CASES)
@pytest.mark.parametrize("with_state", [False, True])
def test_backward(dev, B, T, Hk, Hv, dtype, with_state):
    print(f"backward {dtype} B={B} T={T} Hk={Hk} Hv={Hv} state={with_state}", flush=True)
    x = _inputs(B, T, Hk, Hv, dtype, seed=T + 1)
    gen = torch.Generator().manual_seed(6)
    state = torch.randn(B, Hv, D, D, generator=gen) if with_state else None
    grads = (torch.randn(B, T, Hv, D, generator=gen).to(dtype), torch.randn(B, Hv, D, D, generator=gen))
    spans = [(b, 0, T) for b in range(B)]
    _compare(_run(x, dev, state, with_state, grads=grads), _oracle(x, spans, state, grads, want=with_state), T, Hv // Hk, with_state)


PACKS = [[1], [5, 0, 64, 1, 65, 63], [0, 0, 3], [130, 32, 33], [64, 64, 64]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens", PACKS)
@pytest.mark.parametrize("lead,trail,idx", [(0, 0, torch.int32), (3, 37, torch.int64)])
def test_packed(dev, lens, lead, trail, idx, dtype):
    """Packed sequences, empty ones among them; rows before the first and behind the last stay 0."""
    print(f"packed {dtype} {lens} lead={lead} trail={trail}", flush=True)
    T, N, Hk, Hv = lead + sum(lens) + trail, len(lens), 1, 2
    cu = torch.tensor([lead] + lens).cumsum(0).to(idx)
    x = _inputs(1, T, Hk, Hv, dtype, seed=N)
    gen = torch.Generator().manual_seed(7)
    state = torch.randn(N, Hv, D, D, generator=gen)
    grads = (torch.randn(1, T, Hv, D, generator=gen).to(dtype), torch.randn(N, Hv, D, D, generator=gen))
    spans = [(0, int(cu[i]), int(cu[i + 1])) for i in range(N)]
    got, ref = _run(x, dev, state, cu=cu.to(dev), grads=grads), _oracle(x, spans, state, grads)
    _compare(got, ref, T, Hv // Hk)
    outside = torch.ones(T, dtype=torch.bool)
    outside[lead:T - trail] = False
    for t in (got[0], *(got[2][n] for n in NAMES)):
        assert not t[0, outside.to(dev)].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,T,Hk,Hv,lens", [(1, 900, 1, 1, None), (2, 1537, 1, 2, None), (1, 2200, 1, 2, [900, 0, 1, 1000, 299])])
def test_segments(dev, B, T, Hk, Hv, lens, dtype):
    """Long sequences with few heads: cut into segments that are joined again (packed ones of several lengths)."""
    print(f"segments {dtype} B={B} T={T} {lens}", flush=True)
    x = _inputs(B, T, Hk, Hv, dtype, seed=T)
    N = B if lens is None else len(lens)
    gen = torch.Generator().manual_seed(14)
    state = torch.randn(N, Hv, D, D, generator=gen)
    grads = (torch.randn(B, T, Hv, D, generator=gen).to(dtype), torch.randn(N, Hv, D, D, generator=gen))
    cu = None if lens is None else torch.tensor([0] + lens).cumsum(0)
    spans = [(b, 0, T) for b in range(B)] if lens is None else [(0, int(cu[i]), int(cu[i + 1])) for i in range(N)]
    got = _run(x, dev, state, cu=None if cu is None else cu.to(dev), grads=grads)
    _compare(got, _oracle(x, spans, state, grads), T, Hv // Hk)
    _check(_run(x, dev, cu=None if cu is None else cu.to(dev))[0], _oracle(x, spans)[0], T, 16, "o")


def test_offsets_outside_the_tokens_touch_nothing(dev):
    """Offsets past T or descending: held within the tokens, other sequences are right."""
    x = _inputs(1, 100, 1, 1, torch.bfloat16, seed=3)
    o, S, _ = _run(x, dev, cu=torch.tensor([0, 40, 1 << 30], dtype=torch.int64, device=dev))
    ref = _oracle(x, [(0, 0, 40), (0, 40, 100)])
    _compare((o, S, None), ref, 100)
    o, S, _ = _run(x, dev, cu=torch.tensor([-5, 40, 20], dtype=torch.int32, device=dev))
    ref = _oracle(x, [(0, 0, 40)])
    _check(o[:, :40], ref[0][:, :40], 100, 16, "o")
    assert not o[:, 40:].any() and not S[1].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["reset", "far", "keep", "idle", "alike", "scaled"])
def test_gates(dev, kind, dtype):
    """Decays at both ends, betas of 0, keys that hardly differ, a scale of one's own."""
    print(f"gates {kind} {dtype}", flush=True)
    T = 150
    x = _inputs(2, T, 2, 2, dtype, seed=11, strong=kind == "alike")
    if kind == "reset":                          # e^-inf, also twice in a row and as a chunk's first and last token
        for t in (0, 31, 32, 63, 64, 65, 140):
            x["g"][:, t] = -float("inf")
    elif kind == "far":                          # below fp32's smallest, and sums that lose small terms
        x["g"][:, ::7] = -90.0
        x["g"][:, 50] = -1e30
    elif kind == "keep":
        x["g"].zero_()
    elif kind == "idle":
        x["beta"][:, ::3] = 0
    gen = torch.Generator().manual_seed(8)
    state = torch.randn(2, 2, D, D, generator=gen)
    grads = (torch.randn(2, T, 2, D, generator=gen).to(dtype), torch.randn(2, 2, D, D, generator=gen))
    scale = 0.31 if kind == "scaled" else D ** -0.5
    x64 = {n: t.clone() for n, t in x.items()}
    x64["g"] = x64["g"].clamp_min(-2000.)        # the oracle's e^g is 0 as well, its gradient 0 and not inf * 0
    _compare(_run(x, dev, state, grads=grads, scale=scale), _oracle(x64, [(0, 0, T), (1, 0, T)], state, grads, scale), T)


def test_gradient_against_differences(dev):
    """The kernels' gradient along random directions against differences of the recurrence in 64 bits."""
    T = 70
    x = _inputs(1, T, 1, 2, torch.float32, seed=21)
    gen = torch.Generator().manual_seed(9)
    state = torch.randn(1, 2, D, D, generator=gen)
    do, dS = torch.randn(1, T, 2, D, generator=gen), torch.randn(1, 2, D, D, generator=gen)
    _, _, d = _run(x, dev, state, grads=(do, dS))
    x64, s64 = {n: t.double() for n, t in x.items()}, state.double()

    def loss(x, s):
        o, S, _ = _oracle(x, [(0, 0, T)], s)
        return (o * do.double()).sum() + (S * dS.double()).sum()

    for n in NAMES + ("state",):
        r = torch.randn((state if n == "state" else x[n]).shape, generator=gen).double()
        h = 1e-5
        up, dn = ((loss(x64, s64 + e * r) if n == "state" else loss(x64 | {n: x64[n] + e * r}, s64)) for e in (h, -h))
        want, got = (up - dn) / (2 * h), (d[n].double().cpu() * r).sum()
        # differences: h^2 of a third derivative and 2^-52 / h of the loss; the gradient's own errors add up like a walk
        tol = 64 * (T + 128) * 2.0 ** -24 * d[n].abs().max().item() * r.norm() + 1e-6 * abs(want)
        assert abs(want - got) <= tol, (n, want, got)


def test_strided_views_and_broadcasts(dev):
    """Views of one projection output, heads broadcast with stride 0, transposed layouts: the same bits as copies."""
    gen = torch.Generator().manual_seed(31)
    B, T, H = 2, 90, 2
    big = torch.randn(B, T, 3 * H * D + 64, generator=gen).to(torch.bfloat16).to(dev)
    q, k, v = (big[..., i * H * D:(i + 1) * H * D].view(B, T, H, D) for i in range(3))
    k = torch.nn.functional.normalize(k.float(), dim=-1).to(torch.bfloat16).transpose(1, 2).contiguous().transpose(1, 2)
    gb = torch.rand(B, H, T, 2, generator=gen).to(dev)
    g, beta = -gb[..., 0].transpose(1, 2), gb[..., 1].transpose(1, 2)
    a = gated_delta_rule(q, k, v, g, beta, output_final_state=True)
    b = gated_delta_rule(*(t.contiguous() for t in (q, k, v, g, beta)), output_final_state=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    odd = torch.empty(B * T * H * D + 1, device=dev, dtype=torch.bfloat16)[1:].view(B, T, H, D)
    odd.copy_(q)                                 # 2-byte aligned: copied
    assert torch.equal(gated_delta_rule(odd, k, v, g, beta)[0], b[0])
    one = k[:, :, :1].detach().requires_grad_(True)
    o, _ = gated_delta_rule(q, one.expand(B, T, H, D), v, g, beta)
    do = torch.randn(o.shape, generator=gen).to(torch.bfloat16).to(dev)
    (d1,) = torch.autograd.grad(o, one, do)
    full = k[:, :, :1].expand(B, T, H, D).contiguous().requires_grad_(True)
    (d2,) = torch.autograd.grad(gated_delta_rule(q, full, v, g, beta)[0], full, do)
    assert torch.equal(d1, d2.sum(2, keepdim=True))
    (d3,) = torch.autograd.grad(gated_delta_rule(q, full, v, g, beta)[0].sum(), full)      # an expanded gradient
    (d4,) = torch.autograd.grad(gated_delta_rule(q, full, v, g, beta)[0], full, torch.ones_like(o))
    assert torch.equal(d3, d4)


def test_beta_in_bf16(dev):
    x = _inputs(1, 100, 1, 2, torch.bfloat16, seed=41)
    x["beta"] = x["beta"].to(torch.bfloat16)
    gen = torch.Generator().manual_seed(42)
    grads = (torch.randn(1, 100, 2, D, generator=gen).to(torch.bfloat16), torch.randn(1, 2, D, D, generator=gen))
    got = _run(x, dev, grads=grads)
    assert got[2]["beta"].dtype == torch.bfloat16
    _compare(got, _oracle(x, [(0, 0, 100)], grads=grads), 100, 2)


def test_same_bits_and_other_stream(dev):
    """Two runs, and one on another stream with its own allocations in between: the same bits."""
    x = _inputs(2, 300, 2, 4, torch.bfloat16, seed=51)
    gen = torch.Generator().manual_seed(52)
    grads = (torch.randn(2, 300, 4, D, generator=gen).to(torch.bfloat16), torch.randn(2, 4, D, D, generator=gen))
    a = _run(x, dev, grads=grads)
    s = torch.cuda.Stream(device=dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        b = _run(x, dev, grads=grads)
    torch.cuda.current_stream(dev).wait_stream(s)
    for y in (b, _run(x, dev, grads=grads)):
        assert torch.equal(a[0], y[0]) and torch.equal(a[1], y[1])
        for n in a[2]:
            assert torch.equal(a[2][n], y[2][n]), n


def test_captured_forward_and_step(dev):
    """A prefill and a decoding step in one graph, replayed on new inputs with eager work in between."""
    x = {n: t.to(dev) for n, t in _inputs(2, 130, 1, 2, torch.bfloat16, seed=61).items()}
    one = {n: t[:, 0].contiguous().to(dev) for n, t in _inputs(2, 1, 1, 2, torch.bfloat16, seed=62).items()}

    def both():
        o, S = gated_delta_rule(*(x[n] for n in NAMES), output_final_state=True)
        return o, gated_delta_step(*(one[n] for n in NAMES), S), S

    with torch.no_grad():
        s = torch.cuda.Stream(device=dev)
        s.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(s):
            both()
        torch.cuda.current_stream(dev).wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = both()
        for i in range(4):
            for n, t in _inputs(2, 130, 1, 2, torch.bfloat16, seed=70 + i).items():
                x[n].copy_(t)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, both()):
                assert torch.equal(a, b)


def test_no_gradient_needed_keeps_nothing(dev):
    x = {n: t.to(dev) for n, t in _inputs(1, 64, 1, 1, torch.bfloat16, seed=71).items()}
    assert not gated_delta_rule(*(x[n] for n in NAMES))[0].requires_grad
    x["v"].requires_grad_(True)
    with torch.no_grad():
        assert not gated_delta_rule(*(x[n] for n in NAMES))[0].requires_grad
    o, S = gated_delta_rule(*(x[n] for n in NAMES), output_final_state=True)
    (dv,) = torch.autograd.grad(S.sum(), x["v"])                 # o unused
    assert dv.abs().sum() > 0
    o, _ = gated_delta_rule(*(x[n] for n in NAMES))
    (dv,) = torch.autograd.grad(o.float().sum(), x["v"], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dv.sum(), x["v"])                    # once differentiable


# ---------------------------------------------------------------------------
# The step
# ---------------------------------------------------------------------------

def _step_oracle(x, pool, at, scale=D ** -0.5):
    pool, o = pool.double().clone(), torch.zeros(x["v"].shape, dtype=torch.float64)
    for i, s in enumerate(at):
        if 0 <= s < pool.shape[0]:
            oi, S = orc.rule(*(x[n][i:i + 1].double() for n in NAMES), scale, pool[s])
            o[i], pool[s] = oi[0], S
    return o, pool


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,Hk,Hv,slots,at", [
    (1, 1, 1, 1, None), (3, 2, 4, 5, None), (4, 1, 3, 9, [8, 0, 3, 5]), (5, 2, 2, 4, [3, -1, 0, 4, 1]),
    (6, 1, 2, 3, [1, 2, 1, -7, 1, 0]), (2, 1, 1, 2, [1 << 20, -1])])
@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
def test_step(dev, N, Hk, Hv, slots, at, idx, dtype):
    """States of rows, padding, an index named more than once (consecutive tokens)."""
    x = {n: t[0] for n, t in _inputs(1, N, Hk, Hv, dtype, seed=N).items()}
    pool = torch.randn(slots, Hv, D, D, generator=torch.Generator().manual_seed(3))
    ref = _step_oracle(x, pool, range(N) if at is None else at)
    mine = pool.to(dev)
    o = gated_delta_step(*(x[n].to(dev) for n in NAMES), mine, None if at is None else torch.tensor(at, dtype=idx, device=dev))
    _check(o, ref[0], N, 16, "o")
    _check(mine, ref[1], N, 16, "state")
    for s in set(range(slots)) - set(range(N) if at is None else at):
        assert torch.equal(mine[s].cpu(), pool[s])


def test_step_many_rows(dev):
    """More rows than a block has threads, every third index twice."""
    N, slots = 700, 800
    x = {n: t[0] for n, t in _inputs(1, N, 1, 1, torch.bfloat16, seed=5).items()}
    at = [(i if i % 3 else 2 * i % N) for i in range(N)]
    pool = torch.randn(slots, 1, D, D, generator=torch.Generator().manual_seed(4))
    ref = _step_oracle(x, pool, at)
    mine = pool.to(dev)
    o = gated_delta_step(*(x[n].to(dev) for n in NAMES), mine, torch.tensor(at, device=dev))
    _check(o, ref[0], N, 16, "o")
    _check(mine, ref[1], N, 16, "state")


def test_step_strided_state_and_inputs(dev):
    x = {n: t[0].to(dev) for n, t in _inputs(1, 4, 2, 2, torch.bfloat16, seed=6).items()}
    big = torch.randn(5, 3, 2, D, D, device=dev)
    keep = big.clone()
    a = gated_delta_step(*(x[n] for n in NAMES), big[:, 1])
    st = keep[:, 1].contiguous()
    wide = torch.zeros(4, 2, 2 * D, device=dev, dtype=torch.bfloat16)
    wide[..., 1:D + 1] = x["q"]
    b = gated_delta_step(wide[..., 1:D + 1], *(x[n] for n in NAMES[1:]), st)
    assert torch.equal(a, b) and torch.equal(big[:, 1], st)
    assert torch.equal(big[:, 0], keep[:, 0]) and torch.equal(big[:, 2], keep[:, 2])


# ---------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------

def test_prefill_then_decode(dev):
    """A mixer as it is used: norm with the residual, projections, q and k normed by heads, the rule over
    a prompt, then steps from its state; the same as the rule over prompt and steps, in 64 bits."""
    torch.manual_seed(0)
    B, T, new, H, width = 2, 75, 3, 2, 256
    dt = torch.bfloat16
    x, res = (torch.randn(B, T + new, width).to(dt) for _ in range(2))
    w = {n: (torch.randn(r, width) * 0.05).to(dt).to(dev) for n, r in (("qkv", 3 * H * D), ("gate", 2 * H))}
    wn, unit = (1 + 0.1 * torch.randn(width)).to(dt).to(dev), torch.full((D,), D ** -0.5, dtype=dt, device=dev)

    def heads(x, res):
        y, h = add_rms_norm(x.to(dev), wn, residual=res.to(dev))
        q, k, v = torch.nn.functional.linear(y, w["qkv"]).unflatten(-1, (3, H, D)).unbind(-3)
        q, k = add_rms_norm(q, unit)[0], add_rms_norm(k, unit)[0]
        a, b = torch.nn.functional.linear(y, w["gate"]).float().chunk(2, -1)
        return dict(q=q, k=k, v=v, g=-torch.nn.functional.softplus(a), beta=torch.sigmoid(b)), h

    with torch.no_grad():
        every, h = heads(x, res)
        assert torch.equal(h.cpu(), x + res)
        o, S = gated_delta_rule(*(every[n][:, :T] for n in NAMES), output_final_state=True)
        outs = [o]
        for t in range(T, T + new):
            outs.append(gated_delta_step(*(every[n][:, t] for n in NAMES), S)[:, None])
    ref = _oracle({n: t.cpu() for n, t in every.items()}, [(b, 0, T + new) for b in range(B)])
    _check(torch.cat(outs, 1), ref[0], T + new, 16, "o")
    _check(S, ref[1], T + new, 16, "state")


# --------------------------------------------------------------------------- calls as programs make them

def _leaves(x, dev):
    return [x[n].to(dev).requires_grad_(True) for n in NAMES]


def _train(leaf, do, cu=None):
    o, S = gated_delta_rule(*leaf, output_final_state=True, cu_seqlens=cu)
    return (o, S) + torch.autograd.grad([o, S], leaf, [do, torch.ones_like(S)])


@pytest.mark.parametrize("T,Hk,Hv,offsets", [(130, 2, 2, None), (1500, 1, 2, None), (900, 2, 4, [0, 1, 64, 64, 700, 850])])
def test_captured_training(dev, T, Hk, Hv, offsets):
    """Forward and backward in a graph (in one piece, by segments, packed with rows outside), replayed
    on new inputs with eager calls in between: the eager call's bits."""
    leaf = _leaves(_inputs(1, T, Hk, Hv, torch.bfloat16, seed=81), dev)
    do = torch.randn(1, T, Hv, D, device=dev, dtype=torch.bfloat16)
    cu = None if offsets is None else torch.tensor(offsets, device=dev, dtype=torch.int32)
    s = torch.cuda.Stream(device=dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        _train(leaf, do, cu)
    torch.cuda.current_stream(dev).wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _train(leaf, do, cu)
    for i in range(4):
        new = _inputs(1, T, Hk, Hv, torch.bfloat16, seed=90 + i)
        with torch.no_grad():
            for t, n in zip(leaf, NAMES):
                t.copy_(new[n])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, _train(_leaves(new, dev), do, cu)):
            assert torch.equal(a, b)


def test_two_graphs_at_once(dev):
    """Two graphs with a memory pool each, replayed on two streams at the same time."""
    graphs, outs, ins, want = [], [], [], []
    with torch.no_grad():
        for i in range(2):
            x = {n: t.to(dev) for n, t in _inputs(1, 3000, 2, 4, torch.bfloat16, seed=100 + i).items()}
            want.append(gated_delta_rule(*(x[n] for n in NAMES), output_final_state=True))
            ins.append(x)
        torch.cuda.synchronize()
        for x in ins:
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                outs.append(gated_delta_rule(*(x[n] for n in NAMES), output_final_state=True))
        streams = [torch.cuda.Stream(device=dev) for _ in graphs]
        for _ in range(3):
            for o, S in outs:
                o.zero_(), S.zero_()
            torch.cuda.synchronize()
            for s, graph in zip(streams, graphs):
                with torch.cuda.stream(s):
                    graph.replay()
            torch.cuda.synchronize()
            for (o, S), (o2, S2) in zip(outs, want):
                assert torch.equal(o, o2) and torch.equal(S, S2)


def test_two_threads(dev):
    """Training calls from two threads, each on a stream of its own, at the same time."""
    import threading

    jobs, failed = [], []
    for i in range(2):
        x = _inputs(1, 700 + 900 * i, 1, 2, torch.bfloat16, seed=110 + i)
        do = torch.randn(x["v"].shape, generator=torch.Generator().manual_seed(i)).to(dev, torch.bfloat16)
        jobs.append((x, do, _train(_leaves(x, dev), do)))
    torch.cuda.synchronize()

    def work(x, do, want):
        try:
            s = torch.cuda.Stream(device=dev)
            with torch.cuda.stream(s):
                for _ in range(6):
                    got = _train(_leaves(x, dev), do)
                    s.synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(got, want))
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_nothing_to_do(dev):
    """No tokens, no sequences' tokens, no rows."""
    z = dict(device=dev, dtype=torch.bfloat16)
    S0 = torch.randn(2, 2, D, D, device=dev)
    x = [torch.zeros(2, 0, 1, D, **z), torch.zeros(2, 0, 1, D, **z), torch.zeros(2, 0, 2, D, **z), torch.zeros(2, 0, 2, device=dev),
         torch.zeros(2, 0, 2, device=dev)]
    o, S = gated_delta_rule(*x, initial_state=S0, output_final_state=True)
    assert o.shape == x[2].shape and torch.equal(S, S0) and S.data_ptr() != S0.data_ptr()
    x = {n: t.to(dev) for n, t in _inputs(1, 70, 1, 2, torch.bfloat16, seed=5).items()}
    cu = torch.zeros(3, device=dev, dtype=torch.int64)
    leaf = [t.requires_grad_(True) for t in x.values()]
    st = S0.clone().requires_grad_(True)
    o, S = gated_delta_rule(*leaf, initial_state=st, output_final_state=True, cu_seqlens=cu)
    assert not o.any() and torch.equal(S, S0)
    d = torch.autograd.grad([o, S], leaf + [st], [torch.ones_like(o), S0])
    assert not any(t.any() for t in d[:-1]) and torch.equal(d[-1], S0)
    e = [torch.zeros(0, 1, D, **z), torch.zeros(0, 1, D, **z), torch.zeros(0, 2, D, **z), torch.zeros(0, 2, device=dev),
         torch.zeros(0, 2, device=dev)]
    keep = S0.clone()
    assert gated_delta_step(*e, S0).shape == (0, 2, D) and torch.equal(S0, keep)


def test_same_tensor_in_several_places(dev):
    """q, k and v one leaf: its gradient is the sum of theirs."""
    x = _inputs(1, 200, 2, 2, torch.float32, seed=120)
    one = x["k"].to(dev)
    g, b = x["g"].to(dev), x["beta"].to(dev)
    do = torch.randn(1, 200, 2, D, device=dev)
    leaf = one.clone().requires_grad_(True)
    got, = torch.autograd.grad(gated_delta_rule(leaf, leaf, leaf, g, b)[0], leaf, do)
    three = [one.clone().requires_grad_(True) for _ in range(3)]
    parts = torch.autograd.grad(gated_delta_rule(*three, g, b)[0], three, do)
    # three fp32 addends in another order: two roundings of at most their sum of magnitudes
    tol = 2 * 2.0 ** -24 * sum(p.abs() for p in parts)
    assert bool(((got - sum(parts)).abs() <= tol + 2.0 ** -24 * got.abs()).all())


def test_tokens_far_apart(dev):
    """Tokens 32 MiB and more apart (a view of a large buffer) are copied, not refused."""
    x = _inputs(1, 3, 1, 1, torch.bfloat16, seed=130)
    far = torch.empty(3 * (1 << 24), device=dev, dtype=torch.bfloat16).as_strided((1, 3, 1, D), (1, 1 << 24, D, 1))
    far.copy_(x["k"])
    y = {n: t.to(dev) for n, t in x.items()}
    o, S = gated_delta_rule(y["q"], far, y["v"], y["g"], y["beta"], output_final_state=True)
    o2, S2 = gated_delta_rule(*(y[n] for n in NAMES), output_final_state=True)
    assert torch.equal(o, o2) and torch.equal(S, S2)


def test_offsets_past_32_bits(dev):
    """2**19 tokens of 16 heads: elements of the kept states, and bytes of every input, past 2**31.  The last
    tokens' outputs and gradients are those of a call on them alone from the state before them; the first
    tokens' gradients those of a call on the first 4096 (a decay of e^-0.1 a token leaves
    e^-380 of what lies behind)."""
    T, Hk, Hv, tail = (1 << 19) + 100, 8, 16, 612
    gen = torch.Generator(device=dev).manual_seed(7)

    def rn(*s):
        return torch.randn(*s, generator=gen, device=dev, dtype=torch.bfloat16)

    x = dict(q=rn(1, T, Hk, D), k=rn(1, T, Hk, D).mul_(D ** -0.5), v=rn(1, T, Hv, D))
    x.update(g=torch.full((1, T, Hv), -0.1, device=dev), beta=torch.full((1, T, Hv), 0.5, device=dev))
    do = rn(1, T, Hv, D)

    def run(a, b, state=None):
        leaf = [x[n][:, a:b].requires_grad_(True) if n in ("q", "k", "v") else x[n][:, a:b].clone().requires_grad_(True) for n in NAMES]
        o, S = gated_delta_rule(*leaf, initial_state=state, output_final_state=True)
        return o.detach(), S.detach(), torch.autograd.grad(o, leaf, do[:, a:b])

    whole = run(0, T)
    with torch.no_grad():
        _, S = gated_delta_rule(*(x[n][:, :T - tail] for n in NAMES), output_final_state=True)
    last = run(T - tail, T, S)
    first = run(0, 4096)

    def near(a, b, name):
        # both sides err by fp32 roundings of sums that the decay keeps to some 10 tokens, and round to their type
        scale = b.abs().max().float()
        tol = 2 * torch.finfo(a.dtype).eps / 2 * b.float().abs() + 64 * (64 + 128) * 2.0 ** -24 * scale
        assert bool(((a.float() - b.float()).abs() <= tol).all()), name

    near(whole[0][:, -tail:], last[0], "o")
    near(whole[1], last[1], "state")
    for n, a, b, c in zip(NAMES, whole[2], last[2], first[2]):
        near(a[:, -tail:], b, "d" + n + " at the end")
        near(a[:, :256], c[:, :256], "d" + n + " at the start")


def test_step_in_a_large_pool(dev):
    """States more than 2**31 elements behind the first."""
    slots, Hv = 8200, 16
    pool = torch.zeros(slots, Hv, D, D, device=dev)
    x = {n: t[0].to(dev) for n, t in _inputs(1, 3, 8, Hv, torch.bfloat16, seed=140).items()}
    small = torch.randn(3, Hv, D, D, generator=torch.Generator().manual_seed(3)).to(dev)
    at = torch.tensor([slots - 1, 0, 8195], device=dev)
    pool[at] = small
    o = gated_delta_step(*(x[n] for n in NAMES), pool, at)
    o2 = gated_delta_step(*(x[n] for n in NAMES), small)
    assert torch.equal(o, o2) and torch.equal(pool[at], small)
    pool[at] = 0
    assert not pool.any()


def test_step_counts_as_a_change_of_the_state(dev):
    """A graph that kept the state refuses its backward pass after a step has written to it."""
    x = {n: t[:, 0].to(dev) for n, t in _inputs(1, 1, 1, 1, torch.bfloat16, seed=150).items()}
    state = torch.randn(1, 1, D, D, device=dev)
    w = torch.ones_like(state).requires_grad_(True)
    y = (state * w).sum()
    with torch.no_grad():
        gated_delta_step(*(x[n] for n in NAMES), state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        gated_delta_step(*(x[n] for n in NAMES), torch.zeros(1, 1, D, D, device=dev))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_nan_stays_where_it_is(dev, dtype):
    """NaN in rows outside the sequences, in another sequence and in another batch row changes nothing here."""
    offsets = [5, 75, 75, 140, 900, 1000]        # (not a multiple of the chunk anywhere)
    x = _inputs(1, 1010, 1, 2, dtype, seed=160)
    do = torch.randn(1, 1010, 2, D, generator=torch.Generator().manual_seed(1)).to(dtype)
    cu = torch.tensor(offsets, device=dev)
    want = _train(_leaves(x, dev), do.to(dev), cu)
    bad = {n: t.clone() for n, t in x.items()}
    do2 = do.clone()
    for t in list(bad.values()) + [do2]:
        t[:, :5] = t[:, 1000:] = t[:, 75:140] = float("nan")
    got = _train(_leaves(bad, dev), do2.to(dev), cu)
    for a, b in zip((got[0],) + got[2:], (want[0],) + want[2:]):
        assert not a[:, :5].any() and not a[:, 1000:].any()
        assert torch.equal(a[:, 5:75], b[:, 5:75]) and torch.equal(a[:, 140:1000], b[:, 140:1000])
    assert torch.equal(got[1][[0, 1, 3, 4]], want[1][[0, 1, 3, 4]])

    x = _inputs(3, 70, 1, 2, dtype, seed=161)
    do = torch.randn(3, 70, 2, D, generator=torch.Generator().manual_seed(2)).to(dtype)
    want = _train(_leaves(x, dev), do.to(dev))
    for t in list(x.values()) + [do]:
        t[1] = float("nan")
    for a, b in zip(_train(_leaves(x, dev), do.to(dev)), want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])


@pytest.mark.parametrize("T", [100, 1500])
def test_backward_twice(dev, T):
    """What the forward kept is not used up (in one piece, by segments)."""
    leaf = _leaves(_inputs(1, T, 1, 2, torch.bfloat16, seed=170), dev)
    st = torch.randn(1, 2, D, D, device=dev).requires_grad_(True)
    o, S = gated_delta_rule(*leaf, initial_state=st, output_final_state=True)
    gr = [torch.randn_like(o), torch.randn_like(S)]
    first = torch.autograd.grad([o, S], leaf + [st], gr, retain_graph=True)
    for a, b in zip(first, torch.autograd.grad([o, S], leaf + [st], gr)):
        assert torch.equal(a, b)


def test_finite_padding(dev):
    """What lies behind a row's tokens, however large, changes no output and no gradient before it."""
    x = _inputs(2, 200, 1, 2, torch.bfloat16, seed=180)
    do = torch.randn(2, 200, 2, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    do[:, 150:] = 0
    outs = []
    for fill in (0.0, 1e4):
        y = {n: t.clone() for n, t in x.items()}
        for n in ("q", "v"):
            y[n][:, 150:] = fill
        leaf = _leaves(y, dev)
        o, _ = gated_delta_rule(*leaf)
        outs.append([t[:, :150] for t in (o, *torch.autograd.grad(o, leaf, do.to(dev)))])
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_differentiable_once(dev):
    leaf = _leaves(_inputs(1, 20, 1, 1, torch.float32, seed=190), dev)
    o, _ = gated_delta_rule(*leaf)
    d, = torch.autograd.grad(o.sum(), leaf[:1], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(o.sum() + d.square().sum(), leaf[1:2])
    far = [t.detach().transpose(2, 3).contiguous().transpose(2, 3).requires_grad_(True) for t in leaf[:3]] + leaf[3:]   # copied
    o, _ = gated_delta_rule(*far)
    d, = torch.autograd.grad(o.sum(), far[2], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(o.sum() + d.square().sum(), far[0])


def test_captured_with_other_sequences(dev):
    """Offsets are read on the device: a graph of a packed batch serves other lengths, and states by other indices."""
    x = {n: t.to(dev) for n, t in _inputs(1, 1400, 1, 2, torch.bfloat16, seed=200).items()}
    one = {n: t[0].to(dev) for n, t in _inputs(1, 4, 1, 2, torch.bfloat16, seed=201).items()}
    cu = torch.tensor([0, 10, 20, 1400], device=dev)
    pool, at = torch.zeros(6, 2, D, D, device=dev), torch.tensor([0, 1, 2, -1], device=dev)

    def both():
        o, S = gated_delta_rule(*(x[n] for n in NAMES), output_final_state=True, cu_seqlens=cu)
        pool[:3] = S
        return o, gated_delta_step(*(one[n] for n in NAMES), pool, at)

    with torch.no_grad():
        both()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = both()
        for offsets, idx in (([0, 700, 700, 1300], [2, 2, 0, 1]), ([64, 65, 1399, 1400], [1, -1, 7, 1]), ([0, 10, 20, 1400], [0, 1, 2, -1])):
            cu.copy_(torch.tensor(offsets))
            at.copy_(torch.tensor(idx))
            graph.replay()
            torch.cuda.synchronize()
            states = pool.clone()
            for a, b in zip(got, both()):
                assert torch.equal(a, b)
            assert torch.equal(states, pool)


@pytest.mark.parametrize("B,T", [(2, 0), (0, 5), (0, 0)])
@pytest.mark.parametrize("packed", [False, True])
def test_gradients_of_nothing(dev, B, T, packed):
    """An empty batch in a training step: results in the graph, gradients of their leaves' shapes, a state's handed through."""
    if packed:
        B, T = 1, 0
    x = [torch.zeros(B, T, h, D, device=dev, dtype=torch.bfloat16, requires_grad=True) for h in (1, 1, 2)]
    x += [torch.zeros(B, T, 2, device=dev, requires_grad=True) for _ in range(2)]
    N = 3 if packed else B
    cu = torch.zeros(4, device=dev, dtype=torch.int32) if packed else None
    st = torch.randn(N, 2, D, D, device=dev, requires_grad=True)
    dS = torch.randn(N, 2, D, D, device=dev)
    o, S = gated_delta_rule(*x, initial_state=st, output_final_state=True, cu_seqlens=cu)
    assert o.requires_grad and o.shape == x[2].shape and torch.equal(S, st) and S.data_ptr() != st.data_ptr() or N == 0
    d = torch.autograd.grad([o, S], x + [st], [torch.zeros_like(o), dS])
    assert all(a.shape == b.shape and a.dtype == b.dtype for a, b in zip(d, x + [st])) and torch.equal(d[-1], dS)
    o, S = gated_delta_rule(*x, output_final_state=True, cu_seqlens=cu)
    assert S.shape == st.shape and not S.any()
    (o.sum() + S.sum()).backward()
    assert all(t.grad is not None and t.grad.shape == t.shape for t in x)
    o, S = gated_delta_rule(*x, initial_state=st, cu_seqlens=cu)
    assert S is None
    d = torch.autograd.grad(o.sum(), x + [st])
    assert not d[-1].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_no_gradient_of_what_has_no_effect(dev, dtype):
    """The first decay of a sequence without a state, and one that resets all that came before it, change nothing:
    what the sums of dg from there to the end hold twice has to cancel to the last bits of 64."""
    x = _inputs(1, 200, 1, 2, dtype, seed=191)
    x["g"][:, 140] = -float("inf")
    do = torch.randn(1, 200, 2, D, generator=torch.Generator().manual_seed(4)).to(dtype)
    leaf = _leaves(x, dev)
    o, _ = gated_delta_rule(*leaf)
    (dg,) = torch.autograd.grad(o, leaf[3:4], do.to(dev))
    most = dg.abs().max()
    # sums of some 64 x 64 terms in 64 bits: 2^-52 of each, of the size of the largest gradient
    assert float(dg[:, [0, 140]].abs().max() / most) <= 4096 * 2.0 ** -52


def test_forward_mode(dev):
    """A tangent raises, on the way forward and on the way back; beside one, calls without any are as ever."""
    from torch.autograd import forward_ad as fw

    x = _inputs(1, 70, 1, 1, torch.float32, seed=210)
    leaf = _leaves(x, dev)
    want = gated_delta_rule(*leaf)[0]
    w = torch.ones(D, device=dev)
    with fw.dual_level():
        v = fw.make_dual(leaf[2].detach(), torch.ones_like(leaf[2]))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                gated_delta_rule(leaf[0], leaf[1], v, *leaf[3:])
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                add_rms_norm(v, w)
        o = gated_delta_rule(*leaf)[0]
        assert torch.equal(o, want)
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(o, leaf, fw.make_dual(torch.ones_like(o), torch.ones_like(o)), retain_graph=True)
        d = torch.autograd.grad(o, leaf, torch.ones_like(o))
    for a, b in zip(d, torch.autograd.grad(want, leaf, torch.ones_like(o))):
        assert torch.equal(a, b)


def _not_finite(t):
    return ~torch.isfinite(t.float())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,T,Hk,Hv,lens", [(1, 150, 2, 2, None), (10, 150, 8, 16, None), (20, 150, 8, 16, None), (1, 1500, 1, 2, None),
                                            (1, 150, 1, 2, [5, 100, 45])])
def test_nothing_reaches_tokens_before_it(dev, B, T, Hk, Hv, lens, dtype):
    """A NaN or an infinity in any input of a token leaves the bits of all outputs before it, of other rows and, in v, of
    other columns; behind it a NaN shows wherever the recurrence has it."""
    x = {n: t.to(dev) for n, t in _inputs(B, T, Hk, Hv, dtype, seed=220).items()}
    cu = None if lens is None else torch.tensor([0] + lens, device=dev).cumsum(0)
    state = torch.randn(B if lens is None else len(lens), Hv, D, D, generator=torch.Generator().manual_seed(6)).to(dev)

    def run(y):
        return gated_delta_rule(*(y[n] for n in NAMES), initial_state=state, output_final_state=True, cu_seqlens=cu)

    want, S0 = run(x)
    b, end = (B - 1, T) if lens is None else (0, 105)             # the row, and the end of the sequence that holds the token
    seq = b if lens is None else 1
    for t in ((0, 31, 40, 63, 64, T - 1) if lens is None else (5, 36, 69, 104)):
        for name in NAMES:
            for value in (float("nan"), float("inf"), -float("inf")):
                if name == "g" and value < 0:
                    continue                                      # (a reset)
                y = dict(x)
                y[name] = x[name].clone()
                where = (b, t, 0, 77) if name in ("q", "k", "v") else (b, t, 0)
                y[name][where] = value
                o, S = run(y)
                hv = slice(0, 1) if name in ("v", "g", "beta") else slice(0, Hv // Hk)    # the v heads that it enters
                same = torch.ones_like(want, dtype=torch.bool)
                same[(b, slice(t, t + 1 if name == "q" else end), hv, 77 if name == "v" else slice(None))] = False
                case = f"{name} {value} at {t}"
                assert torch.equal(o[same], want[same]), case
                if name == "q":
                    assert torch.equal(S, S0), case
                else:
                    assert torch.equal(S[:, hv.stop:], S0[:, hv.stop:]), case
                    keep = [i for i in range(S.shape[0]) if i != seq]
                    assert torch.equal(S[keep], S0[keep]), case
                    if name == "v":
                        cols = [c for c in range(D) if c != 77]
                        assert torch.equal(S[seq][..., cols], S0[seq][..., cols]), case
                if value != value:
                    assert bool(_not_finite(o[~same]).all()), case
                    if name == "v":
                        assert bool(S[seq, 0, :, 77].isnan().all()), case
                    elif name != "q":
                        assert bool(S[seq, hv].isnan().all()), case


def test_padding_of_any_kind(dev):
    """Rows of a batch padded behind their ends with what was in memory: real tokens as without it."""
    lens = [150, 64, 1, 97, 130]
    x = _inputs(5, 150, 2, 4, torch.bfloat16, seed=221)
    real = torch.arange(150)[None] < torch.tensor(lens)[:, None]
    outs = []
    for fill in (0.0, float("nan"), float("inf")):
        y = {n: t.clone() for n, t in x.items()}
        for t in y.values():
            t[~real] = fill
        outs.append(gated_delta_rule(*(y[n].to(dev) for n in NAMES))[0].cpu()[real])
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
