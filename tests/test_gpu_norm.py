"""add_rms_norm and add_rms_norm_fp8 on the GPU against the formula in 64 bits.

Tolerances: a result of type t carries one rounding, at most eps(t) / 2 of its value; under it
lie fp32 sums over D elements of a row, held by ROUNDS = 8 + log2(D) roundings of 2^-24 (a
lane's sum of at most 32 squares and the tree over lanes; rsqrt, two products), relative to the
row's largest result; sums over rows (dw) add one rounding a row in a block of rows and a tree
over blocks: rows / 1024 + 64 more, of the sum of the terms' magnitudes.
"""

import math

import pytest
import torch

from gsa_gdn_benchmarkstudy_amd import add_rms_norm, add_rms_norm_fp8
from tests import delta_oracle as orc

pytestmark = pytest.mark.gpu

EPS = 1e-6
WIDTHS = [1, 7, 8, 100, 128, 129, 136, 512, 520, 1000, 1024, 1032, 2048, 2056, 4096, 5000, 8192, 8200, 32760, 32768]


def _make(shape, dtype, residual, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=gen).to(dtype)
    res = (2 * torch.randn(*shape, generator=gen)).to(dtype) if residual else None
    w = (1 + 0.2 * torch.randn(shape[-1], generator=gen)).to(dtype)
    return x, res, w


def _tol(ref, dtype, D, largest=None):
    big = ref.abs().amax(-1, keepdim=True) if largest is None else largest
    return torch.finfo(dtype).eps / 2 * ref.abs() + (8 + math.log2(max(D, 2))) * 2.0 ** -24 * big


def _near(got, ref, tol, name):
    err = (got.double().cpu() - ref).abs()
    assert tuple(got.shape) == tuple(ref.shape) and bool((err <= tol).all()), f"{name}: {(err / tol).max():.2f} of the tolerance"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("rows", [1, 5, 70])
def test_norm(dev, rows, D, residual, dtype):
    print(f"norm {dtype} rows={rows} D={D} residual={residual}", flush=True)
    x, res, w = _make((rows, D), dtype, residual, D)
    gen = torch.Generator().manual_seed(1)
    dy, dh = (torch.randn(rows, D, generator=gen).to(dtype) for _ in range(2))
    ins = [t.to(dev).requires_grad_(True) for t in (x, w, res) if t is not None]
    y, h = add_rms_norm(ins[0], ins[1], residual=ins[2] if residual else None, eps=EPS)
    i64 = [t.double().requires_grad_(True) for t in (x, w, res) if t is not None]
    y64, h64 = orc.norm(i64[0], i64[1], i64[2] if residual else None, EPS, dtype)
    assert torch.equal(h.cpu(), x if res is None else x + res)
    _near(y, y64.detach(), _tol(y64.detach(), dtype, D), "y")
    outs, gr = ([y, h], [dy.to(dev), dh.to(dev)]) if residual else ([y], [dy.to(dev)])
    d = torch.autograd.grad(outs, ins, gr)
    d64 = torch.autograd.grad([y64, h64] if residual else [y64], i64, [dy.double(), dh.double()] if residual else [dy.double()])
    # dx: the terms' magnitudes, not their difference, carry the roundings
    n64 = (y64 / i64[1]).detach()
    r = ((h64.square().mean(-1, keepdim=True) + EPS) ** -0.5).detach()
    terms = r * (2 * (dy.double() * w.double()).abs().amax(-1, keepdim=True) * (1 + n64.abs().amax(-1, keepdim=True) ** 2))
    _near(d[0], d64[0], _tol(d64[0], dtype, D, terms), "dx")
    sums = (dy.double() * n64).abs().sum(0)
    _near(d[1], d64[1], torch.finfo(dtype).eps / 2 * d64[1].abs() + (72 + math.log2(max(D, 2)) + rows / 1024) * 2.0 ** -24 * sums, "dw")
    if residual:
        assert torch.equal(d[2], d[0])
    with torch.no_grad():
        y2, h2 = add_rms_norm(ins[0], ins[1], residual=ins[2] if residual else None, eps=EPS)
    assert torch.equal(y, y2) and torch.equal(h, h2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("D", WIDTHS)
def test_norm_fp8(dev, D, residual, dtype):
    """scale is the row's largest / 448; each value within half a step of e4m3 (2^-4 of it; 2^-10 below 2^-6),
    and what the fp32 value under it is off."""
    rows = 9
    x, res, w = _make((rows, D), dtype, residual, D + 1)
    x[3] = 0
    if residual:
        res[3] = 0                               # a row of zeros: scale 1
    y, scale, h = add_rms_norm_fp8(x.to(dev), w.to(dev), residual=None if res is None else res.to(dev), eps=EPS)
    y64, _ = orc.norm(x.double(), w.double(), None if res is None else res.double(), EPS, dtype)
    assert y.dtype == torch.float8_e4m3fn and torch.equal(h.cpu(), x if res is None else x + res)
    s64 = y64.abs().amax(-1) / 448
    s64[3] = 1
    _near(scale, s64, (10 + math.log2(max(D, 2))) * 2.0 ** -24 * s64, "scale")
    q64 = y64 / s64[:, None]
    tol = (2.0 ** -4 * q64.abs()).clamp_min(2.0 ** -10) + 64 * 2.0 ** -24 * 448
    _near(y.float(), q64, tol, "y")
    assert not y[3].float().any() and scale[3] == 1


def test_many_rows(dev):
    """More rows than blocks: every row's share of dw is in, and every run gives the same bits."""
    for rows, D in [(5003, 128), (3001, 2048), (1500, 5000)]:
        x, res, w = _make((rows, D), torch.bfloat16, True, rows)
        dy = torch.randn(rows, D, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
        ins = [t.to(dev).requires_grad_(True) for t in (x, w, res)]
        y, _ = add_rms_norm(ins[0], ins[1], residual=ins[2], eps=EPS)
        d = torch.autograd.grad(y, ins, dy.to(dev), retain_graph=True)
        again = torch.autograd.grad(y, ins, dy.to(dev))
        assert all(torch.equal(a, b) for a, b in zip(d, again))
        _, h64 = orc.norm(x.double(), w.double(), res.double(), EPS, torch.bfloat16)
        n64 = h64 * (h64.square().mean(-1, keepdim=True) + EPS) ** -0.5
        ref, sums = (dy.double() * n64).sum(0), (dy.double() * n64).abs().sum(0)
        _near(d[1], ref, 2.0 ** -8 * ref.abs() + (90 + rows / 1024) * 2.0 ** -24 * sums, "dw")


def test_strided_rows(dev):
    """Heads of a projection, rows of a wider tensor, transposed and misaligned ones: the same bits as copies."""
    gen = torch.Generator().manual_seed(4)
    big = torch.randn(2, 50, 3, 4, 128, generator=gen).to(torch.bfloat16).to(dev)
    w = torch.randn(128, generator=gen).to(torch.bfloat16).to(dev)
    for t in (big[:, :, 1], big[:1, :, 2], big[0, :, 0, 1], big[:, :, 0].transpose(1, 2), big[0, 0, 0].t()[:, :3].t(),
              big.reshape(-1)[1:1 + 128 * 70].view(70, 128), big[:, ::2, 0, 0]):
        res = torch.randn(t.shape, generator=gen).to(torch.bfloat16).to(dev)
        dy = torch.randn(t.shape, generator=gen).to(torch.bfloat16).to(dev)
        for r in (None, res):
            a = t.detach().requires_grad_(True)
            b = t.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True)
            ya, yb = add_rms_norm(a, w, residual=r)[0], add_rms_norm(b, w, residual=r)[0]
            assert ya.is_contiguous() and torch.equal(ya, yb)
            assert torch.equal(torch.autograd.grad(ya, a, dy)[0], torch.autograd.grad(yb, b, dy)[0])
            qa, qb = (add_rms_norm_fp8(z.detach(), w, residual=r) for z in (a, b))
            assert torch.equal(qa[0].view(torch.uint8), qb[0].view(torch.uint8)) and torch.equal(qa[1], qb[1])
    x = torch.randn(6, 128, generator=gen).to(dev).requires_grad_(True)
    wf = w.float().requires_grad_(True)
    (d,) = torch.autograd.grad(add_rms_norm(x, wf)[0].sum(), x)                 # an expanded gradient
    (e,) = torch.autograd.grad(add_rms_norm(x, wf)[0], x, torch.ones(6, 128, device=dev))
    assert torch.equal(d, e)


def test_rows_keep_to_themselves(dev):
    """NaN and infinities stay in their rows, and show there."""
    x, res, w = _make((6, 300), torch.float32, True, 9)
    ref = add_rms_norm(x.to(dev), w.to(dev), residual=res.to(dev))[0]
    x[1, 5], x[4, 7] = float("nan"), float("inf")
    y, _ = add_rms_norm(x.to(dev), w.to(dev), residual=res.to(dev))
    q, scale, _ = add_rms_norm_fp8(x.to(dev), w.to(dev), residual=res.to(dev))
    keep = [0, 2, 3, 5]
    assert torch.equal(y[keep], ref[keep]) and y[1].isnan().all() and y[4, 7].isnan() and scale[1].isnan() and scale[4].isnan()
    assert q[1].float().isnan().all() and not scale[keep].isnan().any()


def test_only_h_used(dev):
    x, res, w = (t.to(dev).requires_grad_(True) for t in _make((4, 64), torch.float32, True, 10))
    _, h = add_rms_norm(x, w, residual=res)
    dx, dw, dr = torch.autograd.grad(h.sum(), [x, w, res])
    assert torch.equal(dx, torch.ones_like(x)) and torch.equal(dr, dx) and not dw.any()


def test_captured(dev):
    """Forward and backward in a graph, replayed on new inputs."""
    x, res, w = (t.to(dev) for t in _make((300, 512), torch.bfloat16, True, 11))
    dy = torch.randn(300, 512, device=dev, dtype=torch.bfloat16)
    leaf = [t.detach().requires_grad_(True) for t in (x, w, res)]

    def both():
        y, h = add_rms_norm(leaf[0], leaf[1], residual=leaf[2])
        return (y, h) + torch.autograd.grad(y, leaf, dy)

    s = torch.cuda.Stream(device=dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        both()
    torch.cuda.current_stream(dev).wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for i in range(4):
        with torch.no_grad():
            leaf[0].copy_(torch.randn(300, 512, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        y, h = add_rms_norm(leaf[0].detach(), w, residual=res)
        d = [t.detach().requires_grad_(True) for t in leaf]
        y, h = add_rms_norm(d[0], d[1], residual=d[2])
        for a, b in zip(got, (y, h) + torch.autograd.grad(y, d, dy)):
            assert torch.equal(a, b)


def test_no_rows(dev):
    x, w = torch.zeros(3, 0, 64, device=dev), torch.ones(64, device=dev)
    y, h = add_rms_norm(x, w, residual=x)
    assert y.shape == h.shape == x.shape
    y, scale, h = add_rms_norm_fp8(x, w)
    assert y.shape == x.shape and scale.shape == (3, 0) and y.dtype == torch.float8_e4m3fn


def test_gradients_that_are_broadcast(dev):
    """Gradients with strides of 0 (of a sum, of a mean over rows), and of a norm of a transposed x."""
    x, _, w = _make((4, 6, 96), torch.float32, False, 21)
    grads = []
    for at in (dev, "cpu"):
        a, b = x.to(at).requires_grad_(True), w.to(at).requires_grad_(True)
        at_t = a.transpose(0, 1)
        y = add_rms_norm(at_t, b, eps=EPS)[0] if at == dev else torch.nn.functional.rms_norm(at_t.double(), (96,), b.double(), EPS)
        grads.append(torch.autograd.grad(y.sum() + y.mean(0).sum(), (a, b)))
    for got, ref in zip(*grads):
        # rows of 96 and 24 rows: sums of 96 and 24 fp32 terms, a few roundings each; ref itself rounds once to fp32
        assert bool(((got.cpu() - ref).abs() <= (96 + 24 + 16) * 2.0 ** -24 * max(1.0, float(ref.abs().max()))).all())


def test_two_streams(dev):
    """Forward and backward on two streams at once, after the work that makes their inputs."""
    x, res, w = (t.to(dev) for t in _make((6000, 1024), torch.bfloat16, True, 31))

    def train():
        leaf = [t.detach().clone().requires_grad_(True) for t in (x, w, res)]
        y, h = add_rms_norm(leaf[0], leaf[1], residual=leaf[2])
        return (y, h) + torch.autograd.grad([y, h], leaf, [x, res])

    want, got, streams = train(), [], [torch.cuda.Stream(device=dev) for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(s):
            got.append(train())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_differentiable_once(dev):
    x, w = torch.randn(4, 64, device=dev, requires_grad=True), torch.ones(64, device=dev, requires_grad=True)
    d, = torch.autograd.grad(add_rms_norm(x, w)[0].sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad((d * d).sum(), w)


@pytest.mark.parametrize("D,rows,fp8", [(8, (1 << 28) + 5, False), (136, (1 << 26) + 3, True), (1032, (1 << 24) + 1, True),
                                        (8200, (1 << 22) + 1, True)])
def test_more_rows_than_one_launch_dimension_holds(dev, D, rows, fp8):
    """2**32 threads in one direction and more: every row is there, and nothing behind the last.  (All rows
    are one: read with a stride of 0.)"""
    print(f"rows {rows} of {D}", flush=True)
    x, _, w = _make((3, D), torch.bfloat16, False, D)
    x, w = x.to(dev), w.to(dev)
    many = x[1:2].expand(rows, D)
    if fp8:
        y, scale, _ = add_rms_norm_fp8(many, w, eps=EPS)
        y1, s1, _ = add_rms_norm_fp8(x[1:2], w, eps=EPS)
        assert bool((scale == s1[0]).all())
        y, y1 = y.view(torch.uint8), y1.view(torch.uint8)
    else:
        y, y1 = add_rms_norm(many, w, eps=EPS)[0], add_rms_norm(x[1:2], w, eps=EPS)[0]
    for a in range(0, rows, 1 << 22):
        assert bool((y[a:a + (1 << 22)] == y1).all()), a


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [128, 1000, 2048, 4096, 8200])
def test_fp8_is_the_quotient(dev, D, dtype):
    """y in 8 bits is the fp32 row divided by its scale and rounded, ties to even: bit for bit, ties among them
    (quotients of bf16 products often lie between two values of e4m3)."""
    x, _, w = _make((1000, D), dtype, False, D + 2)
    x[7], x[8] = x[7] * 2.0 ** -100, 0
    x, w = x.to(dev), w.to(dev)
    w[3] = 2.0 ** 100 if D == 1000 else 1.0      # (a row's largest far above the others)
    y, scale, _ = add_rms_norm_fp8(x, w, eps=EPS)
    whole, _ = add_rms_norm(x.float(), w.float(), eps=EPS)
    # on the CPU and by tensors: torch divides by a number as a product with its reciprocal
    y, scale, whole = y.cpu(), scale.cpu(), whole.cpu()
    big = whole.abs().amax(-1)
    assert bool((scale == torch.where(big == 0, 1.0, big / torch.full_like(big, 448.0))).all())
    want = (whole / scale[:, None].expand_as(whole)).clamp(-448, 448).to(torch.float8_e4m3fn)
    same = y.view(torch.uint8) == want.view(torch.uint8)
    assert bool(same.all()), f"{int((~same).sum())} of {same.numel()} differ"


def test_fp8_of_an_infinite_row(dev):
    """A weight that makes one value infinite: scale infinite, that value NaN, the others 0, as a division gives."""
    x = torch.randn(4, 256, generator=torch.Generator().manual_seed(5)).to(dev)
    w = torch.ones(256, device=dev)
    x[:, 9], w[9] = 8.0, 3e38
    y, scale, _ = add_rms_norm_fp8(x, w, eps=EPS)
    rest = [i for i in range(256) if i != 9]
    assert bool(scale.isinf().all()) and bool(y.float()[:, 9].isnan().all()) and not y.float()[:, rest].any()
