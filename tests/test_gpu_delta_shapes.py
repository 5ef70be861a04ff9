"""Every way in which the gated delta rule goes from chunk to chunk, forward and backward with states: the size
rule is asked which one a call takes, some heads are compared with the recurrence in 64 bits, and all
of them with calls of one sequence each, which go another way (few heads: the same way).

Tolerance between two calls: each rounds to its type once (eps / 2 of the value each); fp32 results
keep to 16 roundings of 2**-24 in the root mean square (tests/delta_parts.py), and the largest of some
2**20 errors to four times that, on both sides: 128 of the largest value; bf16 results have operands of
two parts under them, 2**-17 in a term, likewise 4 times on both sides: 2**-14 of the largest value.
"""

import pytest
import torch

from gsa_gdn_benchmarkstudy_amd import _abi
from tests import delta_parts as dp
from tests.test_gpu_delta import NAMES, _compare, _oracle, _run

pytestmark = pytest.mark.gpu

D = 128
HALF, ALONE, TWO, SEGMENTS = 1, 2, 3, 4
BF16, F32 = torch.bfloat16, torch.float32


def _shape(B, T, N, packed, Hk, Hv, dtype):
    return _abi.load().gsa_delta_rule_shape(B, T, N, int(packed), Hk, Hv, _abi.dtype_code(dtype))


def _same(a, b, name):
    step = 2.0 ** -14 if a.dtype == BF16 else 128 * 2.0 ** -24
    err = (a.double() - b.double()).abs()
    tol = torch.finfo(a.dtype).eps * b.double().abs() + step * b.double().abs().max()
    assert bool((err <= tol).all()), f"{name}: {(err / tol).max():.2f} of the tolerance"


def _all_ways(dev, B, T, Hk, Hv, dtype, shape, lens=None, samples=()):
    """samples: (sequence, q/k head) to be compared with the oracle."""
    N = B if lens is None else len(lens)
    print(f"shape {shape} {dtype} B={B} T={T} N={N} Hk={Hk} Hv={Hv}", flush=True)
    assert _shape(B, T, N, lens is not None, Hk, Hv, dtype) == shape
    x, state, grads = dp.inputs(B, T, Hk, Hv, dtype, 7, False)
    if lens is not None:
        gen = torch.Generator().manual_seed(8)
        state, dS = torch.randn(N, Hv, D, D, generator=gen), torch.randn(N, Hv, D, D, generator=gen)
        grads = (grads[0], dS)
    cu = None if lens is None else torch.tensor([0] + lens).cumsum(0)
    spans = [(b, 0, T) for b in range(B)] if lens is None else [(0, int(cu[i]), int(cu[i + 1])) for i in range(N)]
    got = _run(x, dev, state, cu=None if cu is None else cu.to(dev), grads=grads)
    again = _run(x, dev, state, cu=None if cu is None else cu.to(dev), grads=grads)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1]) and all(torch.equal(got[2][n], again[2][n]) for n in got[2])

    def part(n, hk, hv):
        """The call's results of sequence n and some heads, and its inputs."""
        b, s, e = spans[n]
        pick = {m: (hk if m in "qk" else hv) for m in NAMES}
        one = {m: t[b:b + 1, s:e, pick[m]] for m, t in x.items()}
        res = (got[0][b:b + 1, s:e, hv], got[1][n:n + 1, hv],
               {m: got[2][m][b:b + 1, s:e, pick[m]] for m in NAMES} | {"state": got[2]["state"][n:n + 1, hv]})
        return one, state[n:n + 1, hv], (grads[0][b:b + 1, s:e, hv], grads[1][n:n + 1, hv]), res

    share = Hv // Hk
    for n, h in samples:
        one, st, gr, res = part(n, slice(h, h + 1), slice(h * share, (h + 1) * share))
        L = one["q"].shape[1]
        ref = _oracle(one, [(0, 0, L)], st, gr)
        _compare(res, ref, L, share)
        for name, a, b in dp.fp32_results(res, ref, dtype):
            if L > 1:
                dp.check(a, b, f"{name} of sequence {n}, head {h}")
    for n in range(N):
        one, st, gr, res = part(n, slice(None), slice(None))
        L = one["q"].shape[1]
        if L == 0:
            assert torch.equal(res[1].cpu(), st) and torch.equal(res[2]["state"].cpu(), gr[1])
            continue
        assert _shape(1, L, 1, False, Hk, Hv, dtype) != shape or shape in (HALF, SEGMENTS + ALONE)
        alone = _run(one, dev, st, grads=gr)
        _same(res[0], alone[0], f"o of sequence {n}")
        _same(res[1], alone[1], f"state of sequence {n}")
        for m, t in alone[2].items():
            _same(res[2][m], t, f"d{m} of sequence {n}")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,T,Hk,Hv,shape", [(10, 200, 16, 16, ALONE), (20, 200, 8, 16, TWO), (17, 321, 16, 16, TWO), (33, 64, 16, 16, TWO),
                                             (40, 129, 4, 8, TWO)])
def test_batch_in_one_piece(dev, B, T, Hk, Hv, shape, dtype):
    _all_ways(dev, B, T, Hk, Hv, dtype, shape, samples=[(0, 0), (B // 2, Hk - 1), (B - 1, Hk // 2)])


RAGGED = [1, 0, 333, 64, 65, 17, 128, 2, 191, 130, 63, 0, 257, 96, 5, 500, 33, 127]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens,shape", [(RAGGED, HALF), (RAGGED * 3, ALONE), ([100] * 50, ALONE)])
def test_packed_in_one_piece(dev, lens, shape, dtype):
    _all_ways(dev, 1, sum(lens), 8, 16, dtype, shape, lens, samples=[(2, 0), (15, 3), (len(lens) - 1, 7)])


@pytest.mark.parametrize("dtype,lens,Hk,Hv,shape", [
    (BF16, [900, 0, 1, 2500, 1100], 1, 2, SEGMENTS + ALONE), (F32, [450, 0, 1, 1250, 549], 1, 2, SEGMENTS + ALONE),
    (BF16, [3000, 1, 0, 4400], 8, 16, SEGMENTS + TWO), (F32, [1500, 1, 0, 2200], 8, 16, SEGMENTS + TWO)])
def test_packed_segments(dev, dtype, lens, Hk, Hv, shape):
    _all_ways(dev, 1, sum(lens), Hk, Hv, dtype, shape, lens, samples=[(0, 0), (2 if lens[2] else 1, Hk - 1), (len(lens) - 1, Hk // 2)])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_batch_by_segments(dev, dtype):
    """A batch whose segments are as many as a chip has CUs."""
    T = 2048 if dtype == BF16 else 1024
    _all_ways(dev, 4, T + 5, 16, 16, dtype, SEGMENTS + ALONE, samples=[(0, 0), (3, 15)])
