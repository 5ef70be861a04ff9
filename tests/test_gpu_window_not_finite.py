"""Window attention beside values that are not finite: what a query does not see leaves its output the same bits, what it sees does to
it what the definition says, and neither costs much.

The bits: a tile's scores are masked before anything else looks at them, and a value that is not finite is left out of the products
and put in afterwards, so a query that does not see it goes through the same arithmetic as with any finite value in its place.
"""

import pytest
import torch

from gsa_gdn_benchmarkstudy_amd import window_attention
from tests import test_gpu_window as tw
from tests import window_oracle as orc

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float32]
NAN, INF = float("nan"), float("inf")


def _spans(B, T, lens):
    if lens is None:
        return [(b, 0, T) for b in range(B)], None
    ends = torch.tensor([0] + lens).cumsum(0)
    return [(0, a, b) for a, b in zip(ends.tolist(), ends[1:].tolist())], ends


# blocks of 64 queries and of 128, first tokens, windows within a tile and over several, the last token of a sequence
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,T,H,Hkv,lens,W,S,at", [(2, 300, 2, 1, None, 70, 3, 150), (2, 300, 2, 1, None, 70, 3, 1), (9, 500, 8, 4, None, 33, 40, 301),
                                                   (9, 500, 8, 4, None, 1000, 0, 499), (1, 900, 4, 2, [200, 1, 0, 333, 64, 302], 90, 2, 260),
                                                   (1, 4100, 8, 8, None, 1, 1, 4099), (1, 4200, 8, 8, [4100, 100], 130, 0, 4097)])
def test_the_others_keep_their_bits(dev, B, T, H, Hkv, lens, W, S, at, dtype):
    print(f"{dtype} B={B} T={T} H={H} Hkv={Hkv} W={W} S={S} at {at}", flush=True)
    x = tw._inputs(B, T, H, Hkv, dtype, seed=T + at)
    spans, cu = _spans(B, T, lens)
    cu = None if cu is None else cu.to(dev)
    clean = tw._run(x, dev, W, S, cu=cu)["o"].cpu()
    b = B - 1
    sees = torch.zeros(B, T, dtype=torch.bool)
    for r, s, e in spans:
        if r == b and s <= at < e:
            sees[r, s:e] = orc.visible(e - s, W, S)[:, at - s]
    for name, values in (("v", (NAN, INF, -INF)), ("k", (NAN,)), ("q", (NAN, INF))):
        for i, bad in enumerate(values):
            y = {n: t.clone() for n, t in x.items()}
            y[name][b, at, 0, 5 + 40 * i:9 + 40 * i] = bad
            got = tw._run(y, dev, W, S, cu=cu)["o"].cpu()
            heads = slice(0, 1 if name == "q" else H // Hkv)                     # those that read key head 0
            hit = torch.zeros(B, T, H, 128, dtype=torch.bool)
            rows = sees if name != "q" else torch.zeros_like(sees)
            if name == "q":
                rows[b, at] = True
            hit[..., heads, slice(5 + 40 * i, 9 + 40 * i) if name == "v" else slice(None)] = rows[..., None, None]
            assert torch.equal(got[~hit], clean[~hit]), (name, bad)
            want = NAN if name != "v" else bad
            assert got[hit].isnan().all() if want != want else (got[hit] == want).all(), (name, bad)


@pytest.mark.parametrize("dtype", TYPES)
def test_infinite_keys(dev, dtype):
    """A key's infinity gives scores of +infinity (the row is NaN) or -infinity (the row does without the key), by q's sign."""
    T, W, S, at = 300, 70, 3, 150
    x = tw._inputs(1, T, 4, 1, dtype, seed=5)
    x["k"][0, at, 0, 33] = INF
    got = tw._run(x, dev, W, S)["o"].cpu()
    sees = orc.visible(T, W, S)[:, at]
    ref, size, score = tw._oracle({n: t.nan_to_num(0, 0, 0) for n, t in x.items()}, [(0, 0, T)], W, S, 128 ** -0.5, None)
    for h in range(4):
        up = sees & (x["q"][0, :, h, 33] > 0)
        assert got[0, up, h].isnan().all() and got[0, ~up, h].isfinite().all()
        tw._check(got[0, ~sees, h], ref["o"][0, ~sees, h], size["o"][0, ~sees, h], score, T, "o")
        down = sees & ~up
        see = orc.visible(T, W, S)
        see[:, at] = False
        q, k, v = x["q"][0, :, h].double(), x["k"][0, :, 0].double().nan_to_num(0, 0, 0), x["v"][0, :, 0].double()
        p = torch.softmax((q @ k.T * 128 ** -0.5).masked_fill(~see, -INF), -1)
        tw._check(got[0, down, h], (p @ v)[down], (p @ v.abs())[down], score, T, "o")


@pytest.mark.parametrize("dtype", TYPES)
def test_several_at_once(dev, dtype):
    """Infinities of both signs and NaN in one column: NaN where a query sees both signs or a NaN, else the infinity it sees."""
    T, W, S = 400, 50, 2
    x = tw._inputs(1, T, 2, 2, dtype, seed=8)
    put = {100: (7, INF), 120: (7, -INF), 140: (7, -INF), 200: (7, NAN), 210: (7, INF), 300: (9, -INF), 0: (127, INF), 399: (0, NAN)}
    for at, (d, bad) in put.items():
        x["v"][0, at, 1, d] = bad
    got = tw._run(x, dev, W, S)["o"].cpu()
    ref, _, _ = tw._oracle(x, [(0, 0, T)], W, S, 128 ** -0.5, None)
    assert torch.equal(got.isnan(), ref["o"].isnan())
    odd = ref["o"].isinf()
    assert odd.any() and torch.equal(got[odd].double(), ref["o"][odd]) and torch.equal(got.isfinite(), ref["o"].isfinite())


@pytest.mark.parametrize("name", ["q", "k", "v"])
def test_fp32_beyond_bf16s_largest_value(dev, name):
    """Finite values that round to an infinity of bf16."""
    T, W = 100, 20
    x = tw._inputs(1, T, 1, 1, torch.float32, seed=9)
    other = {"q": "k", "k": "q"}.get(name)
    scale = 128 ** -0.5 if other is None else 1e-9           # (products of 3e8 as the largest)
    x[name][0, 50, 0, 3], x[name][0, 50, 0, 4], x[name][0, 60, 0, 4] = 3.4e38, -3.4e38, 3.4028e38
    if other:
        x[other][0, :, 0, 3:5] *= 1e-30
    got = tw._run(x, dev, W, 0, scale=scale)["o"].cpu()
    tw._compare({"o": got}, x, [(0, 0, T)], W, 0, scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_time_beside_garbage(dev, dtype):
    """A padded batch with NaN behind its tokens, and a NaN that all queries see: a second walk over the tiles and one over the values, no
    more than 12 times a call without (a walk by query and key was hundreds)."""
    T, H, Hkv, W, S = 6000, 8, 2, 4096, 4
    q, k, v = (torch.randn(2, T, h, 128, device=dev).to(dtype) for h in (H, Hkv, Hkv))

    def time():
        best = INF
        for _ in range(6):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            window_attention(q, k, v, W, sinks=S)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    without = time()
    for t in (q, k, v):
        t[1, 4321:] = NAN
    padded = time()
    v[:, 0, :, 3] = NAN
    seen = time()
    print(f"{dtype} finite {1e3 * without:.0f} us, padding {1e3 * padded:.0f}, seen by all {1e3 * seen:.0f}")
    assert padded <= 12 * without and seen <= 12 * without
