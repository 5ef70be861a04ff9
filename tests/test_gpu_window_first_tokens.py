"""First tokens of window attention in packed batches of many sequences, most of them too short to have far queries."""

import pytest
import torch

from gsa_gdn_benchmarkstudy_amd import window_attention
from tests import test_gpu_window as tw

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float32]


def _compare(dev, lens, H, Hkv, W, S, dtype, lead=0, trail=0):
    T = sum(lens) + lead + trail
    print(f"{dtype} {len(lens)} sequences of {min(lens)} to {max(lens)}, {T} tokens, H={H} Hkv={Hkv} W={W} S={S}", flush=True)
    x, do = tw._inputs(1, T, H, Hkv, dtype, seed=T + S), tw._grad(1, T, H, dtype, 7)
    cu = (torch.tensor([lead] + lens).cumsum(0)).tolist()
    spans = [(0, a, b) for a, b in zip(cu, cu[1:])]
    got = tw._run(x, dev, W, S, cu=torch.tensor(cu, device=dev), do=do)
    tw._compare(got, x, spans, W, S, do)
    for n, t in got.items():
        assert not t[0, :lead].any() and not t[0, T - trail:].any(), n


# a long sequence among short ones (more of them than parts of far queries), first in line, in the middle and last
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("at", [0, 311, 599])
def test_a_long_sequence_among_short_ones(dev, at, dtype):
    lens = [1 + 7 * i % 19 for i in range(599)]
    lens.insert(at, 1700)
    _compare(dev, lens, 16, 4, 100, 4, dtype)


# sequences just below and above the window and a block of keys; first tokens of one block and of several; lengths that leave
# the blocks' places side by side
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("W,S", [(1, 4), (1, 300), (60, 130), (64, 33), (129, 64), (200, 1000)])
def test_lengths_around_the_window(dev, W, S, dtype):
    lens = [W + 63, W + 64, W + 65, 1, 0, W + 127, W + 128, W + 129, W + 192, 2, W + 64, W + 64, 0, 0, W + 321, W + 64, 5, W + 700, W + 65]
    _compare(dev, lens, 2, 1, W, S, dtype, lead=3, trail=70)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_sequences_with_far_queries(dev, dtype):
    """A window of one token: nearly all queries are far ones, of sequences of a block of keys and little more."""
    _compare(dev, [66 + 3 * i % 70 for i in range(40)], 4, 4, 1, 70, dtype)


def test_far_queries_in_parts_however_many_sequences(dev):
    """The time of a long sequence's gradients does not depend on the short sequences beside it: its far queries stay in parts (walked by
    one block a head they took as long as all else together)."""
    long, short, W, S, H = 60000, [17] * 600, 64, 4, 16

    def time(lens):
        T = sum(lens)
        q, k, v = (torch.randn(1, T, h, 128, device=dev, dtype=torch.bfloat16).requires_grad_() for h in (H, 4, 4))
        cu = torch.tensor([0] + lens, device=dev).cumsum(0)
        o, best = window_attention(q, k, v, W, sinks=S, cu_seqlens=cu), float("inf")
        do = torch.randn_like(o)
        for _ in range(12):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            torch.autograd.grad(o, (q, k, v), do, retain_graph=True)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    alone, others, both = time([long]), time(short), time(short[:300] + [long] + short[300:])
    print(f"alone {1e3 * alone:.0f} us, the short ones {1e3 * others:.0f}, together {1e3 * both:.0f}")
    assert both <= 1.5 * (alone + others)
