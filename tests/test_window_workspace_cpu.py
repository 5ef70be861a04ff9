"""The workspace of window attention's gradients is bounded by the tokens, not by how many sequences they are packed from."""

import pytest

from gsa_gdn_benchmarkstudy_amd import _abi


@pytest.mark.parametrize("N", [1, 600, 4096])
@pytest.mark.parametrize("W", [1, 64, 512])
def test_far_queries(N, W):
    """One key head, many query heads: what the far queries of first tokens leave.  A place for each 32 tokens at most, 1 KiB a token
    and head, and 8192 further parts of 32 KiB; near keys' parts and D beside it."""
    T, H = 65536, 64
    n = _abi.load().gsa_window_attn_workspace_bytes(1, T, N, 1, H, 1, W, 4, 1)
    assert 0 < n <= T * H * 1024 + (256 << 20) + N * 2 * 128 * 512 + T * H * 4 + 256


@pytest.mark.parametrize("dtype,size", [(0, 4), (1, 2)])
@pytest.mark.parametrize("N", [1, 100, 600, 1024, 4096])
@pytest.mark.parametrize("H,Hkv", [(16, 16), (16, 4), (64, 1)])
@pytest.mark.parametrize("T", [16384, 65536])
def test_a_small_multiple_of_the_inputs(dtype, size, N, H, Hkv, T):
    """However long the window and however many the first tokens: D, 1 KiB a token and head for near keys' parts (dk and dv in fp32) and
    for far queries' first parts, and what does not grow: 8192 further parts of 64 KiB at most, keys' parts of 512 blocks."""
    f = _abi.load().gsa_window_attn_workspace_bytes
    for W in (1, 16, 64, 512, 4096):
        for S in (0, 1, 4, 130, 1024, 1 << 20):
            n = f(1, T, N, 1, H, Hkv, W, S, dtype)
            assert 0 < n <= T * H * 4 + T * (H + Hkv) * 1024 + (8192 * 64 << 10) + (512 * 128 << 10) + 256, (W, S)


def test_many_sequences_of_short_ones():
    """16 heads, window 512, 4 first tokens: what 4096 sequences of 16 tokens take is what one of 65536 does, within q."""
    f = _abi.load().gsa_window_attn_workspace_bytes
    q = 65536 * 16 * 256
    assert f(1, 65536, 4096, 1, 16, 16, 512, 4, 1) <= f(1, 65536, 1, 1, 16, 16, 512, 4, 1) + q
    # a batch of rows: as before, one part a row
    assert f(4, 4096, 4, 0, 16, 4, 1024, 4, 1) == 16 * 16384 * 4 + 4 * 4 * 2 * 128 * 512 + (4 + 32) * 16 * 2 * 32 * 512
