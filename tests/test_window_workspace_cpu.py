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
