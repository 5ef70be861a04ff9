"""What a write does to the caches' versions."""

import pytest
import torch

from gsa_gdn_benchmarkstudy_amd.window import _written


@pytest.mark.parametrize("inference", [(), (0,), (1,), (0, 1)])
def test_versions_of_written_caches(inference):
    """A graph that kept a cache notices the write, whatever the other one is."""
    caches = [torch.zeros(2) for _ in range(2)]
    for i in inference:
        with torch.inference_mode():
            caches[i] = torch.zeros(2)
    _written(*caches)
    assert [t._version for t in caches if not t.is_inference()] == [1] * (2 - len(inference))
