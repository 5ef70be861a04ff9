"""The precision check of tests/delta_parts.py against the rule in fp32: full operands pass it, and two bf16
parts in any one of the rule's products fail it."""

import pytest
import torch

from tests import delta_parts as dp
from tests.test_gpu_delta import _oracle


@pytest.mark.parametrize("slow", [False, True])
@pytest.mark.parametrize("dtype,C", [(torch.float32, 32), (torch.bfloat16, 64)])
def test_the_check_tells_two_parts_from_three(dtype, C, slow):
    x, state, grads = dp.inputs(1, 200, 1, 2, dtype, 200, slow)
    ref = _oracle(x, [(0, 0, 200)], state, grads)

    def worst(two):
        return max(dp.units(a, b) for _, a, b in dp.fp32_results(dp.chunked(x, state, grads, C, two), ref, dtype))

    assert worst(()) <= dp.UNITS
    assert worst(dp.PRODUCTS) > 2 * dp.UNITS
    for name in dp.PRODUCTS:
        u = worst((name,))
        print(dtype, slow, name, round(u, 1))
        # (bf16: K K^T, Q K^T and P U enter what is rounded to bf16, or their operands are whole in one part)
        if dtype == torch.float32 and (slow or name not in ("KK", "KS")):
            assert u > dp.UNITS, name
