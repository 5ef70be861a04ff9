"""The fp32 results of the gated delta rule on the GPU keep fp32's precision: the measure of tests/delta_parts.py,
which two-part operands in the kernels' products fail (tests/test_delta_parts_cpu.py)."""

import pytest
import torch

from tests import delta_parts as dp
from tests.test_gpu_delta import _oracle, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("slow", [False, True])
@pytest.mark.parametrize("B,T,Hk,Hv", [(2, 33, 1, 1), (1, 64, 1, 2), (2, 200, 1, 2), (1, 1100, 1, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_precision(dev, dtype, B, T, Hk, Hv, slow):
    print(f"precision {dtype} B={B} T={T} Hk={Hk} Hv={Hv} slow={slow}", flush=True)
    x, state, grads = dp.inputs(B, T, Hk, Hv, dtype, T, slow)
    ref = _oracle(x, [(b, 0, T) for b in range(B)], state, grads)
    got = _run(x, dev, state, grads=grads)
    for name, a, b in dp.fp32_results(got, ref, dtype):
        print(f"  {name} {dp.units(a, b):.1f}", flush=True)
    for name, a, b in dp.fp32_results(got, ref, dtype):
        dp.check(a, b, name)
