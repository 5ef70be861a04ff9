"""The fp32 results of the gated delta rule on the GPU keep fp32's precision: the measure of tests/delta_parts.py,
which two-part operands in the kernels' products fail (tests/test_delta_parts_cpu.py)."""

import pytest
import torch

from gsa_gdn_benchmarkstudy_amd import gated_delta_rule, gated_delta_step
from tests import delta_parts as dp
from tests.test_gpu_delta import _oracle, _run, _step_oracle

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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,Hk,Hv", [(1, 1, 1), (37, 2, 4)])
def test_precision_of_a_step(dev, dtype, N, Hk, Hv):
    """Two sums over 128 elements one after the other: 256 roundings."""
    x, _, _ = dp.inputs(1, N, Hk, Hv, dtype, 300 + N, False)
    x = {n: t[0] for n, t in x.items()}
    pool = torch.randn(N, Hv, dp.D, dp.D, generator=torch.Generator().manual_seed(3))
    o64, s64 = _step_oracle(x, pool, range(N))
    mine = pool.to(dev)
    o = gated_delta_step(*(x[n].to(dev) for n in dp.NAMES), mine)
    dp.check(mine, s64, "state")
    if dtype == torch.float32:
        dp.check(o, o64, "o")


def test_precision_past_32_bits(dev):
    """2**19 tokens of 16 heads: the fp32 results of the last ones are those of a call on them alone from the state
    before them, to 16 roundings on either side."""
    T, Hk, Hv, tail = (1 << 19) + 100, 8, 16, 612
    gen = torch.Generator(device=dev).manual_seed(7)

    def rn(*s):
        return torch.randn(*s, generator=gen, device=dev, dtype=torch.bfloat16)

    x = dict(q=rn(1, T, Hk, dp.D), k=rn(1, T, Hk, dp.D).mul_(dp.D ** -0.5), v=rn(1, T, Hv, dp.D))
    x.update(g=torch.full((1, T, Hv), -0.1, device=dev), beta=torch.full((1, T, Hv), 0.5, device=dev))
    do = rn(1, T, Hv, dp.D)

    def run(a, state=None):
        leaf = [x[n][:, a:].clone().requires_grad_(True) for n in dp.NAMES]
        o, S = gated_delta_rule(*leaf, initial_state=state, output_final_state=True)
        return S.detach(), *torch.autograd.grad(o, leaf, do[:, a:])[3:]

    whole = run(0)
    with torch.no_grad():
        _, S = gated_delta_rule(*(x[n][:, :T - tail] for n in dp.NAMES), output_final_state=True)
    for name, a, b in zip(("state", "dg", "dbeta"), whole, run(T - tail, S)):
        a = a if name == "state" else a[:, -tail:]
        assert dp.units(a, b.double().cpu()) <= 2 * dp.UNITS, name
