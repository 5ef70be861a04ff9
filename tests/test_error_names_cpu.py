"""What an operator refuses in torch's name names the operator: these errors come out of tracebacks that pass through autograd."""

import pytest
import torch
from torch.autograd import forward_ad as fw

from gsa_gdn_benchmarkstudy_amd import (
    add_rms_norm, add_rms_norm_fp8, gated_delta_rule, gated_delta_step, linear_attention, linear_attention_step, window_attention,
    window_attention_step, window_cache_write,
)
from gsa_gdn_benchmarkstudy_amd.delta import _once

D = 128


def _z(*s):
    return torch.zeros(*s)


def _calls():
    seq, tok, gates, cache = (_z(1, 3, 1, D),) * 3, (_z(2, 1, D),) * 3, (_z(1, 3, 1),) * 2, (_z(2, 8, 1, D), _z(2, 8, 1, D))
    at = torch.zeros(2, dtype=torch.int64)
    return {
        add_rms_norm: (lambda x: add_rms_norm(x, _z(8)), _z(2, 8)),
        add_rms_norm_fp8: (lambda x: add_rms_norm_fp8(x, _z(8)), _z(2, 8)),
        gated_delta_rule: (lambda q: gated_delta_rule(q, *seq[1:], *gates), seq[0]),
        gated_delta_step: (lambda q: gated_delta_step(q, *tok[1:], _z(2, 1), _z(2, 1), _z(2, 1, D, D)), tok[0]),
        linear_attention: (lambda q: linear_attention(q, *seq[1:], _z(1)), seq[0]),
        linear_attention_step: (lambda q: linear_attention_step(q, *tok[1:], _z(1), _z(2, 1, D, D)), tok[0]),
        window_attention: (lambda q: window_attention(q, *seq[1:], 2), seq[0]),
        window_cache_write: (lambda k: window_cache_write(k, _z(2, 3, 1, D), *cache), _z(2, 3, 1, D)),
        window_attention_step: (lambda q: window_attention_step(q, *tok[1:], *cache, at, 4), tok[0]),
    }


@pytest.mark.parametrize("op", list(_calls()), ids=lambda f: f.__name__)
def test_forward_mode_and_trace(op):
    call, x = _calls()[op]
    with torch.no_grad(), fw.dual_level():
        with pytest.raises(RuntimeError, match=f"^{op.__name__} has no forward-mode"):
            call(fw.make_dual(x, torch.ones_like(x)))
    with torch.no_grad(), pytest.raises(RuntimeError, match=f"^{op.__name__} cannot be recorded by torch.jit.trace"):
        torch.jit.trace(call, (x,), check_trace=False)


def test_second_derivative():
    class Twice(torch.autograd.Function):
        operator = "some_operator"

        @staticmethod
        def forward(ctx, x):
            ctx.save_for_backward(x)
            return 2 * x

        @_once
        def backward(ctx, g):
            return 2 * g,

    x = torch.ones(3, requires_grad=True)
    d, = torch.autograd.grad(Twice.apply(x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="the gradients of some_operator cannot be differentiated"):
        d.sum().backward()
