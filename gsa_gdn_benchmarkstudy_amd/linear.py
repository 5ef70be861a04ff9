"""Linear attention with a decay for each head on MI355X: the gated delta rule's simpler sibling, with
the same states and the same pools of them.

``linear_attention`` runs whole sequences (training, prefill) and is differentiable;
``linear_attention_step`` runs one token of each sequence of a serving batch on the states
that the former leaves::

    S_t = exp(g) S_{t-1} + k_t v_t^T
    o_t = scale * S_t^T q_t                                  S [128, 128]: [k element, v element]

g is one number a head, fixed or learned.  There is no CPU or eager fallback.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.graph import increment_version as _increment_version

from . import _abi
from .delta import D_HEAD, _device, _needs_grad, _once
from .roctx import range_pop as _range_pop, range_push as _range_push


def _check(n: int, q, k, v, g) -> None:
    """The checks that both entry points share; n: dimensions before the heads."""
    qs, vs = q.shape, v.shape
    if len(qs) != n + 2 or len(vs) != n + 2 or k.shape != qs or vs[:n] != qs[:n]:
        raise ValueError(f"q {tuple(qs)}, k {tuple(k.shape)}, v {tuple(vs)}: expected [{'B, T' if n == 2 else 'N'}, heads, {D_HEAD}]")
    if qs[-1] != D_HEAD or vs[-1] != D_HEAD:
        raise ValueError(f"head dims {qs[-1]} and {vs[-1]}: the kernels take {D_HEAD}")
    Hk, Hv = qs[n], vs[n]
    if Hk < 1 or Hv < 1 or Hv % Hk:
        raise ValueError(f"{Hv} v heads are not a multiple of {Hk} q/k heads")
    if tuple(g.shape) != (Hv,):
        raise ValueError(f"g {tuple(g.shape)}: expected one log decay a v head, {(Hv,)}")
    dt = q.dtype
    if k.dtype != dt or v.dtype != dt:
        raise ValueError(f"q, k, v must share a dtype: got {dt}, {k.dtype}, {v.dtype}")
    _abi.dtype_code(dt)
    if g.dtype != torch.float32:
        raise TypeError(f"g is {g.dtype}: log decays are float32")


def _state_in(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """A state (or its gradient) as the kernels read it."""
    if t is None:
        return None
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


class _Linear(torch.autograd.Function):
    operator = "linear_attention"

    @staticmethod
    def forward(ctx, q, k, v, g, state, cu, scale, want_state):
        o, final, saved = _abi.linear_attn(q, k, v, g, state, cu, scale, want_state, True)
        ctx.set_materialize_grads(False)
        ctx.scale = scale
        ctx.save_for_backward(q, k, v, g, state, cu, saved)
        return o, final

    @_once
    def backward(ctx, do, dfinal):
        q, k, v, g, state, cu, saved = ctx.saved_tensors
        _range_push("gsa_hip/linear_attention_backward")
        try:
            do = torch.zeros_like(v, memory_format=torch.contiguous_format) if do is None else _abi._heads(do)
            grads = _abi.linear_attn_backward(q, k, v, g, state, cu, ctx.scale, saved, do, _state_in(dfinal), ctx.needs_input_grad[3],
                                              ctx.needs_input_grad[4])
        finally:
            _range_pop()
        return (*grads, None, None, None)


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, scale: Optional[float] = None,
                     initial_state: Optional[torch.Tensor] = None, output_final_state: bool = False,
                     cu_seqlens: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(o [B,T,Hv,128], final state [N,Hv,128,128] fp32 or None) of linear attention with decays.

    q, k [B,T,Hk,128] and v [B,T,Hv,128] in bf16 or fp32; v head h goes with q/k head
    h // (Hv // Hk).  g [Hv] fp32, the log of each head's decay (at most 0; below -128, down
    to -inf, nothing of earlier tokens is left).  Strided views with contiguous head rows are
    read in place.  scale: 128**-0.5 unless given.  initial_state [N,Hv,128,128] fp32: zeros
    unless given.

    cu_seqlens (int32 or int64 [N+1], on the device, ascending from 0): B is 1 and N sequences
    are packed in T, each with its own state; empty ones are allowed.  Rows of o and of the
    gradients outside every sequence are 0, whatever the inputs hold there.  A NaN or an
    infinity of a token reaches no output before it, so padding behind the tokens of a batch's row
    may hold anything (its outputs are to be ignored); elements of o that it reaches are not finite
    from its token on.  Gradients it reaches, as 0 * NaN does in the recurrence's own: where
    they are wanted, padding has to be finite, or left out by packing.

    Differentiable in q, k, v, g and initial_state, once and backwards (a tangent of
    torch.autograd.forward_ad raises); the gradients are the same bits on every run.  At most
    2**23 chunks of 64 tokens (fp32: 32) times v heads, and fewer than 2**23 sequences times v heads.

    May be captured into a graph, forward and backward, after one call outside of it; as with any
    backward pass no eager graph of the same leaves may live then (capture torch.autograd.grad, or
    use leaves of the graph's own).
    """
    _check(2, q, k, v, g)
    B, _, Hv, d = v.shape
    if cu_seqlens is not None:
        if B != 1:
            raise ValueError(f"packed sequences come in one row: B is {B}")
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2 or cu_seqlens.dtype not in (torch.int32, torch.int64):
            raise ValueError("cu_seqlens: int32 or int64 [N + 1]")
        if cu_seqlens.numel() >= 1 << 31:        # (the C interface counts in 32 bits)
            raise ValueError(f"{cu_seqlens.numel() - 1} sequences: fewer than 2**31 - 1")
        cu_seqlens = cu_seqlens.contiguous()
    N = B if cu_seqlens is None else cu_seqlens.numel() - 1
    if initial_state is not None:
        if tuple(initial_state.shape) != (N, Hv, d, d) or initial_state.dtype != torch.float32:
            raise ValueError(f"initial_state {tuple(initial_state.shape)} {initial_state.dtype}: expected fp32 {(N, Hv, d, d)}")
    scale = d ** -0.5 if scale is None else float(scale)
    with _device("linear_attention", q, k, v, g, initial_state, cu_seqlens):
        initial_state = _state_in(initial_state)
        _range_push("gsa_hip/linear_attention")
        try:
            needed = _needs_grad(q, k, v, g, initial_state)
            q, k, v = _abi._heads(q), _abi._heads(k), _abi._heads(v)
            if needed:
                return _Linear.apply(q, k, v, g, initial_state, cu_seqlens, scale, bool(output_final_state))
            o, final, _ = _abi.linear_attn(q, k, v, g, initial_state, cu_seqlens, scale, output_final_state, False)
            return o, final
        finally:
            _range_pop()


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, state: torch.Tensor,
                          state_indices: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """One token of each row of a serving batch: o [N,Hv,128]; ``state`` is updated in place.

    q, k [N,Hk,128], v [N,Hv,128] and g [Hv] as in ``linear_attention``.  state
    [slots,Hv,128,128] fp32, each matrix contiguous.  state_indices (int32 or int64 [N], on
    the device): the state of each row; row n has state n without it.  A row whose index is
    outside [0, slots) is padding: its output is 0 and no state changes.  Rows with the same
    index are consecutive tokens of one sequence, in the batch's order.  At most 65535 rows; with
    state_indices the time grows with their square from some 8000 on.

    Forward only: it raises where a gradient would be needed.
    """
    _check(1, q, k, v, g)
    N, Hv, d = v.shape
    if state.dim() != 4 or tuple(state.shape[1:]) != (Hv, d, d) or state.dtype != torch.float32:
        raise ValueError(f"state {tuple(state.shape)} {state.dtype}: expected fp32 [slots, {Hv}, {d}, {d}]")
    s0, s1, s2, s3 = state.stride()
    if s2 != d or s3 != 1 or (s0 | s1) % 4 or state.data_ptr() % 16:
        raise ValueError("state is updated in place: its matrices must be contiguous and 16-byte aligned")
    extent = d * d
    for stride, n in sorted(((s0, state.shape[0]), (s1, Hv))):
        if n > 1:
            if stride < extent:
                raise ValueError("state is updated in place: its matrices overlap")
            extent += (n - 1) * stride
    if state_indices is not None:
        if tuple(state_indices.shape) != (N,) or state_indices.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"state_indices: int32 or int64 [{N}]")
        state_indices = state_indices.contiguous()
    elif N > state.shape[0]:
        raise ValueError(f"{N} rows, {state.shape[0]} states")
    if _needs_grad(q, k, v, g, state):
        raise RuntimeError("linear_attention_step is forward only: call it under torch.no_grad()")
    with _device("linear_attention_step", q, k, v, g, state, state_indices):
        if N == 0 or state.shape[0] == 0:
            return v.new_zeros(v.shape)
        _range_push("gsa_hip/linear_step")
        try:
            o = _abi.linear_step(q, k, v, g, state, state_indices, d ** -0.5 if scale is None else float(scale))
            if not state.is_inference():
                _increment_version(state)        # a graph that kept the old state must not use the new one
            return o
        finally:
            _range_pop()
