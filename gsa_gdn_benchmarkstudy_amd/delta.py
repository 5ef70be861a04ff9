"""The gated delta rule on MI355X: the linear-attention mixer of the study's second half.

``gated_delta_rule`` runs whole sequences (training, prefill) and is differentiable;
``gated_delta_step`` runs one token of each sequence of a serving batch on the states that
the former leaves.  The recurrence is the one of the reference's
``recurrent_gated_delta_rule_ref`` (benchmark_models.ipynb:187)::

    S_t = exp(g_t) S_{t-1} + k_t beta_t (v_t - exp(g_t) S_{t-1}^T k_t)^T
    o_t = scale * S_t^T q_t                                  S [128, 128]: [k element, v element]

q and k are taken as they are: normalise them before (``add_rms_norm`` with a weight of
d**-0.5 gives them unit length).  There is no CPU or eager fallback.
"""

from __future__ import annotations

import contextlib
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad as _forward_ad
from torch.autograd.graph import increment_version as _increment_version

from . import _abi
from .roctx import range_pop as _range_pop, range_push as _range_push

D_HEAD = 128


def _check(n: int, q, k, v, g, beta) -> None:
    """The checks that both entry points share; n: dimensions before the heads."""
    qs, vs = q.shape, v.shape
    if len(qs) != n + 2 or len(vs) != n + 2 or k.shape != qs or vs[:n] != qs[:n]:
        raise ValueError(f"q {tuple(qs)}, k {tuple(k.shape)}, v {tuple(vs)}: expected [{'B, T' if n == 2 else 'N'}, heads, {D_HEAD}]")
    if qs[-1] != D_HEAD or vs[-1] != D_HEAD:
        raise ValueError(f"head dims {qs[-1]} and {vs[-1]}: the kernels take {D_HEAD}")
    Hk, Hv = qs[n], vs[n]
    if Hk < 1 or Hv < 1 or Hv % Hk:
        raise ValueError(f"{Hv} v heads are not a multiple of {Hk} q/k heads")
    if g.shape != vs[:-1] or beta.shape != vs[:-1]:
        raise ValueError(f"g {tuple(g.shape)}, beta {tuple(beta.shape)}: expected {tuple(vs[:-1])}")
    dt = q.dtype
    if k.dtype != dt or v.dtype != dt:
        raise ValueError(f"q, k, v must share a dtype: got {dt}, {k.dtype}, {v.dtype}")
    _abi.dtype_code(dt)
    if g.dtype != torch.float32:
        raise TypeError(f"g is {g.dtype}: log decays are float32")
    if beta.dtype != torch.float32 and beta.dtype != dt:
        raise TypeError(f"beta is {beta.dtype}: expected float32 or {dt}")


_HERE = contextlib.nullcontext()


def _refuse_unseen(name: str, *ts: Optional[torch.Tensor]) -> None:
    """Raises where torch follows the call in a way that a kernel's launch escapes, and that would
    lose it in silence: a tangent of forward-mode differentiation, or torch.jit.trace."""
    if _forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled():
        for t in ts:
            if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{name} has no forward-mode derivative (torch.autograd.forward_ad)")
    if torch._C._get_tracing_state() is not None:
        raise RuntimeError(f"{name} cannot be recorded by torch.jit.trace")


def _device(name: str, first: torch.Tensor, *others: Optional[torch.Tensor]):
    """Checks that torch need not see into the call and that all tensors are on one GPU, and makes
    that the current one."""
    _refuse_unseen(name, first, *others)
    at = first.get_device()                      # -1 on the CPU
    for t in others:
        if t is not None and t.get_device() != at:
            _abi._need_cuda(first, *others)
            _abi._on(first.device, *others)
    if at < 0:
        _abi._need_cuda(first)
    return _HERE if torch.cuda.current_device() == at else torch.cuda.device(at)


def _needs_grad(*ts: Optional[torch.Tensor]) -> bool:
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


class _Twice(torch.autograd.Function):
    """The first n tensors as they are, depending on all of them, with an error for their gradient."""

    @staticmethod
    def forward(ctx, name, n, *ts):
        ctx.name = name
        return tuple(t if t is None else t.view_as(t) for t in ts[:n])

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"the gradients of {ctx.name} cannot be differentiated: it is differentiable once")


def _once(backward):
    """A backward pass that is differentiable once: where a graph of it is being built, what comes out
    depends on the gradients that came in and on the inputs, with an error behind it.  (torch's
    once_differentiable costs 15 us a call, and its outputs do not depend on the inputs: a
    penalty on the gradients would lose its part in silence.)  Errors name the Function's `operator`."""

    def run(ctx, *grads):
        name = getattr(getattr(ctx, "_forward_cls", None), "operator", "this operator")
        _refuse_unseen(name, *grads)
        if not torch.is_grad_enabled():
            return backward(ctx, *grads)
        with torch.no_grad():
            out = backward(ctx, *grads)
        return _Twice.apply(name, len(out), *out, *grads, *ctx.saved_tensors)

    return staticmethod(run)


class _Rule(torch.autograd.Function):
    operator = "gated_delta_rule"

    @staticmethod
    def forward(ctx, q, k, v, g, beta, state, cu, scale, want_state):
        o, final, saved = _abi.delta_rule(q, k, v, g, beta, state, cu, scale, want_state, True)
        ctx.set_materialize_grads(False)
        ctx.scale, ctx.has_state = scale, state is not None
        ctx.save_for_backward(q, k, v, g, beta, cu, saved)
        return o, final

    @_once
    def backward(ctx, do, dfinal):
        q, k, v, g, beta, cu, saved = ctx.saved_tensors
        _range_push("gsa_hip/delta_rule_backward")
        try:
            do = torch.zeros_like(v, memory_format=torch.contiguous_format) if do is None else _abi._heads(do)
            if dfinal is not None:
                dfinal = dfinal.contiguous()
                if dfinal.data_ptr() % 16:
                    dfinal = dfinal.clone()
            grads = _abi.delta_rule_backward(q, k, v, g, beta, cu, ctx.scale, saved, do, dfinal, ctx.has_state)
        finally:
            _range_pop()
        return (*grads, None, None, None)


def gated_delta_rule(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                     scale: Optional[float] = None, initial_state: Optional[torch.Tensor] = None,
                     output_final_state: bool = False,
                     cu_seqlens: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(o [B,T,Hv,128], final state [N,Hv,128,128] fp32 or None) of the gated delta rule.

    q, k [B,T,Hk,128] and v [B,T,Hv,128] in bf16 or fp32; v head h goes with q/k head
    h // (Hv // Hk).  g [B,T,Hv] fp32, the log of the decay (at most 0; below -128, down to
    -inf, it is a reset); beta [B,T,Hv] in fp32 or q's dtype.  Strided views with contiguous
    head rows are read in place.  scale: 128**-0.5 unless given.  initial_state
    [N,Hv,128,128] fp32: zeros unless given.

    cu_seqlens (int32 or int64 [N+1], on the device, ascending from 0): B is 1 and N sequences
    are packed in T, each with its own state; empty ones are allowed.  Rows of o and of the
    gradients outside every sequence are 0, whatever the inputs hold there.  A NaN or an
    infinity of a token reaches no output before it, so padding behind the tokens of a batch's row
    may hold anything (its outputs are to be ignored).  Gradients it reaches, as 0 * NaN does in
    the recurrence's own: where they are wanted, padding has to be finite, or left out by packing.

    Differentiable in q, k, v, g, beta and initial_state, once and backwards (a tangent of
    torch.autograd.forward_ad raises); the gradients are the same bits on every run.  A forward
    that needs gradients keeps 1.5 KiB (bf16; fp32: 2.5 KiB) a token and v head, and where it
    works by segments up to 0.25 KiB (0.5 KiB) more.  At most 2**23 chunks times v heads, and
    fewer than 2**23 sequences times v heads.

    May be captured into a graph, forward and backward, after one call outside of it; as with any
    backward pass no eager graph of the same leaves may live then (capture torch.autograd.grad, or
    use leaves of the graph's own).
    """
    _check(2, q, k, v, g, beta)
    B, _, Hv, d = v.shape
    if cu_seqlens is not None:
        if B != 1:
            raise ValueError(f"packed sequences come in one row: B is {B}")
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2 or cu_seqlens.dtype not in (torch.int32, torch.int64):
            raise ValueError("cu_seqlens: int32 or int64 [N + 1]")
        cu_seqlens = cu_seqlens.contiguous()
    N = B if cu_seqlens is None else cu_seqlens.numel() - 1
    if initial_state is not None:
        if tuple(initial_state.shape) != (N, Hv, d, d) or initial_state.dtype != torch.float32:
            raise ValueError(f"initial_state {tuple(initial_state.shape)} {initial_state.dtype}: expected fp32 {(N, Hv, d, d)}")
    scale = d ** -0.5 if scale is None else float(scale)
    with _device("gated_delta_rule", q, k, v, g, beta, initial_state, cu_seqlens):
        if initial_state is not None:
            initial_state = initial_state.contiguous()
            if initial_state.data_ptr() % 16:
                initial_state = initial_state.clone()
        _range_push("gsa_hip/delta_rule")
        try:
            needed = _needs_grad(q, k, v, g, beta, initial_state)
            q, k, v = _abi._heads(q), _abi._heads(k), _abi._heads(v)
            if needed:
                return _Rule.apply(q, k, v, g, beta, initial_state, cu_seqlens, scale, bool(output_final_state))
            o, final, _ = _abi.delta_rule(q, k, v, g, beta, initial_state, cu_seqlens, scale, output_final_state, False)
            return o, final
        finally:
            _range_pop()


def gated_delta_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                     state: torch.Tensor, state_indices: Optional[torch.Tensor] = None,
                     scale: Optional[float] = None) -> torch.Tensor:
    """One token of each row of a serving batch: o [N,Hv,128]; ``state`` is updated in place.

    q, k [N,Hk,128], v [N,Hv,128], g, beta [N,Hv] as in ``gated_delta_rule``.  state
    [slots,Hv,128,128] fp32, each matrix contiguous.  state_indices (int32 or int64 [N], on
    the device): the state of each row; row n has state n without it.  A row whose index is
    outside [0, slots) is padding: its output is 0 and no state changes.  Rows with the same
    index are consecutive tokens of one sequence, in the batch's order.  At most 65535 rows; with
    state_indices the time grows with their square from some 8000 on (4096 rows: 1.2 times that
    without, 65535: 5 times).

    Forward only: it raises where a gradient would be needed.
    """
    _check(1, q, k, v, g, beta)
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
    if _needs_grad(q, k, v, g, beta, state):
        raise RuntimeError("gated_delta_step is forward only: call it under torch.no_grad()")
    with _device("gated_delta_step", q, k, v, g, beta, state, state_indices):
        if N == 0 or state.shape[0] == 0:
            return v.new_zeros(v.shape)
        _range_push("gsa_hip/delta_step")
        try:
            o = _abi.delta_step(q, k, v, g, beta, state, state_indices, d ** -0.5 if scale is None else float(scale))
            if not state.is_inference():
                _increment_version(state)        # a graph that kept the old state must not use the new one
            return o
        finally:
            _range_pop()
