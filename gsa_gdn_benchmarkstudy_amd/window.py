"""Attention in a sliding window on MI355X, with a few first tokens that stay visible: the selected
attention's counterpart whose selection is known beforehand, and whose cache has a constant size.

Key j is visible to query i where ``j <= i`` and (``j > i - window`` or ``j < sinks``), positions
counted in each sequence.  ``window_attention`` runs whole sequences (training, prefill) and is
differentiable; ``window_attention_step`` runs one token of each row of a serving batch on caches
that ``window_cache_write`` filled.  There is no CPU or eager fallback.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.graph import increment_version as _increment_version

from . import _abi
from .delta import D_HEAD, _device, _needs_grad, _once
from .roctx import range_pop as _range_pop, range_push as _range_push

_MOST = (1 << 30) - 1                            # keys of a window and first tokens


def _check_heads(n: int, q, k, v) -> None:
    """Shapes and types; n: dimensions before the heads."""
    qs, ks = q.shape, k.shape
    lead = "B, T" if n == 2 else "N"
    if len(qs) != n + 2 or len(ks) != n + 2 or v.shape != ks or qs[:n] != ks[:n]:
        raise ValueError(f"q {tuple(qs)}, k {tuple(ks)}, v {tuple(v.shape)}: expected [{lead}, heads, {D_HEAD}]")
    if qs[-1] != D_HEAD or ks[-1] != D_HEAD:
        raise ValueError(f"head dims {qs[-1]} and {ks[-1]}: the kernels take {D_HEAD}")
    _check_groups(qs[n], ks[n])
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"q, k, v must share a dtype: got {q.dtype}, {k.dtype}, {v.dtype}")
    _abi.dtype_code(q.dtype)


def _check_groups(H: int, Hkv: int) -> None:
    if Hkv < 1 or H < 1 or H % Hkv or H > 65535:
        raise ValueError(f"{H} query heads are not a multiple of {Hkv} key heads (65535 at most)")


def _check_window(window, sinks) -> None:
    if isinstance(window, bool) or not isinstance(window, int) or not 1 <= window <= _MOST:
        raise ValueError(f"window {window!r}: an integer from 1")
    _check_sinks(sinks)
    if window + sinks > _MOST:
        raise ValueError(f"window {window} and sinks {sinks}: at most {_MOST} keys")


def _check_sinks(sinks) -> None:
    if isinstance(sinks, bool) or not isinstance(sinks, int) or not 0 <= sinks <= _MOST:
        raise ValueError(f"sinks {sinks!r}: an integer from 0")


def _check_packed(cu, B: int):
    if B != 1:
        raise ValueError(f"packed sequences come in one row: B is {B}")
    if cu.dim() != 1 or cu.numel() < 2 or cu.dtype not in (torch.int32, torch.int64):
        raise ValueError("cu_seqlens: int32 or int64 [N + 1]")
    if cu.numel() >= 1 << 31:                    # (the C interface counts in 32 bits)
        raise ValueError(f"{cu.numel() - 1} sequences: fewer than 2**31 - 1")
    return cu.contiguous()


def _index(t: Optional[torch.Tensor], N: int, name: str):
    if t is None:
        return None
    if t.shape != (N,) or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name}: int32 or int64 [{N}]")
    return t.contiguous()


class _Window(torch.autograd.Function):
    operator = "window_attention"

    @staticmethod
    def forward(ctx, q, k, v, cu, window, sinks, scale):
        o, lse, low = _abi.window_attn(q, k, v, cu, window, sinks, scale, True)
        ctx.set_materialize_grads(False)
        ctx.window, ctx.sinks, ctx.scale = window, sinks, scale
        ctx.save_for_backward(q, k, v, cu, o, lse, low)
        return o

    @_once
    def backward(ctx, do):
        q, k, v, cu, o, lse, low = ctx.saved_tensors
        if do is None:
            return (None,) * 7
        _range_push("gsa_hip/window_attention_backward")
        try:
            grads = _abi.window_attn_backward(q, k, v, cu, ctx.window, ctx.sinks, ctx.scale, o, lse, low, _abi._heads(do))
        finally:
            _range_pop()
        return (*grads, None, None, None, None)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int = 0, scale: Optional[float] = None,
                     cu_seqlens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """o [B,T,H,128] of causal attention over the last ``window`` tokens and the first ``sinks``.

    q [B,T,H,128], k and v [B,T,Hkv,128] in bf16 or fp32; query head h goes with key head
    h // (H // Hkv).  Strided views with contiguous head rows are read in place.  window: at least 1
    (a token sees itself); from T on the attention is causal.  scale: 128**-0.5 unless given.

    cu_seqlens (int32 or int64 [N+1], on the device, ascending from 0): B is 1 and N sequences are
    packed in T, each with its own window and first tokens; empty ones are allowed.  Rows of o and
    of the gradients outside every sequence are 0, whatever the inputs hold there.  What a query
    does not see may hold a NaN or an infinity without changing a bit of its output, so padding behind the tokens of
    a batch's row may hold anything (its outputs are to be ignored; queries that stand with it in a block of 64 or 128 take
    up to some six times as long).
    Gradients it reaches, as 0 * NaN does: where they are wanted, padding has to be finite, or
    left out by packing.

    Differentiable in q, k and v, once and backwards (a tangent of torch.autograd.forward_ad raises);
    the gradients are the same bits on every run.  Fewer than 2**31 tokens and at most 2**23 blocks of
    32 tokens (a sequence's last one may be shorter) times heads.

    May be captured into a graph, forward and backward, after one call outside of it; as with any
    backward pass no eager graph of the same leaves may live then (capture torch.autograd.grad, or
    use leaves of the graph's own).
    """
    _check_heads(2, q, k, v)
    _check_window(window, sinks)
    if cu_seqlens is not None:
        cu_seqlens = _check_packed(cu_seqlens, q.shape[0])
    scale = D_HEAD ** -0.5 if scale is None else float(scale)
    with _device("window_attention", q, k, v, cu_seqlens):
        _range_push("gsa_hip/window_attention")
        try:
            needed = _needs_grad(q, k, v)
            q, k, v = _abi._heads(q), _abi._heads(k), _abi._heads(v)
            if needed:
                return _Window.apply(q, k, v, cu_seqlens, window, sinks, scale)
            return _abi.window_attn(q, k, v, cu_seqlens, window, sinks, scale, False)[0]
        finally:
            _range_pop()


def _check_caches(k_cache, v_cache, Hkv: int, dtype, rows: int) -> None:
    for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if t.dim() != 4 or t.shape[2:] != (Hkv, D_HEAD) or t.dtype != dtype:
            raise ValueError(f"{name} {tuple(t.shape)} {t.dtype}: expected {dtype} [slots, rows, {Hkv}, {D_HEAD}]")
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("caches are written in place: call it under torch.no_grad()")
        if t.is_contiguous() and t.data_ptr() % 16 == 0:
            continue
        s0, s1, s2, s3 = t.stride()
        if s3 != 1 or ((s0 | s1 | s2) * t.element_size() | t.data_ptr()) % 16:
            raise ValueError(f"{name} is updated in place: its rows must be contiguous and 16-byte aligned")
        extent = D_HEAD
        for stride, n in sorted(zip((s0, s1, s2), t.shape)):
            if n > 1:
                if stride < extent:
                    raise ValueError(f"{name} is updated in place: its rows overlap")
                extent += (n - 1) * stride
    if k_cache.shape != v_cache.shape:
        raise ValueError(f"k_cache {tuple(k_cache.shape)} != v_cache {tuple(v_cache.shape)}")
    if not rows <= k_cache.shape[1] <= _MOST:
        raise ValueError(f"caches of {k_cache.shape[1]} rows: at least {rows}, and at most {_MOST}")
    if k_cache.data_ptr() == v_cache.data_ptr() and k_cache.numel():
        raise ValueError("k_cache and v_cache are the same memory")


def _written(*ts: torch.Tensor) -> None:
    ts = tuple(t for t in ts if not t.is_inference())
    if ts:
        _increment_version(ts)                   # a graph that kept the old caches must not use the new ones


def window_cache_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, sinks: int = 0,
                       positions: Optional[torch.Tensor] = None, cache_indices: Optional[torch.Tensor] = None,
                       cu_seqlens: Optional[torch.Tensor] = None) -> None:
    """Keys and values of B sequences (or N packed ones) to their caches, in place.

    k, v [B,T,Hkv,128] as ``window_attention`` takes them; k_cache, v_cache [slots,rows,Hkv,128]
    in the same dtype, more rows than ``sinks``.  The token at position p of its sequence is kept in row p
    (p < sinks) or in sinks + (p - sinks) % (rows - sinks): first tokens stay, the others turn in a ring, in which
    later tokens take the rows of earlier ones.  positions (int32 or int64 [N], on the device): of
    each sequence's first token here; 0 without it (a prompt's beginning).  cache_indices (int32 or int64 [N],
    on the device): each sequence's slot; sequence n has slot n without it.  A slot outside
    [0, slots) and a position outside [0, 2**62) are skipped.  Two sequences of one call that write one
    row leave either's key and either's value there.  k and v are not parts of the caches.  Fewer than 2**29 tokens, in
    fewer than 2**23 blocks of 64.
    """
    _check_sinks(sinks)
    if k.dim() != 4 or v.shape != k.shape or k.shape[-1] != D_HEAD or k.shape[2] < 1:
        raise ValueError(f"k {tuple(k.shape)}, v {tuple(v.shape)}: expected [B, T, heads, {D_HEAD}]")
    if v.dtype != k.dtype:
        raise ValueError(f"k and v must share a dtype: got {k.dtype}, {v.dtype}")
    _abi.dtype_code(k.dtype)
    B, T, Hkv, _ = k.shape
    if B * T >= 1 << 29:
        raise ValueError(f"{B} x {T} tokens: fewer than 2**29")
    _check_caches(k_cache, v_cache, Hkv, k.dtype, sinks + 1)
    if cu_seqlens is not None:
        cu_seqlens = _check_packed(cu_seqlens, B)
    N = B if cu_seqlens is None else cu_seqlens.numel() - 1
    positions, cache_indices = _index(positions, N, "positions"), _index(cache_indices, N, "cache_indices")
    if cache_indices is None and N > k_cache.shape[0]:
        raise ValueError(f"{N} sequences, {k_cache.shape[0]} caches")
    if _needs_grad(k, v):
        raise RuntimeError("window_cache_write is forward only: call it under torch.no_grad()")
    with _device("window_cache_write", k, v, k_cache, v_cache, positions, cache_indices, cu_seqlens):
        if B * T == 0 or k_cache.shape[0] == 0:
            return
        _range_push("gsa_hip/window_cache_write")
        try:
            _abi.window_cache_write(_abi._rows16(k), _abi._rows16(v), k_cache, v_cache, sinks, positions, cache_indices, cu_seqlens)
            _written(k_cache, v_cache)
        finally:
            _range_pop()


def window_attention_step(q: torch.Tensor, k: Optional[torch.Tensor], v: Optional[torch.Tensor], k_cache: torch.Tensor, v_cache: torch.Tensor,
                          positions: torch.Tensor, window: int, sinks: int = 0, cache_indices: Optional[torch.Tensor] = None,
                          scale: Optional[float] = None) -> torch.Tensor:
    """One token of each row of a serving batch: o [N,H,128]; the caches are updated in place.

    q [N,H,128], k and v [N,Hkv,128] of the tokens at ``positions`` (int32 or int64 [N], on the
    device) of their sequences; caches and cache_indices as in ``window_cache_write``, of at least
    window + sinks rows.  First k and v of all rows go to the caches, then each row's attention is
    taken over the tokens that it sees there, its own among them.  k and v may both be None: they
    are in the caches already.  A row whose index is outside [0, slots) or whose position is
    outside [0, 2**62) is padding: its output is 0 and no cache changes.  Rows with the same index are
    tokens of one sequence, each at its own position: up to rows - sinks - window + 1 consecutive ones (more would take
    each other's rows).  Rows of a cache that the token does not see are not read.  At most 65535 rows.

    Forward only: it raises where a gradient would be needed.
    """
    if (k is None) != (v is None):
        raise ValueError("k and v: both, or neither")
    if k is None:
        if q.dim() != 3 or q.shape[-1] != D_HEAD or k_cache.dim() != 4:
            raise ValueError(f"q {tuple(q.shape)}, k_cache {tuple(k_cache.shape)}: expected [N, heads, {D_HEAD}], [slots, rows, heads, {D_HEAD}]")
        _check_groups(q.shape[1], k_cache.shape[2])
        _abi.dtype_code(q.dtype)
    else:
        _check_heads(1, q, k, v)
    _check_window(window, sinks)
    N, Hkv = q.shape[0], k_cache.shape[2] if k is None else k.shape[1]
    _check_caches(k_cache, v_cache, Hkv, q.dtype, window + sinks)
    positions, cache_indices = _index(positions, N, "positions"), _index(cache_indices, N, "cache_indices")
    if cache_indices is None and N > k_cache.shape[0]:
        raise ValueError(f"{N} rows, {k_cache.shape[0]} caches")
    if _needs_grad(q, k, v):
        raise RuntimeError("window_attention_step is forward only: call it under torch.no_grad()")
    with _device("window_attention_step", q, k, v, k_cache, v_cache, positions, cache_indices):
        if N == 0 or k_cache.shape[0] == 0:
            return q.new_zeros(q.shape)
        _range_push("gsa_hip/window_step")
        try:
            o = _abi.window_step(_abi._rows16(q), None if k is None else _abi._rows16(k), None if v is None else _abi._rows16(v), k_cache,
                                 v_cache, positions, cache_indices, window, sinks, D_HEAD ** -0.5 if scale is None else float(scale))
            if k is not None:
                _written(k_cache, v_cache)
            return o
        finally:
            _range_pop()
