"""RMS norm with the residual's addition on MI355X: what stands before both mixers of the
study, and by heads on q and k of the gated delta rule.

    h = x + residual (rounded to their type: the stream that the next layer adds to)
    y = h / sqrt(mean(h**2) + eps) * weight

``add_rms_norm`` is differentiable; ``add_rms_norm_fp8`` gives y in 8 bits with one scale a
row, for a product in 8 bits.  Statistics are fp32 of the rounded h.  There is no CPU or
eager fallback.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _abi
from .delta import _device, _needs_grad, _once
from .roctx import range_pop as _range_pop, range_push as _range_push

MAX_D = 32768


def _check(x, weight, residual) -> None:
    shape, dt = x.shape, x.dtype
    if not shape or not 1 <= shape[-1] <= MAX_D:
        raise ValueError(f"x {tuple(shape)}: rows of 1 to {MAX_D} elements")
    if weight.shape != shape[-1:]:
        raise ValueError(f"weight {tuple(weight.shape)} != {(shape[-1],)}")
    if residual is not None and residual.shape != shape:
        raise ValueError(f"residual {tuple(residual.shape)} != x {tuple(shape)}")
    if weight.dtype != dt or residual is not None and residual.dtype != dt:
        raise ValueError("x, weight and residual must share a dtype")
    _abi.dtype_code(dt)


class _Norm(torch.autograd.Function):
    operator = "add_rms_norm"

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, h, rstd = _abi.rms_norm(x, weight, residual, eps, want_rstd=True)
        ctx.set_materialize_grads(False)
        ctx.added = residual is not None
        ctx.save_for_backward(h if ctx.added else x, weight, rstd)
        return (y, h) if ctx.added else y

    @_once
    def backward(ctx, dy, dh=None):
        h, weight, rstd = ctx.saved_tensors
        if dy is None:                           # only h was used
            return dh, torch.zeros_like(weight), dh, None
        _range_push("gsa_hip/rms_norm_backward")
        try:
            dx, dw = _abi.rms_norm_backward(h, dy, dh, weight, rstd)
        finally:
            _range_pop()
        return dx, dw, dx if ctx.added else None, None


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None,
                 eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, h) of x [..., D] (bf16 or fp32), weight [D] and residual (x's shape) in x's dtype;
    h is x itself without a residual.  D up to 32768, fewer than 2**31 rows.  Rows of a strided
    x are read in place where its leading dimensions but one collapse (heads of a projection);
    y and h are contiguous.  Differentiable in all three, once and backwards; the gradients are
    the same bits on every run, and with a residual x and the residual get the same tensor."""
    _check(x, weight, residual)
    with _device("add_rms_norm", x, weight, residual):
        if x.numel() == 0:
            h = x if residual is None else x + residual
            return h * weight, h
        _range_push("gsa_hip/rms_norm")
        try:
            needed = _needs_grad(x, weight, residual)
            weight = weight.contiguous()
            if needed:
                out = _Norm.apply(x, weight, residual, float(eps))
                return out if residual is not None else (out, x)
            y, h, _ = _abi.rms_norm(x, weight, residual, float(eps))
            return y, x if h is None else h
        finally:
            _range_pop()


def add_rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None,
                     eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, scale, h): add_rms_norm with y as float8_e4m3fn [..., D] and fp32 scale [...], so that
    y * scale[..., None] is the normed row; scale is the row's largest magnitude / 448 (1 for a
    row of zeros).  Forward only: it raises where a gradient would be needed."""
    _check(x, weight, residual)
    if _needs_grad(x, weight, residual):
        raise RuntimeError("add_rms_norm_fp8 is forward only: call it under torch.no_grad()")
    with _device("add_rms_norm_fp8", x, weight, residual):
        if x.numel() == 0:
            return (torch.empty_like(x, dtype=torch.float8_e4m3fn), x.new_ones(x.shape[:-1], dtype=torch.float32),
                    x if residual is None else x + residual)
        _range_push("gsa_hip/rms_norm_fp8")
        try:
            y, scale, h = _abi.rms_norm_fp8(x, weight.contiguous(), residual, float(eps))
            return y, scale, x if h is None else h
        finally:
            _range_pop()
