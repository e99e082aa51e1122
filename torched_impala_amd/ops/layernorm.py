"""Layer norm over the last axis (csrc/norm_kernels.hip): one pass forward,
one pass backward with the weight's and the bias's gradients reduced from
per-block partial sums in a fixed order.

    y = (x - mean) * rstd * weight + bias

Statistics, products and sums are fp32 whatever the input's type; the output
and the gradients are rounded once, to the type of what they belong to.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from torched_impala_amd import ops

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _check(x, weight, bias, eps):
    if x.dtype not in _TYPES:
        raise TypeError(f"layer_norm: x must be fp32, bf16 or fp16, "
                        f"not {x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("layer_norm: x needs a last axis of one or more")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.shape != x.shape[-1:]:
            raise ValueError(f"layer_norm: {name} must be "
                             f"({x.shape[-1]},), not {tuple(p.shape)}")
        if p.dtype is not torch.float32 and p.dtype is not x.dtype:
            raise TypeError(f"layer_norm: {name} must be fp32 or of x's "
                            f"type, not {p.dtype}")
        if p.device != x.device:
            raise ValueError(f"layer_norm: {name} is on {p.device}, "
                             f"x on {x.device}")
    if weight is not None and bias is not None \
            and weight.dtype is not bias.dtype:
        raise TypeError("layer_norm: weight and bias must have one type")
    if not (math.isfinite(eps) and eps >= 0.0):
        raise ValueError(f"layer_norm: eps must be finite and >= 0, "
                         f"not {eps}")


def _rows(x: torch.Tensor) -> torch.Tensor:
    """(rows, cols) with unit column stride: a view where strides allow."""
    x = x.reshape(-1, x.shape[-1]) if x.dim() != 2 else x
    if x.shape[1] > 1 and x.stride(1) != 1:
        x = x.contiguous()
    return x


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        w = weight.contiguous() if weight is not None else None
        b = bias.contiguous() if bias is not None else None
        y, stats = ops.ext_hip().layer_norm_fwd(_rows(x), w, b, eps, True)
        # x itself is saved, not its 2-D view, so that an in-place change
        # of it before backward is caught
        ctx.save_for_backward(x, w, stats)
        p = bias if weight is None else weight
        ctx.param_fp32 = p is None or p.dtype is torch.float32
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, stats = ctx.saved_tensors
        nx, nw, nb = ctx.needs_input_grad[:3]
        xr = _rows(x)
        dx, dw, db = ops.ext_hip().layer_norm_bwd(
            dy.reshape(xr.shape).contiguous(), xr, w, stats, nx, nw, nb,
            ctx.param_fp32)
        return (dx.view(x.shape) if nx else None), dw, db, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5,
               force_eager: bool = False) -> torch.Tensor:
    """Layer norm of ``x`` (..., cols) over its last axis.

    ``x`` is fp32, bf16 or fp16 with any strides (a copy is made only where
    its rows have no common stride or its columns are not adjacent).
    ``weight`` and ``bias`` are (cols,), fp32 or of x's type, each optional.
    Returns a contiguous tensor of x's shape and type; differentiable once
    in x, weight and bias. ``force_eager`` takes torch's ops instead of the
    kernels. Raises TypeError or ValueError for anything else.
    """
    _check(x, weight, bias, eps)
    if force_eager or not (x.is_cuda and ops.hip_available()):
        # eager fallback (CPU tests / escape hatch) — same math
        f32 = torch.float32
        return torch.nn.functional.layer_norm(
            x.to(f32), x.shape[-1:],
            None if weight is None else weight.to(f32),
            None if bias is None else bias.to(f32), eps).to(x.dtype)
    if torch.is_grad_enabled() and (
            x.requires_grad
            or (weight is not None and weight.requires_grad)
            or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    y, _ = ops.ext_hip().layer_norm_fwd(
        _rows(x), None if weight is None else weight.contiguous(),
        None if bias is None else bias.contiguous(), float(eps), False)
    return y.view(x.shape)
