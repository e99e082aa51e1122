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

from torched_impala_amd import ops

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _check(x, weight, bias, eps):
    """What the kernels' host side (csrc/core_ops.cpp) checks, for the eager
    path."""
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
    kernels, which raise RuntimeError where an input carries a forward-mode
    derivative. Raises TypeError or ValueError for anything else.
    """
    ext = None if force_eager else ops.ext_for(x)
    if ext is not None:   # checks, saves and differentiates by itself
        return ext.layer_norm(x, weight, bias, eps)
    # eager fallback (CPU tests / escape hatch) — same math
    _check(x, weight, bias, eps)
    f32 = torch.float32
    return torch.nn.functional.layer_norm(
        x.to(f32), x.shape[-1:],
        None if weight is None else weight.to(f32),
        None if bias is None else bias.to(f32), eps).to(x.dtype)
