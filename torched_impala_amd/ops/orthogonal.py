"""Orthogonalised updates by Newton-Schulz products (csrc/ortho_kernels.hip).

    X = G / (|G| + eps);   `steps` times:  A = X X^T
                                           X = (a I + b A + c A A) X

with (a, b, c) = (3.4445, -4.7750, 2.0315), on the side of the matrix with
the fewer rows. Five rounds bring the singular values of G to a band around
one and leave its singular vectors: the update direction of FlatMuon
(ops/optim.py).
"""
from __future__ import annotations

import bisect
import math
from typing import List, Optional, Sequence

import torch

from torched_impala_amd import ops

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
_TYPES = (torch.float32, torch.bfloat16, torch.float16)
_MAX_SIDE, _MAX_SMALL_SIDE = (1 << 20) - 1, 32768


def _span(t):
    """First byte and the byte behind the last (t not empty)."""
    n = sum((s - 1) * st for s, st in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (n + 1) * t.element_size()


def _check_out(mats, out):
    if len(out) != len(mats):
        raise ValueError(f"orthogonalize: {len(out)} results for "
                         f"{len(mats)} matrices")
    for i, (g, o) in enumerate(zip(mats, out)):
        if o.dtype is not g.dtype:
            raise TypeError(f"orthogonalize: result {i} is {o.dtype}, its "
                            f"matrix {g.dtype}")
        if o.shape != g.shape or o.device != g.device:
            raise ValueError(f"orthogonalize: result {i} does not match its "
                             "matrix")
        if not (o.is_contiguous() or o.t().is_contiguous()):
            raise ValueError(f"orthogonalize: result {i} must be dense")
        if o.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("orthogonalize writes its results in place; "
                               "they must not require grad")
    if ops.has_tangent(out):
        raise RuntimeError("orthogonalize writes its results in place; they "
                           "must not carry a forward-mode derivative")
    # a result may lie on its own matrix, on nothing else
    spans = sorted((*_span(o), i) for i, o in enumerate(out) if o.numel())
    for (_, e, i), (s, _, j) in zip(spans, spans[1:]):
        if s < e:
            raise ValueError(f"orthogonalize: results {i} and {j} overlap")
    starts = [s for s, _, _ in spans]
    for j, g in enumerate(mats):
        if not g.numel():
            continue
        s, e = _span(g)
        k = max(0, bisect.bisect_right(starts, s) - 1)
        while k < len(spans) and spans[k][0] < e:
            if spans[k][1] > s and spans[k][2] != j:
                raise ValueError(f"orthogonalize: result {spans[k][2]} "
                                 f"overlaps matrix {j}")
            k += 1


def _eager_one(g, steps, eps):
    a, b, c = COEFFICIENTS
    x = g.float()
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.t()
    x = x / (torch.linalg.vector_norm(x) + eps)
    for _ in range(steps):
        m = x @ x.t()
        x = a * x + (b * m + c * (m @ m)) @ x
    return (x.t() if tall else x).to(g.dtype)


def orthogonalize(mats: Sequence[torch.Tensor], steps: int = 5,
                  eps: float = 1e-7,
                  out: Optional[Sequence[torch.Tensor]] = None
                  ) -> List[torch.Tensor]:
    """Orthogonalise a list of matrices, all in the same few launches.

    Each matrix is 2-D, fp32, bf16 or fp16 (they may differ), of any strides
    and any sizes up to 32768 on its shorter and 2^20 - 1 on its longer side;
    empty ones give empty results. The products run at fp32 accuracy; a
    result is rounded once, to its matrix's type. ``steps`` is one or more,
    ``eps`` finite and at least 0 (with 0 a zero matrix gives NaN).

    Results are new contiguous tensors, or written to ``out``: dense tensors
    of the matrices' shapes and types, each apart from the other results and
    matrices (its own it may overwrite). Not differentiable: raises
    RuntimeError where a matrix requires grad or carries a forward-mode
    derivative, TypeError or ValueError for anything else that does not fit.
    """
    mats = list(mats)
    for i, g in enumerate(mats):
        if g.dtype not in _TYPES:
            raise TypeError(f"orthogonalize: matrix {i} must be fp32, bf16 "
                            f"or fp16, not {g.dtype}")
        if g.dim() != 2:
            raise ValueError(f"orthogonalize: matrix {i} must have 2 axes, "
                             f"not {g.dim()}")
        if g.device != mats[0].device:
            raise ValueError(f"orthogonalize: matrix {i} is on {g.device}, "
                             f"the first on {mats[0].device}")
        if max(g.shape) > _MAX_SIDE or min(g.shape) > _MAX_SMALL_SIDE:
            raise ValueError(f"orthogonalize: matrix {i} is too large: "
                             f"{tuple(g.shape)}")
        if g.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("orthogonalize has no gradient; pass the "
                               "matrices detached")
    if ops.has_tangent(mats):
        raise RuntimeError("orthogonalize has no forward-mode derivative")
    if not isinstance(steps, int) or steps < 1:
        raise ValueError(f"orthogonalize: steps must be an integer of one "
                         f"or more, not {steps}")
    if not (math.isfinite(eps) and eps >= 0.0):
        raise ValueError(f"orthogonalize: eps must be finite and >= 0, "
                         f"not {eps}")
    if out is not None:
        out = list(out)
        _check_out(mats, out)
    if not mats:
        return []
    if not (mats[0].is_cuda and ops.hip_available()):
        # eager fallback (CPU tests / escape hatch) — same math
        with torch.no_grad():
            res = [_eager_one(g, steps, eps) for g in mats]
            if out is None:
                return [r.contiguous() for r in res]
            return [o.copy_(r) for o, r in zip(out, res)]
    if out is None:
        out = [torch.empty(g.shape, dtype=g.dtype, device=g.device)
               for g in mats]
    else:
        for o in out:
            if not o.is_inference():
                torch.autograd.graph.increment_version(o)
    ops.ext_hip().orthogonalize(mats, out, steps, float(eps))
    return out
