"""Linear attention with one decay per head (csrc/attn_kernels.hip): a
recurrent core that runs in parallel over the unroll.

    S_t = exp(log_decay_h) * (0 if done_t else S_{t-1}) + k_t v_t^T
    o_t = scale * q_t^T S_t

``done_t`` cuts the memory before step t, as it does for the LSTM core: a
step flagged done is the first of its episode. The state S is (dk, dv) a
head, fp32.

* ``linear_attention``       a whole unroll, (T, B, H, d), differentiable in
                             q, k, v and the state;
* ``linear_attention_step``  one step of a batch, for acting.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from torched_impala_amd import ops

_TYPES = (torch.float32, torch.bfloat16, torch.float16)
MAX_HEAD = 128
MAX_HEADS = ((1 << 32) - 1) // (3 * 512)   # of a batch, as the kernels launch


def _check(name, q, k, v, log_decay, done, state, scale, lead):
    """Shapes, types and devices of a call, as the kernels' host side
    (csrc/core_ops.cpp) checks them, for the eager path; returns the scale."""
    if q.dtype not in _TYPES:
        raise TypeError(f"{name}: q must be fp32, bf16 or fp16, "
                        f"not {q.dtype}")
    for n, t in (("k", k), ("v", v)):
        if t.dtype is not q.dtype:
            raise TypeError(f"{name}: {n} is {t.dtype}, q {q.dtype}")
        if t.device != q.device:
            raise ValueError(f"{name}: {n} is on {t.device}, q on "
                             f"{q.device}")
    if q.dim() != lead + 2:
        raise ValueError(f"{name}: q must have {lead + 2} axes, "
                         f"not {q.dim()}")
    if k.shape != q.shape:
        raise ValueError(f"{name}: k is {tuple(k.shape)}, "
                         f"q {tuple(q.shape)}")
    if v.dim() != q.dim() or v.shape[:-1] != q.shape[:-1]:
        raise ValueError(f"{name}: v is {tuple(v.shape)}, "
                         f"q {tuple(q.shape)}")
    dk, dv = q.shape[-1], v.shape[-1]
    if not (1 <= dk <= MAX_HEAD and 1 <= dv <= MAX_HEAD):
        raise ValueError(f"{name}: head sizes must be 1 to {MAX_HEAD}, "
                         f"not {dk} and {dv}")
    H = q.shape[-2]
    if q.shape[lead - 1] * H > MAX_HEADS:
        raise ValueError(f"{name}: batch times heads must be at most "
                         f"{MAX_HEADS}")
    if log_decay.dtype is not torch.float32:
        raise TypeError(f"{name}: log_decay must be fp32, "
                        f"not {log_decay.dtype}")
    if log_decay.shape != (H,) or log_decay.device != q.device:
        raise ValueError(f"{name}: log_decay must be ({H},) on {q.device}, "
                         f"not {tuple(log_decay.shape)} on "
                         f"{log_decay.device}")
    if log_decay.requires_grad:
        raise ValueError(f"{name}: log_decay is a head's fixed slope and "
                         "gets no gradient; pass it detached")
    if done is not None:
        if done.dtype is not torch.bool:
            raise TypeError(f"{name}: done must be bool, not {done.dtype}")
        if done.shape != q.shape[:lead] or done.device != q.device:
            raise ValueError(f"{name}: done must be "
                             f"{tuple(q.shape[:lead])} on {q.device}, not "
                             f"{tuple(done.shape)} on {done.device}")
    if state is not None:
        want = (q.shape[lead - 1], H, dk, dv)
        if state.dtype is not torch.float32:
            raise TypeError(f"{name}: the state must be fp32, "
                            f"not {state.dtype}")
        if state.shape != want or state.device != q.device:
            raise ValueError(f"{name}: the state must be {want} on "
                             f"{q.device}, not {tuple(state.shape)} on "
                             f"{state.device}")
    if scale is None:
        return dk ** -0.5
    if not math.isfinite(scale):
        raise ValueError(f"{name}: scale must be finite, not {scale}")
    return float(scale)


def _eager(q, k, v, log_decay, done, state, scale):
    """The recurrence in fp32 torch ops (CPU tests / escape hatch)."""
    T, B, H, dk = q.shape
    lam = torch.exp(log_decay).view(1, H, 1, 1)
    s = (torch.zeros(B, H, dk, v.shape[-1], device=q.device)
         if state is None else state)
    qf, kf, vf = q.float(), k.float(), v.float()
    outs = []
    for t in range(T):
        s = s * lam
        if done is not None:
            s = torch.where(done[t].view(B, 1, 1, 1), torch.zeros_like(s), s)
        s = s + kf[t].unsqueeze(-1) * vf[t].unsqueeze(-2)
        outs.append(scale * (qf[t].unsqueeze(-1) * s).sum(-2))
    out = (torch.stack(outs) if outs else vf.new_empty(v.shape))
    return out.to(q.dtype), (s if T else s.clone())


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                     log_decay: torch.Tensor, *,
                     done: Optional[torch.Tensor] = None,
                     state: Optional[torch.Tensor] = None,
                     scale: Optional[float] = None,
                     force_eager: bool = False
                     ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Linear attention over a time-major unroll.

    ``q``, ``k`` (T, B, H, dk) and ``v`` (T, B, H, dv) share one type, fp32,
    bf16 or fp16; head sizes are 1 to 128; T, B or H may be 0, B * H up to
    2796202 (the threads of a launch). Any strides:
    the three may be parts of one projection, or broadcast over an axis
    (a copy is made only where a head's features are not adjacent).
    ``log_decay`` (H,) fp32 is each head's slope, at most 0; larger values
    are not refused (that would wait for the device) and make the state
    grow. -inf keeps nothing of the step before.
    ``done`` (T, B) bool cuts the memory before a step. ``state``
    (B, H, dk, dv) fp32 is what enters the first step, zero if left out.
    ``scale`` defaults to dk ** -0.5. ``force_eager`` takes torch's ops, a
    step at a time, instead of the kernels.

    Returns ``(out, final)``: out (T, B, H, dv) of q's type and the state
    behind the last step, fp32. Differentiable once in q, k, v and state,
    through both results; log_decay gets no gradient. The kernels raise
    RuntimeError where an input carries a forward-mode derivative, which
    torch's ops carry on. NaN and infinities
    reach the steps that the recurrence carries them to, never an earlier
    step or another episode. Raises TypeError or ValueError for anything
    else.
    """
    ext = None if force_eager else ops.ext_for(q)
    if ext is not None:   # checks, saves and differentiates by itself
        return ext.linear_attention(q, k, v, log_decay, done, state, scale)
    scale = _check("linear_attention", q, k, v, log_decay, done, state,
                   scale, 2)
    return _eager(q, k, v, log_decay, done, state, scale)


def _span(t: torch.Tensor, axis: int) -> int:
    """Bytes from a tensor's first one to behind the last, of the axes from
    ``axis`` on."""
    n = sum((s - 1) * st for s, st in zip(t.shape[axis:], t.stride()[axis:]))
    return (n + 1) * t.element_size()


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Two tensors of environments, neither empty, without common memory: one
    behind the other, or an environment's parts of both side by side in
    records of one size."""
    p, q = a.data_ptr(), b.data_ptr()
    if p + _span(a, 0) <= q or q + _span(b, 0) <= p:
        return True
    record = a.stride(0) * a.element_size()
    if record <= 0 or b.stride(0) * b.element_size() != record:
        return False
    at = (q - p) % record
    return at >= _span(a, 1) and at + _span(b, 1) <= record


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                          log_decay: torch.Tensor, state: torch.Tensor, *,
                          done: Optional[torch.Tensor] = None,
                          scale: Optional[float] = None,
                          out_state: Optional[torch.Tensor] = None
                          ) -> Tuple[torch.Tensor, torch.Tensor]:
    """One step of a batch: q, k (B, H, dk), v (B, H, dv), state
    (B, H, dk, dv) fp32, done (B,). Returns ``(out, new_state)``.

    The new state is written to ``out_state`` if given, which may be
    ``state`` itself (in place) or memory apart from it, and is apart from all
    other inputs; its environments may lie apart (a slice of a larger pool),
    an environment's heads are contiguous. Not differentiable: raises RuntimeError where a gradient is
    asked for (``linear_attention`` with T = 1 has one) or an input carries a
    forward-mode derivative.
    """
    ext = ops.ext_for(q)
    if ext is not None:
        return ext.linear_attention_step(q, k, v, log_decay, state, done,
                                         scale, out_state)
    scale = _check("linear_attention_step", q, k, v, log_decay, done, state,
                   scale, 1)
    if torch.is_grad_enabled() and any(
            t.requires_grad for t in (q, k, v, state)):
        raise RuntimeError("linear_attention_step has no gradient; use "
                           "linear_attention with T = 1")
    if ops.has_tangent(t for t in (q, k, v, log_decay, state, out_state)
                       if t is not None):
        raise RuntimeError("linear_attention_step has no forward-mode "
                           "derivative")
    if out_state is not None:
        if out_state.dtype is not torch.float32:
            raise TypeError("linear_attention_step: out_state must be fp32, "
                            f"not {out_state.dtype}")
        if out_state.shape != state.shape \
                or out_state.device != state.device:
            raise ValueError("linear_attention_step: out_state must match "
                             "the state")
        if out_state.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("linear_attention_step writes out_state in "
                               "place; it must not require grad")
        heads = state.shape[1] * state.shape[2] * state.shape[3]
        if out_state.numel():
            if not out_state[0].is_contiguous() or (
                    out_state.shape[0] > 1
                    and out_state.stride(0) < heads):
                raise ValueError("linear_attention_step: out_state needs an "
                                 "environment's heads contiguous and "
                                 "environments that do not overlap")
            same = (out_state.data_ptr() == state.data_ptr()
                    and out_state.stride() == state.stride())
            if not (same or _apart(out_state, state)):
                raise ValueError("linear_attention_step: out_state overlaps "
                                 "the state without being it")
            if not all(_apart(out_state, t) for t in (q, k, v, log_decay, done)
                       if t is not None):
                raise ValueError("linear_attention_step: out_state overlaps "
                                 "an input")
    with torch.no_grad():
        out, new = _eager(q.unsqueeze(0), k.unsqueeze(0), v.unsqueeze(0),
                          log_decay,
                          None if done is None else done.unsqueeze(0),
                          state, scale)
        if out_state is not None:
            new = out_state.copy_(new)
    return out[0], new
