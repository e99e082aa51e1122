"""Linear-attention recurrent core: an alternative to the LSTM whose unroll
runs in parallel over time (ops/linear_attention.py).

    z   = proj_in(x)
    q, k, v = qkv(layer_norm(z))                     4 heads of 64
    S_t = lambda_h * (0 if done_t else S_{t-1}) + k_t v_t^T
    out = z + proj_out(layer_norm_per_head(q_t^T S_t / 8))

The decays are fixed, spread over the heads: memories of 8, 32, 128 and 512
steps. The state is carried flat, (B, heads * 64 * 64), so that it travels
through the rollout buffers like any other core state.
"""
from __future__ import annotations

from typing import Tuple

import torch
import torch.nn as nn

from torched_impala_amd.ops.layernorm import layer_norm
from torched_impala_amd.ops.linear_attention import (linear_attention,
                                                     linear_attention_step)


class LinearAttentionCore(nn.Module):
    def __init__(self, input_size: int, hidden_size: int = 256,
                 heads: int = 4):
        super().__init__()
        if hidden_size % heads:
            raise ValueError(f"{heads} heads do not divide {hidden_size}")
        self.hidden_size = hidden_size
        self.heads = heads
        self.head_size = hidden_size // heads
        self.proj_in = nn.Linear(input_size, hidden_size)
        self.norm = nn.LayerNorm(hidden_size)
        self.qkv = nn.Linear(hidden_size, 3 * hidden_size, bias=False)
        self.head_norm = nn.LayerNorm(self.head_size)
        self.proj_out = nn.Linear(hidden_size, hidden_size)
        # not a parameter and not in the checkpoint: it follows from `heads`
        memory = 8.0 * 4.0 ** torch.arange(heads, dtype=torch.float64)
        self.register_buffer("log_decay", torch.log1p(-1.0 / memory).float(),
                             persistent=False)

    @property
    def state_size(self) -> int:
        return self.heads * self.head_size * self.head_size

    def initial_state(self, batch_size: int) -> Tuple[torch.Tensor]:
        return (torch.zeros(batch_size, self.state_size,
                            device=self.log_decay.device),)

    def forward(self, x: torch.Tensor, done: torch.Tensor,
                state: Tuple[torch.Tensor], force_eager: bool = False):
        """x (T, B, F), done (T, B) bool -> (T * B, hidden), state."""
        T, B = x.shape[:2]
        H, D = self.heads, self.head_size
        s, = state
        s = s.view(B, H, D, D)
        z = self.proj_in(x)
        y = layer_norm(z, self.norm.weight, self.norm.bias, self.norm.eps,
                       force_eager=force_eager)
        q, k, v = self.qkv(y).view(T, B, 3, H, D).unbind(2)
        if T == 1 and not torch.is_grad_enabled() and not force_eager:
            o, s = linear_attention_step(q[0], k[0], v[0], self.log_decay, s,
                                         done=done[0])
            o = o.unsqueeze(0)
        else:
            o, s = linear_attention(q, k, v, self.log_decay, done=done,
                                    state=s, force_eager=force_eager)
        o = layer_norm(o, self.head_norm.weight, self.head_norm.bias,
                       self.head_norm.eps, force_eager=force_eager)
        out = z + self.proj_out(o.flatten(-2))
        return out.view(T * B, self.hidden_size), (s.reshape(B, -1),)
