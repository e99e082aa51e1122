"""Flat-arena RMSProp with fused global-norm clipping.

All parameters, grads and RMSProp state live in single contiguous fp32
buffers; ``p.data`` / ``p.grad`` are views into them (ordered by REVERSE
parameter order ≈ backward completion order, so DP buckets fill
contiguously). Consequences:

* optimizer + clip = 2 HIP kernels total (csrc/optim_kernels.hip), with
  lr / DP-scale as device scalars -> hipGraph-capturable;
* data-parallel gradient reduction = zero-copy all-reduce of (slices of)
  ``flat_grad`` (parallel/ddp.py FlatGradReducer);
* ``zero_grad`` = one memset.

Semantics match ``torch.nn.utils.clip_grad_norm_`` +
``torch.optim.RMSprop`` (momentum=0; eps added AFTER sqrt), verified in
tests/test_optim.py. ``state_dict`` emits the torch-RMSprop-compatible
layout (per-param ``square_avg``), keeping the checkpoint format
contract.
"""
from __future__ import annotations

from typing import List

import torch

from torched_impala_amd import ops
from torched_impala_amd.ops.orthogonal import orthogonalize


class FlatRMSprop(torch.optim.Optimizer):
    def __init__(self, params, lr=6e-4, alpha=0.99, eps=0.01,
                 max_grad_norm=40.0, world_size=1):
        params = [p for p in params if p.requires_grad]
        assert params, "no parameters"
        super().__init__(params, dict(lr=lr, alpha=alpha, eps=eps))
        device = params[0].device
        dtype = params[0].dtype
        assert all(p.device == device and p.dtype == torch.float32
                   for p in params), "FlatRMSprop requires fp32 params on one device"
        del dtype
        self.max_grad_norm = float(max_grad_norm)
        # reverse order ~ backward completion order
        self._order: List[torch.nn.Parameter] = self._arena_order(params)
        total = sum(p.numel() for p in self._order)
        self.flat_param = torch.zeros(total, device=device)
        self.flat_grad = torch.zeros(total, device=device)
        self.flat_sqavg = torch.zeros(total, device=device)
        self.slices = {}
        off = 0
        with torch.no_grad():
            for p in self._order:
                n = p.numel()
                self.flat_param[off:off + n].copy_(p.data.reshape(-1))
                p.data = self.flat_param[off:off + n].view_as(p)
                p.grad = self.flat_grad[off:off + n].view_as(p)
                self.slices[p] = (off, n)
                off += n
        self.lr_t = torch.zeros(1, device=device)
        self.norm_sq = torch.zeros(1, device=device)
        # non-finite-gradient skip counter (device; graph-capturable):
        # the fused kernel refuses to apply an update whose global norm
        # is inf/NaN — one poisoned gradient otherwise NaNs the params
        # permanently (0*inf=NaN even at lr=0)
        self.skip_t = torch.zeros(1, device=device)
        self.scale_t = torch.full((1,), 1.0 / world_size, device=device)
        self._steps = 0

    def _arena_order(self, params):
        return list(reversed(params))

    def state_arenas(self):
        """Every flat buffer that a step changes (snapshots, broadcasts)."""
        return [self.flat_param, self.flat_sqavg]

    # --- torch Optimizer API ---
    def zero_grad(self, set_to_none: bool = False):  # noqa: ARG002
        self.flat_grad.zero_()
        # re-establish the grad views if something (e.g. module.zero_grad
        # with set_to_none=True) detached them
        for p in self._order:
            if p.grad is None or p.grad.data_ptr() != \
                    self.flat_grad[self.slices[p][0]].data_ptr():
                off, n = self.slices[p]
                p.grad = self.flat_grad[off:off + n].view_as(p)

    @torch.no_grad()
    def step(self, closure=None):  # noqa: ARG002
        self.sync_lr()
        self.step_device()
        return None

    # --- split API for graph capture ---
    def sync_lr(self):
        """Host-side: push the (scheduler-updated) python lr to device.
        Call OUTSIDE any captured graph, once per step."""
        self.lr_t.fill_(self.param_groups[0]["lr"])
        self._steps += 1
        # keep LRScheduler's step-order bookkeeping happy in graph mode,
        # where optimizer.step() itself is inside the captured graph
        self._step_count = getattr(self, "_step_count", 0) + 1
        self._opt_called = True  # torch>=2.4 scheduler-order check

    @torch.no_grad()
    def step_device(self):
        """Device-side update; every op here is graph-capturable."""
        self.norm_sq.zero_()
        g = self.param_groups[0]
        alpha, eps = g["alpha"], g["eps"]
        if self.flat_param.is_cuda and ops.hip_available():
            ops.ext_hip().fused_clip_rmsprop(
                self.flat_param, self.flat_grad, self.flat_sqavg,
                self.lr_t, self.norm_sq, self.scale_t,
                self.max_grad_norm, alpha, eps, self.skip_t)
            return
        # eager reference path (CPU tests / escape hatch) — same math
        gr = self.flat_grad * self.scale_t
        if self.max_grad_norm > 0:
            norm = gr.norm()
            if not torch.isfinite(norm):
                self.skip_t += 1  # skip the poisoned update (see above)
                return
            coef = torch.clamp(self.max_grad_norm / (norm + 1e-6), max=1.0)
            gr = gr * coef
        self.flat_sqavg.mul_(alpha).addcmul_(gr, gr, value=1.0 - alpha)
        denom = self.flat_sqavg.sqrt().add_(eps)
        self.flat_param.addcdiv_(gr, denom, value=-float(self.lr_t.item()))

    # --- checkpoint interop (torch.optim.RMSprop-compatible layout) ---
    def state_dict(self):
        params = self.param_groups[0]["params"]
        state = {}
        for i, p in enumerate(params):
            off, n = self.slices[p]
            state[i] = {
                "step": self._steps,
                "square_avg": self.flat_sqavg[off:off + n].view_as(p).clone(),
            }
        g = self.param_groups[0]
        groups = [{"lr": g["lr"], "alpha": g["alpha"], "eps": g["eps"],
                   "momentum": 0.0, "weight_decay": 0.0, "centered": False,
                   "params": list(range(len(params)))}]
        return {"state": state, "param_groups": groups}

    def _load_entries(self, sd, wanted):
        """wanted: (parameter, key of its entry) in the state's order. An
        entry that is missing leaves what is there; nothing is changed before
        every entry is known to fit."""
        found = []
        for i, (p, key) in enumerate(wanted):
            ent = sd["state"].get(i, sd["state"].get(str(i)))
            if ent is None:
                continue
            if key not in ent:
                raise ValueError(f"parameter {i} has no {key} in the state: "
                                 "another optimizer's")
            if ent[key].numel() != p.numel():
                raise ValueError(f"parameter {i} has {p.numel()} values, "
                                 f"{ent[key].numel()} in the state")
            found.append((p, ent, key))
        with torch.no_grad():
            for p, ent, key in found:
                off, n = self.slices[p]
                self.flat_sqavg[off:off + n].copy_(
                    ent[key].reshape(-1).to(self.flat_sqavg.device))
                self._steps = int(ent.get("step", self._steps))

    def load_state_dict(self, sd):
        self._load_entries(sd, [(p, "square_avg") for p in
                                self.param_groups[0]["params"]])
        for k in ("lr", "alpha", "eps"):
            if sd.get("param_groups"):
                self.param_groups[0][k] = sd["param_groups"][0].get(
                    k, self.param_groups[0][k])


def muon_matrices(model) -> List[torch.nn.Parameter]:
    """The parameters of a policy net that FlatMuon updates by
    orthogonalised momentum: weights of two axes or more (a convolution's
    as (out, in * kh * kw)), the heads' excepted."""
    heads = {id(p) for name in ("policy", "baseline")
             for p in getattr(model, name).parameters()}
    return [p for p in model.parameters()
            if p.requires_grad and p.dim() >= 2 and id(p) not in heads]


class FlatMuon(FlatRMSprop):
    """Orthogonalised momentum for matrices, RMSProp for the rest, over the
    same flat arenas (the matrices' behind the others').

    For each matrix W (rows x cols) with clipped gradient g:

        m = mu m + g;   u = g + mu m (Nesterov)
        W = W - muon_lr * sqrt(max(1, rows / cols)) * orthogonalize(u)

    Clipping and the non-finite skip are FlatRMSprop's, with the norm over
    all gradients. param_groups[0] holds the RMSProp parameters, [1] the
    matrices; a scheduler moves both rates, which reach the device as
    scalars, so a step is graph-capturable.
    """

    def __init__(self, params, matrices, lr=6e-4, alpha=0.99, eps=0.01,
                 max_grad_norm=40.0, world_size=1, muon_lr=0.02,
                 muon_momentum=0.95, ns_steps=5):
        self._matrices = [p for p in matrices if p.requires_grad]
        params = [p for p in params if p.requires_grad]
        assert self._matrices, "no matrices"
        assert all(p.dim() >= 2 for p in self._matrices), \
            "FlatMuon's matrices need two axes or more"
        mine = {id(p) for p in self._matrices}
        self._rms = [p for p in params if id(p) not in mine]
        assert len(self._rms) + len(self._matrices) == len(params), \
            "every matrix must be among the parameters, once"
        super().__init__(params, lr=lr, alpha=alpha, eps=eps,
                         max_grad_norm=max_grad_norm, world_size=world_size)
        self.param_groups[0]["params"] = self._rms
        self.add_param_group(dict(
            params=self._matrices, lr=muon_lr, momentum=muon_momentum,
            ns_steps=ns_steps, alpha=alpha, eps=eps))
        # the base arena for square averages covers every parameter; the
        # matrices' part of it is their momentum
        n = self._n_rms = sum(p.numel() for p in self._rms)
        total = self.flat_param.numel()
        device = self.flat_param.device
        self.flat_momentum = self.flat_sqavg[n:]
        self.flat_update = torch.zeros(total - n, device=device)
        self.muon_lr_t = torch.zeros(1, device=device)
        self._views = []
        shape_scale = torch.empty(total - n, device=device)
        for p in reversed(self._matrices):
            off, cnt = self.slices[p]
            self._views.append(self.flat_update[off - n:off - n + cnt].view(
                p.shape[0], -1))
            rows, cols = self._views[-1].shape
            shape_scale[off - n:off - n + cnt] = max(1.0, rows / cols) ** 0.5
        self._shape_scale = shape_scale

    def _arena_order(self, params):
        return list(reversed(self._rms)) + list(reversed(self._matrices))

    def sync_lr(self):
        super().sync_lr()
        self.muon_lr_t.fill_(self.param_groups[1]["lr"])

    @torch.no_grad()
    def step_device(self):
        self.norm_sq.zero_()
        g0, g1 = self.param_groups
        n, mu = self._n_rms, g1["momentum"]
        hip = self.flat_param.is_cuda and ops.hip_available()
        if hip:
            ext = ops.ext_hip()
            ext.grad_sqnorm(self.flat_grad, self.scale_t, self.norm_sq)
            # the count of skipped steps is the first kernel's to keep
            ext.muon_momentum(self.flat_grad[n:], self.flat_momentum,
                              self.flat_update, self.norm_sq, self.scale_t,
                              self.max_grad_norm, mu, self.skip_t)
            if n:
                ext.rmsprop_update(
                    self.flat_param[:n], self.flat_grad[:n],
                    self.flat_sqavg[:n], self.lr_t, self.norm_sq,
                    self.scale_t, self.max_grad_norm, g0["alpha"],
                    g0["eps"])
        else:
            # eager path (CPU tests / escape hatch) — same math
            gr = self.flat_grad * self.scale_t
            norm = gr.norm()
            if not torch.isfinite(norm):
                self.skip_t += 1
                return
            if self.max_grad_norm > 0:
                gr = gr * torch.clamp(self.max_grad_norm / (norm + 1e-6),
                                      max=1.0)
            sq = self.flat_sqavg[:n]
            sq.mul_(g0["alpha"]).addcmul_(gr[:n], gr[:n],
                                          value=1.0 - g0["alpha"])
            self.flat_param[:n].addcdiv_(gr[:n], sq.sqrt().add_(g0["eps"]),
                                         value=-float(self.lr_t.item()))
            self.flat_momentum.mul_(mu).add_(gr[n:])
            torch.add(gr[n:], self.flat_momentum, alpha=mu,
                      out=self.flat_update)
        orthogonalize(self._views, steps=g1["ns_steps"], out=self._views)
        self.flat_update.mul_(self._shape_scale)
        self.flat_param[n:].addcmul_(self.flat_update, self.muon_lr_t,
                                     value=-1.0)

    # --- checkpoints: torch's layout, square_avg or momentum_buffer ---
    def state_dict(self):
        state, groups, i = {}, [], 0
        for k, g in enumerate(self.param_groups):
            key = "momentum_buffer" if k else "square_avg"
            ids = []
            for p in g["params"]:
                off, cnt = self.slices[p]
                state[i] = {"step": self._steps,
                            key: self.flat_sqavg[off:off + cnt]
                            .view_as(p).clone()}
                ids.append(i)
                i += 1
            groups.append({**{a: b for a, b in g.items() if a != "params"},
                           "params": ids})
        return {"state": state, "param_groups": groups}

    def load_state_dict(self, sd):
        if len(sd.get("param_groups", ())) != 2:
            raise ValueError("not a FlatMuon state: two parameter groups "
                             "expected")
        for g, old in zip(self.param_groups, sd["param_groups"]):
            if len(g["params"]) != len(old["params"]):
                raise ValueError("the state's parameters do not match")
        self._load_entries(
            sd, [(p, "momentum_buffer" if k else "square_avg")
                 for k, g in enumerate(self.param_groups)
                 for p in g["params"]])
        for g, old in zip(self.param_groups, sd["param_groups"]):
            for a in ("lr", "alpha", "eps", "momentum", "ns_steps"):
                if a in g:
                    g[a] = old.get(a, g[a])
