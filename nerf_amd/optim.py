"""Adam over one flat parameter buffer, one kernel per step.

`torch.optim.Adam` (what the reference's CLI builds, train.py:246) launches a handful of
multi-tensor kernels per step and, behind a GradScaler, makes the host wait for the inf check
before it may launch them.  This optimizer keeps the parameters, both moments and the update
count in flat device buffers and applies the same update in a single launch that also honours
the scaler's `found_inf` on the device, so a training step never waits for the host.  It plugs
into `torch.amp.GradScaler` through the protocol torch's own fused optimizers use
(`_step_supports_amp_scaling`).  Same hyper-parameters and arithmetic as `torch.optim.Adam`
(no amsgrad, no maximize); results agree to fp32 rounding.

`Muon` steps the matrices of a model along orthogonalised momentum instead and leaves the rest to
Adam; it goes wherever `Adam` does (`NeRF.fit`, `train.batch_step`, the schedulers, a GradScaler).
"""
from typing import Iterable

import torch
from torch import Tensor

from . import ops
from .distributed import flat_gradient


class Adam(torch.optim.Optimizer):
    _step_supports_amp_scaling = True

    def __init__(self, params: Iterable[Tensor], lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.0):
        if lr < 0 or eps < 0 or not (0 <= betas[0] < 1 and 0 <= betas[1] < 1) or weight_decay < 0:
            raise ValueError("invalid Adam hyper-parameters")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))
        for group in self.param_groups:
            self._flatten(group)

    def _flatten(self, group) -> None:
        """Move the group's parameters into one contiguous buffer; each parameter becomes a view."""
        params = group["params"]
        first = params[0]
        if any(not p.is_cuda or p.dtype != torch.float32 or p.device != first.device for p in params):
            raise RuntimeError("nerf_amd.optim.Adam takes fp32 parameters on one ROCm device")
        sizes = [p.numel() for p in params]
        flat = torch.cat([p.detach().reshape(-1) for p in params])
        for p, v in zip(params, flat.split(sizes)):
            p.data = v.view(p.shape)
        state = self.state[first]                       # the group's state hangs off its first parameter
        state["flat_param"] = flat
        state["sizes"] = sizes
        state["exp_avg"] = torch.zeros_like(flat)
        state["exp_avg_sq"] = torch.zeros_like(flat)
        state["step"] = torch.zeros(2, device=flat.device)          # [applied so far, scratch], swapped per call
        state["which"] = 0
        state["flat_grad"] = torch.zeros_like(flat)                 # used only when the gradients are not flat

    def _ensure_flat(self, group) -> None:
        """Parameters must still be the views made by _flatten (a later `module.to(...)`,
        `load_state_dict(assign=True)` or `p.data = ...` replaces them): if not, adopt the current
        values into the flat buffer again and keep the moments."""
        params = group["params"]
        state = self.state[params[0]]
        flat = state["flat_param"]
        ptr = flat.data_ptr()
        for p, n in zip(params, state["sizes"]):
            if p.data_ptr() != ptr or p.device != flat.device or not p.is_contiguous():
                break
            ptr += 4 * n
        else:
            return
        if any(p.device != flat.device or p.dtype != torch.float32 for p in params):
            raise RuntimeError("nerf_amd.optim.Adam: parameters moved to another device or dtype after construction")
        with torch.no_grad():
            for p, v in zip(params, flat.split(state["sizes"])):
                v.copy_(p.detach().reshape(-1))
                p.data = v.view(p.shape)

    def load_state_dict(self, state_dict) -> None:
        """As torch's, then the flat buffers go back onto the parameters' device as fp32 (a
        checkpoint read with map_location="cpu" would otherwise hand host pointers to the kernel)
        and the parameters are re-adopted as views of the loaded flat buffer's values."""
        super().load_state_dict(state_dict)
        for group in self.param_groups:
            self._adopt(group)

    def _adopt(self, group) -> None:
        params = group["params"]
        state = self.state[params[0]]
        dev = params[0].device
        for key in ("flat_param", "exp_avg", "exp_avg_sq", "step", "flat_grad"):
            state[key] = state[key].to(device=dev, dtype=torch.float32).contiguous()
        state["which"] = int(state["which"])
        state["sizes"] = [int(n) for n in state["sizes"]]
        # the live parameters (what load_state_dict of the module set) win over the saved copy
        with torch.no_grad():
            for p, v in zip(params, state["flat_param"].split(state["sizes"])):
                v.copy_(p.detach().reshape(-1))
                p.data = v.view(p.shape)

    @property
    def steps_applied(self) -> int:
        """Number of updates actually applied to the first group (synchronises)."""
        state = self.state[self.param_groups[0]["params"][0]]
        return int(state["step"][state["which"]].item())

    @torch.no_grad()
    def step_scaled(self, grad_scale: Tensor, found_inf: Tensor) -> None:
        """`scaler.unscale_(self); scaler.step(self)` (reference train.py:81-83) as one launch: the
        gradients still carry the loss scale `grad_scale` (the scaler's device float), `found_inf` is the
        device float the backward raised if a gradient was not finite (nerf_amd.amp)."""
        self._update(grad_scale, found_inf)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        found_inf = getattr(self, "found_inf", None)        # set by GradScaler.step around this call
        grad_scale = getattr(self, "grad_scale", None)      # None once unscale_ has run
        self._update(grad_scale, found_inf)
        return loss

    def _update(self, grad_scale, found_inf):
        for group in self.param_groups:
            self._update_group(group, grad_scale, found_inf)

    def _update_group(self, group, grad_scale, found_inf):
        params = group["params"]
        state = self.state[params[0]]
        if all(p.grad is None for p in params):
            return
        self._ensure_flat(group)
        grad = flat_gradient(params)
        if grad is None:                                # gradients from elsewhere: gather them
            if any(p.grad is None for p in params):
                # torch.optim.Adam leaves a parameter without a gradient untouched (moments
                # included); one flat update cannot, so say so instead of moving those weights
                raise RuntimeError("nerf_amd.optim.Adam: every parameter of a group needs a gradient "
                                   "(put frozen parameters in a group of their own or leave them out)")
            grad = state["flat_grad"]
            for p, v in zip(params, grad.split(state["sizes"])):
                v.copy_(p.grad.reshape(-1))
        scale = None if grad_scale is None else grad_scale.to(torch.float32).reshape(1)   # no copy when already fp32
        finf = None if found_inf is None else found_inf.to(torch.float32).reshape(1)
        w = state["which"]
        step = state["step"]
        ops.adam_step(state["flat_param"], grad, state["exp_avg"], state["exp_avg_sq"], group["lr"],
                      group["betas"][0], group["betas"][1], group["eps"], group["weight_decay"],
                      None, finf, step[w:w + 1], step[1 - w:2 - w], grad_scale=scale)
        state["which"] = 1 - w
        for p in params:                                # written through raw pointers: tell autograd
            torch.autograd.graph.increment_version(p)   # and the packed-weight cache of ops.ModelHandle


class Muon(Adam):
    """Momentum with orthogonalised updates for the matrices (`ops.muon_step`), Adam for everything else.

    A 2-D parameter whose smaller side is at least `MATRIX_SIDE` is a matrix: a field's hidden layers are (their
    sides are its width and its encoders'), its output heads and its biases are not.  A param group may say
    `"muon": True` or `False` to decide for all of its parameters.  Matrices of a group take one call, however
    many they are and whatever their shapes.

    `lr` applies to both kinds (the schedulers push one rate into every group): with adjust_lr="match_rms_adamw" an
    update of a matrix is as large as Adam's usual one, so an Adam rate carries over; "original" is
    lr * sqrt(max(1, rows / cols)).  `weight_decay` is decoupled for the matrices and 0 for the rest unless a group
    names its own.  Behind a GradScaler it behaves like `Adam`: nothing waits for the host."""

    MATRIX_SIDE = 16

    def __init__(self, params: Iterable[Tensor], lr: float = 5e-4, momentum: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.0, ns_coefficients=ops.NS_COEFFICIENTS, ns_steps: int = 5, ns_eps: float = 1e-7,
                 adjust_lr: str = "match_rms_adamw", betas=(0.9, 0.999), eps: float = 1e-8):
        own = dict(momentum=momentum, nesterov=nesterov, ns_coefficients=ns_coefficients, ns_steps=ns_steps, ns_eps=ns_eps,
                   adjust_lr=adjust_lr, weight_decay=weight_decay)
        self._check(own)
        groups = list(params)
        if not groups or not isinstance(groups[0], dict):
            groups = [{"params": groups}]
        split = []
        for group in groups:
            group = dict(group)
            members, kind = group.pop("params"), group.pop("muon", None)
            members = [members] if isinstance(members, Tensor) else list(members)
            tensors = [p[1] if isinstance(p, tuple) else p for p in members]                # (name, parameter) pairs stay pairs
            if kind and any(p.dim() != 2 for p in tensors):
                raise ValueError("nerf_amd.optim.Muon: a group of matrices holds 2-D parameters only")
            matrix = [p.dim() == 2 and min(p.shape) >= self.MATRIX_SIDE if kind is None else bool(kind) for p in tensors]
            if any(is_matrix and max(p.shape) > 32768 for p, is_matrix in zip(tensors, matrix)):
                raise ValueError('nerf_amd.optim.Muon: matrices have sides of up to 32768 (a group with "muon": False gets Adam\'s step)')
            for muon in (True, False):
                chosen = [p for p, is_matrix in zip(members, matrix) if is_matrix == muon]
                if chosen:
                    split.append({**(own if muon else {}), **group, "params": chosen, "muon": muon})
        for group in split:
            if group["muon"]:
                self._check(group)
        super().__init__(split, lr=lr, betas=betas, eps=eps)

    @staticmethod
    def _check(own) -> None:
        """What a group of matrices is stepped by: refused here, not in the first step."""
        if not 0 <= own["momentum"] < 1 or not own["ns_eps"] > 0 or not 0 <= own["weight_decay"] < float("inf"):
            raise ValueError("invalid Muon hyper-parameters")
        if own["adjust_lr"] not in ("original", "match_rms_adamw"):
            raise ValueError(f"unknown adjust_lr {own['adjust_lr']!r}")
        ops.check_ns_schedule(own["ns_coefficients"], own["ns_steps"], own["ns_eps"])

    def _flatten(self, group) -> None:
        if not group["muon"]:
            return super()._flatten(group)
        first = group["params"][0]
        if any(not p.is_cuda or p.dtype != torch.float32 or p.device != first.device or not p.is_contiguous()
               for p in group["params"]):
            raise RuntimeError("nerf_amd.optim.Muon takes contiguous fp32 parameters on one ROCm device")

    def load_state_dict(self, state_dict) -> None:
        """As Adam's; the momenta go back onto their parameters' device as contiguous fp32."""
        torch.optim.Optimizer.load_state_dict(self, state_dict)
        for group in self.param_groups:
            if not group["muon"]:
                self._adopt(group)
                continue
            for p in group["params"]:
                if "momentum" in self.state[p]:
                    self.state[p]["momentum"] = self.state[p]["momentum"].to(device=p.device, dtype=torch.float32).contiguous()

    @property
    def steps_applied(self) -> int:
        """Number of updates actually applied to the first group that Adam steps (synchronises)."""
        for group in self.param_groups:
            if not group["muon"]:
                state = self.state[group["params"][0]]
                return int(state["step"][state["which"]].item())
        raise RuntimeError("nerf_amd.optim.Muon counts the updates of its Adam groups, and has none")

    def _update_group(self, group, grad_scale, found_inf):
        if not group["muon"]:
            return super()._update_group(group, grad_scale, found_inf)
        params = [p for p in group["params"] if p.grad is not None]
        if not params:
            return
        for p in params:
            if "momentum" not in self.state[p]:
                self.state[p]["momentum"] = torch.zeros_like(p)
        ops.muon_step(params, [p.grad for p in params], [self.state[p]["momentum"] for p in params], lr=group["lr"],
                      momentum=group["momentum"], nesterov=group["nesterov"], weight_decay=group["weight_decay"],
                      steps=group["ns_steps"], coefficients=group["ns_coefficients"], eps=group["ns_eps"],
                      adjust_lr=group["adjust_lr"],
                      grad_scale=None if grad_scale is None else grad_scale.to(torch.float32).reshape(1),
                      found_inf=None if found_inf is None else found_inf.to(torch.float32).reshape(1))
