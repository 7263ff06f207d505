"""AdamW over all parameter tensors at once, with the clipping of their gradients by the global norm in the same call.

What the reference's update does behind its backward (ppo.py:2011-2051: ``clip_grad_norm_``, a guard against gradients that are not finite,
``optim.step``), as two launches for any number of tensors up to some hundreds; ``weight_decay=0`` is Adam.
"""

from __future__ import annotations

import math
from typing import Any, Callable, Iterable, Optional, Tuple, Union

import torch

from .. import _capi

_BLOCK = 256   # elements that share a scale of 8-bit states


class AdamW(torch.optim.Optimizer):
    """Adam with decoupled weight decay for parameters in float32, bfloat16 or float16 on one CUDA device.

        c = min(1, max_norm / (norm + 1e-6)) of the gradients' norm over all groups, g = c grad        (without max_norm: c = 1)
        m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - beta1^t) m / (sqrt(v) / sqrt(1 - beta2^t) + eps)

    computed in float32 and rounded to p's type.

    Args:
        params, lr, betas, eps, weight_decay: as ``torch.optim.AdamW`` has them.  ``lr`` may be a tensor of one number on the device, which a
            captured graph reads at every replay.
        max_norm: clip the gradients by their global norm.  The gradients themselves stay as they are; ``grad_norm`` has the norm
            of the last step, on the device.  A norm that is not finite leaves parameters and states as they were.
        state_bits: 32 (``exp_avg`` and ``exp_avg_sq`` in float32) or 8 (``exp_avg`` and ``exp_avg_sq_root``, its square root, in float8_e4m3fn
            with a float32 scale for every 256 elements; the root is rounded at random, since an average that moves by 1 - beta2 of
            the way would stand still otherwise.  The first moment is rounded to nearest and needs the noise of real gradients to follow small
            changes: with beta1 = 0.9 and the same gradient at every step it may stop a third short of it).
        seed: of those roundings; the same seed gives the same steps.

    A parameter without a gradient is left out.  The step counts stand on the device, so that steps can be captured once every parameter has its
    state: make a step first, or load one.  ``step`` writes in place, on the current stream.
    """

    def __init__(self, params: Iterable, lr: Union[float, torch.Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, max_norm: Optional[float] = None, state_bits: int = 32, seed: int = 0) -> None:
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: states have 32 or 8 bits, got {state_bits!r}")
        if max_norm is not None and not max_norm >= 0:
            raise ValueError(f"AdamW: max_norm must not be negative, got {max_norm!r}")
        self._max_norm, self._state_bits, self._seed = max_norm, state_bits, int(seed) & 0xFFFFFFFF
        self.grad_norm: Optional[torch.Tensor] = None
        self._control: Optional[torch.Tensor] = None
        self._plan = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def add_param_group(self, param_group: dict) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            self._check(group)
        except (ValueError, RuntimeError):
            self.param_groups.pop()
            raise

    @staticmethod
    def _check(group: dict) -> None:
        lr, betas = group["lr"], group["betas"]
        if not (isinstance(lr, torch.Tensor) and lr.numel() == 1) and not (isinstance(lr, (int, float)) and lr >= 0):
            raise ValueError(f"AdamW: lr must not be negative, got {lr!r}")
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError(f"AdamW: betas must be in [0, 1), got {betas!r}")
        if not (group["eps"] >= 0 and math.isfinite(group["eps"])) or not group["weight_decay"] >= 0:
            raise ValueError(f"AdamW: eps and weight_decay must not be negative, got {group['eps']!r} and {group['weight_decay']!r}")
        for p in group["params"]:
            if p.dtype not in (torch.float32, torch.bfloat16, torch.float16):
                raise ValueError(f"AdamW: parameters must be float32, bfloat16 or float16, got {p.dtype}")

    def __getstate__(self) -> dict:
        return {**super().__getstate__(), "_max_norm": self._max_norm, "_state_bits": self._state_bits, "_seed": self._seed}

    def __setstate__(self, state: dict) -> None:
        super().__setstate__(state)
        self._plan = None
        self.__dict__.setdefault("grad_norm", None)
        self.__dict__.setdefault("_control", None)

    def load_state_dict(self, state_dict: dict) -> None:
        """States of ``torch.optim.AdamW`` are taken too, by an optimizer of 32-bit states."""
        kept = {"exp_avg", "exp_avg_sq"} if self._state_bits == 32 else set(self._shapes(torch.empty(0)))
        for state in state_dict["state"].values():
            if not kept <= set(state):
                raise ValueError(f"AdamW: a state with {sorted(state)} does not fit an optimizer of {self._state_bits}-bit states")
        super().load_state_dict(state_dict)
        # the base class takes states to their parameters' types: they have types of their own here
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        params = [p for group in self.param_groups for p in group["params"]]
        for i, p in zip(ids, params):
            if i in state_dict["state"]:
                saved = state_dict["state"][i]
                state = {"step": torch.as_tensor(saved["step"], dtype=torch.float32).to(p.device, copy=True).reshape(())}
                for name, like in self._shapes(p).items():
                    state[name] = torch.empty_like(like, device=p.device).copy_(saved[name].detach().reshape(like.shape))
                self.state[p] = state

    def _shapes(self, p: torch.Tensor) -> dict:
        """Empty tensors like a parameter's state."""
        if self._state_bits == 32:
            m = torch.empty_like(p, dtype=torch.float32, device="meta", memory_format=torch.preserve_format)
            return {"exp_avg": m, "exp_avg_sq": m}
        m = torch.empty_like(p, dtype=torch.float8_e4m3fn, device="meta", memory_format=torch.preserve_format)
        scale = torch.empty((p.numel() + _BLOCK - 1) // _BLOCK, device="meta")
        return {"exp_avg": m, "exp_avg_scale": scale, "exp_avg_sq_root": m, "exp_avg_sq_root_scale": scale}

    def _new_state(self, p: torch.Tensor) -> dict:
        if not p.is_cuda:
            raise RuntimeError(f"AdamW: a parameter is on {p.device}; the kernels run on CUDA only (sm_100a) and have no CPU path")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: a captured step would clear its states at every replay; make a step, or load its states, before the capture")
        state: dict[str, Any] = {"step": torch.zeros((), dtype=torch.float32, device=p.device)}
        for name, like in self._shapes(p).items():
            state[name] = torch.zeros_like(like, device=p.device) if like.dtype == torch.float32 else \
                torch.zeros_like(like, dtype=torch.uint8, device=p.device).view(like.dtype)
        return state

    @torch.no_grad()
    def step(self, closure: Optional[Callable] = None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        norm = False if self._plan is None else self._launch()
        if norm is False:
            if not self._prepare():
                self.grad_norm = None
                return loss
            norm = self._launch()
            if norm is False:
                raise RuntimeError("AdamW: parameter groups must be lists of parameters that stay as they are during a step")
        self.grad_norm = norm
        return loss

    def _launch(self):
        return self._plan.step(self.param_groups, self.state, self._max_norm, self._seed, self._control)

    def _prepare(self) -> bool:
        """States for the parameters that have a gradient and none yet, and a plan of all; whether there is anything to do."""
        some = None
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is not None:
                    some = p if some is None else some
                    if not self.state[p]:
                        self.state[p].update(self._new_state(p))
        if some is None:
            return False
        if self._control is None or self._control.device != some.device:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW: a captured step needs a word of its own that outlives it; make a step before the capture")
            self._control = torch.zeros(1, dtype=torch.int32, device=some.device)
        self._plan = _capi.host.AdamWPlan(self.param_groups, self.state, self._state_bits)
        return True
