"""AdamW over many tensors at once, its moments in 32 or in 8 bits, and the global gradient-norm clip
(lpg_adamw, lpg_adamw8, lpg_grad_norm).

``AdamW`` is the optimizer (``make_optimizer(model, "adamw")`` / ``"adamw8"``, the command line's ``--opt``);
``adamw_step`` / ``adamw_step_8bit`` / ``clip_scale`` are its steps as functions, on lists of tensors.  Every
tensor of a call is updated in one launch (a few where there are very many), in place, on the current
stream, with no host synchronisation: the clip's factor stays on the device.

8-bit moments: per parameter ``m8`` and ``r8`` (torch.float8_e4m3fn, the parameter's shape) hold the first
moment and the root of the second, each block of 256 consecutive elements times an fp32 scale
(``m_scale`` / ``r_scale``): 2.06 bytes a number instead of 8.  Rounding is random, from a counter hash of
(seed, step, the tensor's place in the list, element): the same call gives the same bits.  The argument
checks and the tables of pointers are C++ (csrc/host.cpp).
"""
from __future__ import annotations

import torch
from torch import Tensor

from . import _lib

BLOCK = 256  # elements that share a scale
_F8 = torch.float8_e4m3fn


def rounding_keys(places, step: int, seed: int) -> list[int]:
    """The rounding key of the tensors at these places of the list, for one step (an 8-bit step's random bits
    are the hash of key ^ element)."""
    return [_lib.host().rounding_key(t, step, seed) for t in places]


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, step: int, lr: float = 1e-3, betas=(0.9, 0.999),
               eps: float = 1e-8, weight_decay: float = 1e-2, grad_scale: Tensor | None = None) -> None:
    """One AdamW step (number ``step``, from 1) over lists of contiguous tensors, in place.  params and grads
    float32 or bfloat16 (one type a call), the moments float32; the update is computed in fp32 and rounded
    once.  ``grad_scale``: a device scalar every gradient is multiplied by (``clip_scale``).  No tensor
    that is written may overlap another of the call, ``grad_scale`` among them (refused); gradients may share
    memory."""
    _lib.host().adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, lr, betas, eps, weight_decay, grad_scale, False)


def adamw_step_8bit(params, grads, m8, m_scales, r8, r_scales, *, step: int, seed: int = 0, lr: float = 1e-3,
                    betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                    grad_scale: Tensor | None = None, places=None) -> None:
    """``adamw_step`` with 8-bit moments: per parameter m8 / r8 (float8_e4m3fn, its size) and m_scales /
    r_scales (float32, one a block of 256 elements), all zero before the first step.  ``places``: the tensors'
    places in the rounding's numbering (default 0, 1, ...), for a call on part of a model's list."""
    _lib.host().adamw_step_8bit(params, grads, m8, m_scales, r8, r_scales, places, seed, step, lr, betas, eps,
                                weight_decay, grad_scale, False)


def clip_scale(grads, max_norm: float) -> tuple[Tensor, Tensor]:
    """(norm, scale): the 2-norm of all gradients together and min(1, max_norm / (norm + 1e-6)), the factor
    torch.nn.utils.clip_grad_norm_ would multiply them by -- device scalars, for ``grad_scale``; the gradients
    stay as they are.  Summed in fp64 in a fixed order.  A NaN or an infinity among the gradients shows in the
    norm, and the scaled gradients are then NaN or zero, as there."""
    return _lib.host().clip_scale(grads, max_norm)


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update on the kernels above.  ``state_bits``: 32 (state names and types as torch's,
    whose state dicts it loads, but for ``maximize`` and ``amsgrad``, which are refused) or 8;
    ``max_grad_norm``: clip the gradients' global 2-norm inside the step (the stored gradients are not
    changed; ``last_norm`` is the norm before the clip, a device scalar), over all parameters of the
    optimizer, which then must share a type and a device; ``seed``: of the 8-bit rounding.

    Parameters float32 or bfloat16, contiguous, on HIP devices, gradients dense.  The step number is a host
    number, so ``step()`` refuses to be captured into a graph."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 state_bits: int = 32, max_grad_norm: float | None = None, seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError(f"lpgnn AdamW: state_bits must be 8 or 32, got {state_bits}")
        if max_grad_norm is not None and not max_grad_norm >= 0:
            raise ValueError(f"lpgnn AdamW: max_grad_norm must not be negative, got {max_grad_norm}")
        if not 0 <= int(seed) < 1 << 64:
            raise ValueError(f"lpgnn AdamW: seed must be a whole number of 64 bits, got {seed}")
        adamw_step([], [], [], [], step=1, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay)  # (checks them)
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))
        self.state_bits, self.max_grad_norm, self.seed = int(state_bits), max_grad_norm, int(seed)
        self.last_norm = None

    def __getstate__(self) -> dict:  # (torch's holds the groups and the state; __setstate__ takes whatever is in it)
        own = {k: getattr(self, k) for k in ("state_bits", "max_grad_norm", "seed", "last_norm")}
        return {**super().__getstate__(), **own}

    @staticmethod
    def _refuse_others(groups) -> None:
        """torch's options that make another update of it, which groups and state dicts may carry."""
        for g in groups:
            for k in ("maximize", "amsgrad"):
                if g.get(k):
                    raise RuntimeError(f"lpgnn AdamW: {k} is not supported")

    def add_param_group(self, param_group) -> None:
        self._refuse_others([param_group])
        super().add_param_group(param_group)

    def _init(self, p: Tensor) -> dict:
        zeros = lambda n, dt: torch.zeros(n, dtype=dt, device=p.device)
        if self.state_bits == 32:
            return dict(step=0, exp_avg=zeros(p.shape, torch.float32), exp_avg_sq=zeros(p.shape, torch.float32))
        nb = -(-p.numel() // BLOCK)
        f8 = lambda: zeros(p.shape, torch.uint8).view(_F8)
        return dict(step=0, m8=f8(), m_scale=zeros(nb, torch.float32), r8=f8(), r_scale=zeros(nb, torch.float32))

    @torch.no_grad()
    def step(self, closure=None):
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("lpgnn AdamW: step() cannot be captured into a graph (its step number would not advance)")
        self._refuse_others(self.param_groups)
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        place, calls, grads = 0, {}, []
        for gi, group in enumerate(self.param_groups):
            for p in group["params"]:
                place += 1
                if p.grad is None:
                    continue
                if p.grad.layout != torch.strided:
                    raise RuntimeError("lpgnn AdamW: sparse gradients are not supported")
                st = self.state[p]
                if not st:
                    st.update(self._init(p))
                if ("m8" in st) != (self.state_bits == 8):
                    raise RuntimeError(f"lpgnn AdamW: the state holds {8 if 'm8' in st else 32}-bit moments, "
                                       f"state_bits is {self.state_bits}")
                g = p.grad if p.grad.is_contiguous() else p.grad.contiguous()
                grads.append(g)
                # one launch per group, type, device and step number
                calls.setdefault((gi, p.dtype, p.device, int(st["step"]) + 1), []).append((p, g, st, place - 1))
        scale = None

        def update(key, items, check_only):
            group, step = self.param_groups[key[0]], key[3]
            ps, gs, sts, places = zip(*items)
            of = lambda k: [s[k] for s in sts]
            hyper = (step, float(group["lr"]), group["betas"], group["eps"], group["weight_decay"], scale, check_only)
            if self.state_bits == 32:
                _lib.host().adamw_step(ps, gs, of("exp_avg"), of("exp_avg_sq"), *hyper)
            else:
                _lib.host().adamw_step_8bit(ps, gs, of("m8"), of("m_scale"), of("r8"), of("r_scale"), places, self.seed,
                                            *hyper)
            if not check_only:
                for s in sts:
                    s["step"] = step

        if len(calls) > 1:  # no parameter is updated where another's call is refused (one call checks all of its own)
            for key, items in calls.items():
                update(key, items, True)
        if self.max_grad_norm is not None and grads:
            self.last_norm, scale = clip_scale(grads, self.max_grad_norm)
        for key, items in calls.items():
            update(key, items, False)
        return loss

    def load_state_dict(self, state_dict) -> None:
        """As torch's, but the moments keep their own types (torch would cast them to the parameter's): the 8-bit
        codes, and fp32 for everything else, whatever the saved optimizer kept it in."""
        self._refuse_others(state_dict["param_groups"])
        super().load_state_dict(state_dict)
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(saved, (p for g in self.param_groups for p in g["params"])):
            for k, v in state_dict["state"].get(i, {}).items():
                if k == "step":
                    self.state[p][k] = int(v)
                elif isinstance(v, Tensor):
                    dt = v.dtype if v.dtype == _F8 else torch.float32
                    self.state[p][k] = v.to(device=p.device, dtype=dt, copy=True).contiguous()
