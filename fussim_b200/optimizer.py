"""The AdamW step over many tensors at once, after the loss's backward pass.

* ``adamw_step_``: one step of lists of tensors, with moments in 32 bits or in 8 and the clipping
  of ``clip_grad_norm_`` on the way.
* ``AdamW``: the same as a ``torch.optim.Optimizer``, with ``torch.optim.AdamW``'s settings, states
  and state dicts.

Hand-written sm_100a kernels without a CPU path. The reference (OpsiClear/fussim) has no
counterpart of these; users pair its loss with torch's optimisers, whose definition is kept.
"""

from __future__ import annotations

from itertools import chain
from typing import Iterable, Optional, Tuple, Union

import torch

from .functional import _ensure_cuda_extension
from .training import grad_norm


def adamw_step_(
    params: Iterable[torch.Tensor],
    grads: Iterable[torch.Tensor],
    exp_avgs: Iterable[torch.Tensor],
    exp_avg_sqs: Iterable[torch.Tensor],
    scales: Optional[Iterable[torch.Tensor]] = None,
    *,
    step: Union[int, torch.Tensor],
    lr: Union[float, torch.Tensor],
    betas: Tuple[float, float] = (0.9, 0.999),
    eps: float = 1e-8,
    weight_decay: float = 1e-2,
    maximize: bool = False,
    max_norm: Optional[float] = None,
    norm: Optional[torch.Tensor] = None,
    copies: Optional[Iterable[torch.Tensor]] = None,
    seed: int = 0,
) -> Optional[torch.Tensor]:
    """One AdamW step of many tensors, in place, in one launch for up to 448 of them.

    With g a gradient (negated where ``maximize``)::

        m = beta1 * m + (1 - beta1) * g            v = beta2 * v + (1 - beta2) * g^2
        p = (1 - lr * weight_decay) * p
            - lr / (1 - beta1^step) * m / (sqrt(v / (1 - beta2^step)) + eps)

    in FP32, p rounded once to its type. ``params`` are dense CUDA tensors of one device, float32,
    float16 or bfloat16; ``grads`` have their parameter's type or float32 (beside a float32
    parameter also a 16-bit type). ``copies`` are 16-bit tensors that get float32 parameters
    rounded: the weights that a mixed-precision model computes with.

    ``exp_avgs`` and ``exp_avg_sqs`` hold m and v: float32 tensors, or float8_e4m3fn ones, all
    with their parameter's shape and strides. Those of 8 bits hold codes of m and of the root of v,
    and ``scales`` a float32 tensor (blocks, 2) for each parameter: column 0 for m, 1 for the
    root, a row for each 256 numbers in the order of memory. A code stands for itself times its
    scale, which is the block's largest finite number (at least 2^-100) / 448. A number goes to
    one of its two neighbouring codes at random, in proportion (below 2^-6 scales to the nearest),
    so that slow changes are kept on average; a root that is not zero is held as 2^-6 scales at
    least; an infinite or NaN moment as NaN. The random bits are a hash of ``seed``, ``step``, the
    tensor's position in the list and the number's in its tensor.

    ``max_norm`` multiplies the gradients by min(1, max_norm / (norm + 1e-6)) on their way in
    (``grads`` stay as they are) and returns the norm, that of all ``grads`` unless ``norm`` (one
    float32 on the device) gives it; NaN makes everything NaN. Without it the result is None.
    ``step`` counts from 1; it and ``lr`` may be one float32 on the device, for captured graphs:
    they are then read when the work runs. No host synchronisation; results repeat bit for bit.
    Tensors that are written must not share memory with any other: ValueError. A gradient whose
    strides are not its parameter's is copied once more. Not differentiable; tracing raises
    RuntimeError.
    """
    as_list = lambda v: None if v is None else list(v)  # noqa: E731
    return _ensure_cuda_extension().adamw_step_(
        list(params), list(grads), list(exp_avgs), list(exp_avg_sqs), as_list(scales), step, lr,
        betas[0], betas[1], eps, weight_decay, maximize, max_norm, norm, as_list(copies), seed
    )


def adamw_moments(
    param: torch.Tensor, bits: int = 32
) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """(exp_avg, exp_avg_sq, scales) of a parameter before its first step, for ``adamw_step_``: zeros
    of its shape and strides, float32 (and no scales), or codes of 8 bits with their scales."""
    if bits not in (32, 8):
        raise ValueError(f"bits must be 32 or 8, got {bits}")
    moment = torch.float32 if bits == 32 else torch.float8_e4m3fn
    first, second = (torch.zeros_like(param, dtype=moment, memory_format=torch.preserve_format,
                                      requires_grad=False) for _ in range(2))
    if bits == 32:
        return first, second, None
    return first, second, torch.zeros(-(-param.numel() // 256), 2, device=param.device, dtype=torch.float32)


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` by ``adamw_step_``: a launch for each group of parameters (for each count of
    steps in it, where some have had fewer gradients than others).

    ``state_bits`` 8 keeps both moments in 8 bits (2 bytes a number and 8 a block of 256, instead of
    8 bytes a number); their rounding draws on ``seed``. ``master_weights`` keeps a float32 copy of
    16-bit parameters, which the step updates and rounds into the parameter. ``max_norm`` clips by
    the norm of all gradients together on the way, without writing to them; ``grad_norm`` is then
    the last step's norm, a 0-d tensor. ``capturable`` keeps the count of steps on the device, one
    for each group, and steps may be captured in a CUDA graph after a first one that makes the
    states (``lr`` may then be a 0-d float32 CUDA tensor; other captures raise RuntimeError); a
    parameter that gets its first gradient late counts with its group.

    States are named as torch's (``step``, ``exp_avg``, ``exp_avg_sq``; ``scales`` and ``master``
    besides), and 32-bit states go into and out of torch's optimiser by their state dicts. State
    dicts keep the states' own types. Sparse gradients, amsgrad and parameters that do not fill
    their memory raise an error.
    """

    def __init__(
        self,
        params,
        lr: Union[float, torch.Tensor] = 1e-3,
        betas: Tuple[float, float] = (0.9, 0.999),
        eps: float = 1e-8,
        weight_decay: float = 1e-2,
        *,
        maximize: bool = False,
        capturable: bool = False,
        state_bits: int = 32,
        master_weights: bool = False,
        max_norm: Optional[float] = None,
        seed: int = 0,
    ):
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits must be 32 or 8, got {state_bits}")
        if isinstance(lr, torch.Tensor) and not capturable:
            raise ValueError("lr as a tensor goes with capturable")
        if not isinstance(lr, torch.Tensor) and not lr >= 0.0:
            raise ValueError(f"lr must not be negative, got {lr}")
        if max_norm is not None and not max_norm >= 0.0:
            raise ValueError(f"max_norm must not be negative, got {max_norm}")
        if not 0 <= seed < 1 << 32:
            raise ValueError(f"seed must be from 0 to 2^32 - 1, got {seed}")
        for name, beta in zip(("first", "second"), betas):
            if not 0.0 <= beta < 1.0:
                raise ValueError(f"the {name} of betas must be at least 0 and below 1, got {beta}")
        for name, value in (("eps", eps), ("weight_decay", weight_decay)):
            if not value >= 0.0:
                raise ValueError(f"{name} must not be negative, got {value}")
        self.state_bits = state_bits
        self.master_weights = master_weights
        self.max_norm = max_norm
        self.seed = seed
        self.grad_norm: Optional[torch.Tensor] = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                                      maximize=maximize, capturable=capturable))

    def _first_state(self, p, count):
        first, second, scales = adamw_moments(p, self.state_bits)
        state = dict(step=count, exp_avg=first, exp_avg_sq=second)
        if scales is not None:
            state["scales"] = scales
        if self.master_weights and p.dtype != torch.float32:
            state["master"] = p.detach().float()
        return state

    def _count(self, group, device):
        """A capturable group's count of steps: the tensor that its parameters' states share; None of another."""
        for q in group["params"]:
            state = self.state.get(q)
            if state:
                if isinstance(state["step"], torch.Tensor) != bool(group["capturable"]):
                    self._settle()  # (the setting has changed since)
                return state["step"] if group["capturable"] else None
        return torch.zeros((), device=device, dtype=torch.float32) if group["capturable"] else None

    @torch.no_grad()
    def step(self, closure=None):
        """One step; the closure's result, if one is given. Without any gradient nothing is done. What may be
        refused is refused before any parameter, state or count changes."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        calls, grads, new, counts = [], [], {}, []
        for group in self.param_groups:
            if group.get("amsgrad"):
                raise ValueError("amsgrad is not supported")
            batches = {}  # by count of steps, device, and whether there are 32-bit copies
            count = None  # a capturable group's
            seen = False
            for p in group["params"]:
                grad = p.grad
                if grad is None:
                    continue
                state = self.state.get(p)
                if not seen:
                    seen = True
                    if group["capturable"] or not state or type(state["step"]) is not int:
                        count = self._count(group, p.device)
                    if count is not None:
                        counts.append(count)
                if not state:
                    state = new[p] = self._first_state(p, 0 if count is None else count)
                step = state["step"] + 1 if count is None else count
                key = (step if count is None else 0, "master" in state, p.device)
                _, params, states = batches.setdefault(key, (step, [], []))
                params.append(p)
                states.append(state)
                grads.append(grad)
            calls.extend((group, key[1], *batch) for key, batch in batches.items())
        if not calls:
            return loss
        norm = grad_norm(grads) if self.max_norm is not None else None
        ready = _ensure_cuda_extension().AdamWStep
        steps = []
        for call, (group, master, step, params, states) in enumerate(calls):
            beta1, beta2 = group["betas"]
            steps.append(ready(
                [s["master"] for s in states] if master else params, [p.grad for p in params],
                [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states],
                [s["scales"] for s in states] if self.state_bits == 8 else None,
                step, group["lr"], beta1, beta2, group["eps"], group["weight_decay"], group["maximize"],
                self.max_norm, norm, params if master else None,
                # (tensors of different calls draw different numbers)
                (self.seed + 0x9E3779B1 * call) & 0xFFFFFFFF,
            ))
        # (replays would take one count again and again, or begin with states of zeros each)
        if (new or len(counts) < len(self.param_groups)) and torch.cuda.is_current_stream_capturing():
            if any(not group["capturable"] for group, *_ in calls):
                raise RuntimeError("a step that is captured in a CUDA graph goes with capturable")
            if new:
                raise RuntimeError("the states have to be made by a step before the captured one")
        if new:
            self.state.update(new)
        self.grad_norm = norm
        for count in counts:
            count += 1
        for checked, (group, _, step, _, states) in zip(steps, calls):
            checked.run()
            if not group["capturable"]:
                for state in states:
                    state["step"] = step
        return loss

    def _check_saved(self, saved):
        """Refuses a state dict whose states do not fit the parameters."""
        for theirs, ours in zip(saved["param_groups"], self.param_groups):
            states = [(p, saved["state"].get(k)) for k, p in zip(theirs["params"], ours["params"])]
            states = [(p, s) for p, s in states if s]
            for p, state in states:
                if (state["exp_avg"].dtype == torch.float8_e4m3fn) != (self.state_bits == 8):
                    raise ValueError(f"the state dict's moments are not of {self.state_bits} bits")
                for name in ("exp_avg", "exp_avg_sq", "master"):
                    t = state.get(name)
                    if t is None and name == "master":
                        continue
                    if t.shape != p.shape:
                        raise ValueError(f"{name} must have its parameter's shape {tuple(p.shape)}, got {tuple(t.shape)}")
                    if t.dtype == torch.float8_e4m3fn and t.stride() != p.stride():
                        raise ValueError("codes of 8 bits go with parameters of the strides they were made for")
                blocks = -(-p.numel() // 256)
                if self.state_bits == 8 and ("scales" not in state or state["scales"].shape != (blocks, 2)):
                    raise ValueError(f"moments of 8 bits need their scales, of shape ({blocks}, 2)")
            if theirs.get("capturable") and len({int(s["step"]) for _, s in states}) > 1:
                raise ValueError("a capturable group's parameters must have had the same number of steps")

    def load_state_dict(self, state_dict):
        """As torch's, but states keep their types (torch's casts them to the parameters'). One that does not
        fit the parameters raises ValueError and changes nothing."""
        saved = state_dict
        self._check_saved(saved)
        ids = list(chain.from_iterable(g["params"] for g in saved["param_groups"]))
        super().load_state_dict(saved)
        own = list(chain.from_iterable(g["params"] for g in self.param_groups))
        for k, p in zip(ids, own):
            state = saved["state"].get(k)
            if not state:
                continue
            mine = self.state[p]
            for name in ("exp_avg", "exp_avg_sq", "scales", "master"):
                if name not in state:
                    continue
                t = state[name].detach()
                if name in ("exp_avg", "exp_avg_sq", "master"):
                    wide = torch.float8_e4m3fn if name != "master" and self.state_bits == 8 else torch.float32
                    mine[name] = torch.empty_like(p, dtype=wide, requires_grad=False).copy_(t)
                else:
                    mine[name] = torch.empty_like(t, device=p.device, dtype=torch.float32).copy_(t)
            if self.master_weights and p.dtype != torch.float32 and "master" not in state:
                mine["master"] = p.detach().float()
        self._settle()

    def __getstate__(self):
        names = ("state_bits", "master_weights", "max_norm", "seed", "grad_norm")
        return {**super().__getstate__(), **{k: getattr(self, k) for k in names}}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._settle()

    def _settle(self):
        """Counts of steps as this class keeps them: whole numbers, or a group's tensor."""
        for group in self.param_groups:
            group.setdefault("maximize", False)
            group.setdefault("capturable", False)
            states = [(p, self.state[p]) for p in group["params"] if self.state.get(p)]
            counts = [int(s["step"]) for _, s in states]
            if group["capturable"] and states:
                if min(counts) != max(counts):
                    raise ValueError("a capturable group's parameters must have had the same number of steps")
                count = torch.full((), float(counts[0]), device=states[0][0].device, dtype=torch.float32)
                counts = [count] * len(states)
            for (_, s), count in zip(states, counts):
                s["step"] = count
