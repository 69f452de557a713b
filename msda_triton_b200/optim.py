"""AdamW over many tensors in one launch, with moments in fp32 or in 8 bits.

    m = beta1 m + (1 - beta1) g,   v = beta2 v + (1 - beta2) g^2
    p = p (1 - lr wd) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)

`AdamW` is the optimizer; `adamw_step` the step as a function of its tensors.
Runs in the sm_100a kernel of libmsda_b200.so (msda_adamw_step); there is no
CPU fallback.
"""

from __future__ import annotations

import copy
from collections.abc import Sequence

import torch
from torch import Tensor

from msda_triton_b200 import _core, _lib

# Elements of 8-bit moments that share an exponent; each tensor's states start
# at a multiple of it, in fp32 too.
BLOCK = 128


def _padded(n: int) -> int:
    return -(-n // BLOCK) * BLOCK


def adamw_state(params: Sequence[Tensor], bits: int = 32, master: bool = False
                ) -> dict[str, Tensor]:
    """Zero moments for `params` (all of one dtype and device), as adamw_step takes them.

    One flat tensor per kind, in which tensor i's states start at the sum of
    the earlier tensors' sizes, each rounded up to 128: "exp_avg" and
    "exp_avg_sq", fp32 or (bits = 8) uint8 codes with "exp_avg_exponent" and
    "exp_avg_sq_exponent", a byte for every 128; with `master`, "master" holds
    fp32 copies of 16-bit parameters."""
    if bits not in (8, 32):
        raise ValueError(f"states of 32 or 8 bits expected, got {bits}")
    _one_kind(params)
    if master and params and params[0].dtype == torch.float32:
        raise ValueError("fp32 parameters take no master copy")
    n = sum(_padded(p.numel()) for p in params)
    device = params[0].device if params else None
    state = {}
    for name in ("exp_avg", "exp_avg_sq"):
        dt = torch.float32 if bits == 32 else torch.uint8
        state[name] = torch.zeros(n, device=device, dtype=dt)
        if bits == 8:
            state[name + "_exponent"] = torch.zeros(n // BLOCK, device=device, dtype=dt)
    if master:
        state["master"] = torch.zeros(n, device=device, dtype=torch.float32)
        at = 0
        for p in params:
            _flat(state["master"], at, p).copy_(p.detach())
            at += _padded(p.numel())
    return state


def _flat(t: Tensor, at: int, p: Tensor) -> Tensor:
    """The part of a state tensor that belongs to p, in p's shape and memory order."""
    return t.as_strided(p.shape, p.stride(), at)


def _one_kind(params: Sequence[Tensor]) -> None:
    if not params:
        return
    dtype = params[0].dtype
    if not params[0].is_cuda:
        raise ValueError("AdamW requires CUDA tensors. Got CPU tensors instead.")
    if dtype not in _core._DTYPE_CODE:
        raise NotImplementedError(f"AdamW only supports fp32, fp16, and bf16. Got {dtype}.")
    if any(p.dtype != dtype or p.device != params[0].device for p in params):
        raise ValueError("the tensors of a step must share their dtype and device")


def _is_dense(p: Tensor) -> bool:
    """Whether p's elements fill one range of memory, in any order of its axes."""
    expect = 1
    for stride, n in sorted((s, n) for s, n in zip(p.stride(), p.shape) if n > 1):
        if stride != expect:
            return False
        expect *= n
    return True


def _order(shape, strides) -> list[int]:
    """What tells one order of a dense tensor's elements in memory from another: its strides,
    but those of axes of one element, which are arbitrary."""
    return [s for s, n in zip(strides, shape) if n > 1]


# Elements of a parameter for each element of a state.
_SIZES = {"exp_avg": 1, "exp_avg_sq": 1, "exp_avg_exponent": BLOCK, "exp_avg_sq_exponent": BLOCK,
          "master": 1}


def adamw_step(params: Sequence[Tensor], grads: Sequence[Tensor | None],
               state: dict[str, Tensor], *, step: int | Sequence[int], lr: float = 1e-3,
               betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, seed: int = 0,
               grad_scale: Tensor | None = None) -> None:
    """One AdamW step in place over `params` and `state`.

    Args:
        params: CUDA tensors of one dtype (fp32, fp16, bf16) and device, each
            filling one range of memory.
        grads: a gradient of the same dtype and shape for each, or None: that
            tensor and its states stay as they are.
        state: adamw_state(params, ...).
        step: t of the bias corrections, from 1: one number, or one per tensor.
        lr, betas, eps, weight_decay: as in the formula above.
        seed: of the random rounding of 8-bit states; the bits follow from the
            seed, the step and the element's place.
        grad_scale: one fp32 value on the device that multiplies the gradients
            (the inverse of a loss scale, or a clipping factor); None: 1.

    Raises:
        ValueError: CPU tensors, sizes, dtypes or states that do not fit.
        NotImplementedError: dtype other than fp32/fp16/bf16.
        RuntimeError: under CUDA graph capture, where `step` would be frozen.
    """
    _lib.binding().adamw_step(params, grads, state, step, lr, betas[0], betas[1], eps,
                              weight_decay, seed & 0xFFFFFFFF, grad_scale, None)


def adamw_state_values(state: dict[str, Tensor]) -> tuple[Tensor, Tensor]:
    """(exp_avg, exp_avg_sq) that a state stands for, flat as the state is.
    8-bit moments come as bf16, which holds them exactly; fp32 ones as they are."""
    return _lib.binding().adamw_values(state)


# What torch's Adam family keeps in its groups for other updates than this one.
_OTHER_UPDATES = ("maximize", "amsgrad", "decoupled_weight_decay")


def _refuse_other_updates(group: dict) -> None:
    """ValueError for a group that asks for another update than AdamW's."""
    for key in ("maximize", "amsgrad"):
        if group.get(key):
            raise ValueError(f"AdamW has no {key}: a group with {key}=True is another update")
    if not group.get("decoupled_weight_decay", True) and group.get("weight_decay", 0) != 0:
        raise ValueError("a group with decoupled_weight_decay=False and a weight_decay of "
                         f"{group['weight_decay']} is another update than AdamW's")


class _Part:
    """The parameters of one group that share a dtype and device, and their states."""

    def __init__(self, params: list[Tensor], bits: int, master: bool) -> None:
        for p in params:
            if not _is_dense(p):
                raise ValueError("a parameter's elements must fill one range of memory, got "
                                 f"strides {p.stride()} for {tuple(p.shape)}")
        self.params = params
        master = master and params[0].dtype != torch.float32
        self.state = adamw_state([p.detach() for p in params], bits, master)
        self.steps = [0] * len(params)
        # the order of the states' elements, which a step holds its parameters to
        self.layouts = [torch.empty_strided(p.shape, p.stride(), device="meta") for p in params]

    def own(self, i: int, at: int) -> dict[str, Tensor]:
        """Parameter i's part of each state tensor."""
        p, n = self.params[i], _padded(self.params[i].numel())
        out = {}
        for name, t in self.state.items():
            size = _SIZES[name]
            flat = t.dtype == torch.uint8
            out[name] = (t[at // size:(at + n) // size] if flat else _flat(t, at, p))
        return out

    def places(self) -> list[int]:
        at, out = 0, []
        for p in self.params:
            out.append(at)
            at += _padded(p.numel())
        return out


class AdamW(torch.optim.Optimizer):
    """AdamW whose step is one launch per parameter group, dtype and device.

    Args:
        params, lr, betas, eps, weight_decay: as torch.optim.AdamW; groups may
            differ in them.
        state_bits: 32, or 8: moments in one byte each, with random rounding.  128
            neighbouring elements share a range, 2^15 for the first moment and 2^31
            for the second; below it the first is zero (no momentum where a gradient
            stays that far below a neighbour's) and the second the range's end.
        master_weights: keep fp32 copies of 16-bit parameters, which the step
            updates and rounds into the parameters.
        seed: of the 8-bit states' rounding.

    Parameters without a gradient are skipped, and count their own steps.  A
    state_dict of torch.optim.AdamW can be loaded where state_bits is 32; an
    8-bit one holds the codes and exponents themselves, and loads where the
    parameters lie in memory in the same order.  A group that asks for
    another update (maximize, amsgrad, a decay that is not decoupled) is a
    ValueError.  `step` cannot be captured in a CUDA graph.
    """

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, *, state_bits: int = 32,
                 master_weights: bool = False, seed: int = 0) -> None:
        if state_bits not in (8, 32):
            raise ValueError(f"states of 32 or 8 bits expected, got {state_bits}")
        if lr < 0 or eps < 0 or weight_decay < 0:
            raise ValueError("lr, eps and weight_decay must not be negative, got "
                             f"{lr}, {eps}, {weight_decay}")
        if not all(0 <= b < 1 for b in betas):
            raise ValueError(f"betas must lie in [0, 1), got {betas}")
        self.state_bits, self.master_weights, self.seed = state_bits, master_weights, seed
        self._parts: list[list[_Part]] = []
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def __getstate__(self):
        return {**super().__getstate__(), "state_bits": self.state_bits, "seed": self.seed,
                "master_weights": self.master_weights, "_parts": self._parts}

    def add_param_group(self, param_group: dict) -> None:
        """As torch.optim.Optimizer's."""
        _refuse_other_updates({**self.defaults, **param_group})
        super().add_param_group(param_group)

    def _allocate(self) -> None:
        """States for groups that have none yet (the first step, or a group added later)."""
        for group in self.param_groups[len(self._parts):]:
            kinds: dict[tuple, list[Tensor]] = {}
            for p in group["params"]:
                kinds.setdefault((p.dtype, p.device), []).append(p)
            parts = [_Part(ps, self.state_bits, self.master_weights) for ps in kinds.values()]
            self._parts.append(parts)
            for part in parts:
                for i, at in enumerate(part.places()):
                    p = part.params[i]
                    self.state[p] = {"step": 0, **part.own(i, at)}
                    if self.state_bits == 8:
                        self.state[p]["strides"] = p.stride()

    @torch.no_grad()
    def step(self, closure=None):
        """One step; returns the closure's loss, if one is given."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._allocate()
        for group, parts in zip(self.param_groups, self._parts):
            for part in parts:
                grads = [p.grad for p in part.params]
                if all(g is None for g in grads):
                    continue
                steps = [s + (g is not None) for s, g in zip(part.steps, grads)]
                _lib.binding().adamw_step(part.params, grads, part.state,
                                          [max(s, 1) for s in steps], group["lr"],
                                          *group["betas"], group["eps"], group["weight_decay"],
                                          self.seed & 0xFFFFFFFF, None, part.layouts)
                part.steps = steps
        return loss

    def state_dict(self):
        """As torch.optim.Optimizer's; parameters that never took a step have no state."""
        for parts in self._parts:
            for part in parts:
                for p, s in zip(part.params, part.steps):
                    self.state[p]["step"] = s
        saved = super().state_dict()
        saved["state"] = {i: s for i, s in saved["state"].items() if s["step"] > 0}
        return saved

    def load_state_dict(self, state_dict) -> None:
        """Hyperparameters and states of a state_dict of this optimizer's (or, with 32-bit
        states, of torch.optim.AdamW's) over the same parameters.  Every key of a group is
        taken over."""
        state_dict = state_dict.copy()
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            replaced = hook(self, state_dict)
            state_dict = state_dict if replaced is None else replaced
        groups = state_dict["param_groups"]
        for group in groups:
            _refuse_other_updates(group)
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("the state_dict's parameter groups differ from the optimizer's")
        self._allocate()
        place = {id(p): (part, i, at) for parts in self._parts for part in parts
                 for i, (p, at) in enumerate(zip(part.params, part.places()))}
        todo = []
        for saved, group in zip(groups, self.param_groups):
            for index, p in zip(saved["params"], group["params"]):
                part, i, at = place[id(p)]
                own, got = part.own(i, at), state_dict["state"].get(index)
                if got is not None:
                    # codes are in the order of their parameter's elements in memory
                    if self.state_bits == 8 and _order(p.shape, p.stride()) != _order(
                            p.shape, got.get("strides", p.stride())):
                        raise ValueError(f"8-bit states of strides {got['strides']} for a "
                                         f"parameter {tuple(p.shape)} of strides {p.stride()}")
                    for name, t in own.items():
                        if name not in got and name == "master":
                            got = {**got, "master": p.detach()}
                        if name not in got:
                            raise ValueError(f"the state_dict has no {name!r} for a parameter "
                                             f"{tuple(p.shape)}")
                        v = got[name]
                        if v.shape != t.shape or ((v.dtype == torch.uint8)
                                                  != (t.dtype == torch.uint8)):
                            raise ValueError(f"{name!r} is {v.dtype} {tuple(v.shape)} where "
                                             f"{t.dtype} {tuple(t.shape)} is needed")
                todo.append((part, i, own, got, p))
        for part, i, own, got, p in todo:
            part.steps[i] = 0 if got is None else int(got["step"])
            for name, t in own.items():
                if got is not None:
                    t.copy_(got[name])
                elif name == "master":
                    t.copy_(p.detach())
                else:
                    t.zero_()
        for saved, group in zip(groups, self.param_groups):
            group.update((key, copy.deepcopy(value)) for key, value in saved.items()
                         if key not in ("params", "param_names", *_OTHER_UPDATES))
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)


__all__ = ["AdamW", "adamw_step", "adamw_state", "adamw_state_values"]
