"""AdamW over many tensors in one launch, with moments in fp32 or in 8 bits.

    m = beta1 m + (1 - beta1) g,   v = beta2 v + (1 - beta2) g^2
    p = p (1 - lr wd) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)

`AdamW` is the optimizer; `adamw_step` the step as a function of its tensors.
Runs in the sm_100a kernel of libmsda_b200.so (msda_adamw_step); there is no
CPU fallback.
"""

from __future__ import annotations

from array import array
from collections.abc import Sequence
from operator import attrgetter, eq

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


_dtype_of, _shape_of = attrgetter("dtype"), attrgetter("shape")


def _one_kind(params: Sequence[Tensor]) -> None:
    if not params:
        return
    dtype = params[0].dtype
    if not params[0].is_cuda:
        raise ValueError("AdamW requires CUDA tensors. Got CPU tensors instead.")
    if dtype not in _core._DTYPE_CODE:
        raise NotImplementedError(f"AdamW only supports fp32, fp16, and bf16. Got {dtype}.")
    if len(set(map(_dtype_of, params))) > 1 or len(set(map(Tensor.get_device, params))) > 1:
        raise ValueError("the tensors of a step must share their dtype and device")


def _is_dense(p: Tensor) -> bool:
    """Whether p's elements fill one range of memory, in any order of its axes."""
    expect = 1
    for stride, n in sorted((s, n) for s, n in zip(p.stride(), p.shape) if n > 1):
        if stride != expect:
            return False
        expect *= n
    return True


def _laid_out(p: Tensor, g: Tensor) -> Tensor:
    """g in p's memory order."""
    if g.layout != torch.strided:
        raise ValueError(f"gradients must be dense, got {g.layout}")
    if g.shape != p.shape:
        raise ValueError(f"gradient {tuple(g.shape)} for a tensor {tuple(p.shape)}")
    if not _is_dense(p):
        raise ValueError("a parameter's elements must fill one range of memory, got strides "
                         f"{p.stride()} for {tuple(p.shape)}")
    if all(a == b for a, b, n in zip(g.stride(), p.stride(), p.shape) if n > 1):
        return g
    return torch.empty_like(p).copy_(g)


_SIZES = {"exp_avg": 1, "exp_avg_sq": 1, "exp_avg_exponent": BLOCK, "exp_avg_sq_exponent": BLOCK,
          "master": 1}


def _state_tensors(state: dict[str, Tensor], dtype: torch.dtype, device) -> tuple[int, int]:
    """(bits, elements) of a checked state."""
    for name in ("exp_avg", "exp_avg_sq"):
        if name not in state:
            raise ValueError(f"the state has no {name!r}")
    m = state["exp_avg"]
    bits = {torch.float32: 32, torch.uint8: 8}.get(m.dtype)
    if bits is None:
        raise ValueError(f"states must be fp32 or uint8 codes, got {m.dtype}")
    wanted = {"exp_avg", "exp_avg_sq"} | ({"exp_avg_exponent", "exp_avg_sq_exponent"}
                                         if bits == 8 else set())
    if dtype in (torch.float16, torch.bfloat16):
        wanted |= {"master"} & state.keys()
    if state.keys() != wanted:
        raise ValueError(f"a state of {bits} bits holds {sorted(wanted)}, got {sorted(state)}")
    n = m.numel()
    for name, t in state.items():
        dt = torch.float32 if name == "master" else m.dtype
        if (t.dtype != dt or t.dim() != 1 or t.numel() * _SIZES[name] != n or t.device != device
                or not t.is_contiguous()):
            raise ValueError(f"state {name!r} must be dense {dt} of {n // _SIZES[name]} elements "
                             f"on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return bits, n


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
    n = len(params)
    if len(grads) != n:
        raise ValueError(f"{n} tensors and {len(grads)} gradients")
    if n == 0:
        return
    _one_kind(params)
    first = params[0]
    dtype, device, index = first.dtype, first.device, first.get_device()
    bits, elements = _state_tensors(state, dtype, device)
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("adamw_step cannot be captured in a CUDA graph: the step's bias "
                           "corrections are computed on the host")
    given, live = grads, params
    if any(g is None for g in grads):
        given = [g for g in grads if g is not None]
        live = [p for p, g in zip(params, grads) if g is not None]
        if not live:
            return
    if set(map(_dtype_of, given)) != {dtype} or set(map(Tensor.get_device, given)) != {index}:
        raise ValueError(f"gradients must be {dtype} on {device}, as the tensors")
    # the usual case, dense tensors of the same shape, is checked without a loop in Python
    if not (all(map(Tensor.is_contiguous, params)) and all(map(Tensor.is_contiguous, given))
            and all(map(eq, map(_shape_of, live), map(_shape_of, given)))):
        given = [_laid_out(p, g) for p, g in zip(live, given)]
    g_ptr = array("q", map(Tensor.data_ptr, given))
    if live is not params:
        rest = iter(g_ptr)
        g_ptr = array("q", [0 if g is None else next(rest) for g in grads])
    if grad_scale is not None and (grad_scale.dtype != torch.float32 or grad_scale.numel() != 1
                                   or grad_scale.device != device):
        raise ValueError(f"grad_scale must be one fp32 value on {device}")
    if isinstance(step, int):
        steps = array("q", [step]) * n
    else:
        steps = array("q", map(int, step))
        if len(steps) != n:
            raise ValueError(f"{n} tensors and {len(steps)} steps")
    p_ptr = array("q", map(Tensor.data_ptr, params))
    counts = array("q", map(Tensor.numel, params))
    address = lambda a: a.buffer_info()[0]  # noqa: E731
    ptr = lambda name: state[name].data_ptr() if name in state else None  # noqa: E731
    _core.launch(
        _lib.lib().msda_adamw_step, index,
        _core._DTYPE_CODE[dtype], bits, n, address(p_ptr), address(g_ptr), address(counts),
        address(steps), lr, betas[0], betas[1], eps, weight_decay, int(seed) & 0xFFFFFFFF,
        None if grad_scale is None else grad_scale.data_ptr(), ptr("exp_avg"),
        ptr("exp_avg_sq"), ptr("exp_avg_exponent"), ptr("exp_avg_sq_exponent"),
        ptr("master"), elements)
    torch.autograd.graph.increment_version(live)
    torch.autograd.graph.increment_version(state.values())


def adamw_state_values(state: dict[str, Tensor]) -> tuple[Tensor, Tensor]:
    """(exp_avg, exp_avg_sq) that a state stands for, flat as the state is.
    8-bit moments come as bf16, which holds them exactly; fp32 ones as they are."""
    m, v = state["exp_avg"], state["exp_avg_sq"]
    if not m.is_cuda:
        raise ValueError("AdamW requires CUDA tensors. Got CPU tensors instead.")
    bits, n = _state_tensors({k: t for k, t in state.items() if k != "master"}, torch.float32,
                             m.device)
    if bits == 32:
        return m, v
    out = [torch.empty(n, device=m.device, dtype=torch.bfloat16) for _ in range(2)]
    _core.launch(_lib.lib().msda_adamw_values, m.get_device(),
                 m.data_ptr(), state["exp_avg_exponent"].data_ptr(), v.data_ptr(),
                 state["exp_avg_sq_exponent"].data_ptr(), n, out[0].data_ptr(),
                 out[1].data_ptr())
    return out[0], out[1]


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
        state_bits: 32, or 8: moments in one byte each, with random rounding.
        master_weights: keep fp32 copies of 16-bit parameters, which the step
            updates and rounds into the parameters.
        seed: of the 8-bit states' rounding.

    Parameters without a gradient are skipped, and count their own steps.  A
    state_dict of torch.optim.AdamW can be loaded where state_bits is 32; an
    8-bit one holds the codes and exponents themselves.  `step` cannot be
    captured in a CUDA graph.
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
                    self.state[part.params[i]] = {"step": 0, **part.own(i, at)}

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
                adamw_step(part.params, grads, part.state, step=[max(s, 1) for s in steps],
                           lr=group["lr"], betas=group["betas"], eps=group["eps"],
                           weight_decay=group["weight_decay"], seed=self.seed)
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
        states, of torch.optim.AdamW's) over the same parameters."""
        groups = state_dict["param_groups"]
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
            for key in ("lr", "betas", "eps", "weight_decay"):
                if key in saved:
                    group[key] = saved[key]


__all__ = ["AdamW", "adamw_step", "adamw_state", "adamw_state_values"]
