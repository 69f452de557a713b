"""Rotary positions on several axes (width, height, depth, time).

A pair of channels j of every head turns by the angle
positions[b, t, axis_index[j]] * inv_freq[j], so the product of a query and a
key depends on how far apart they lie on each axis.  Positions are one set of
coordinates per token -- grid cells, or the continuous reference points of
deformable attention's queries, for which there is a gradient.

Runs in the sm_100a kernel of libmsda_b200.so (msda_rotary); there is no CPU
fallback.
"""

from __future__ import annotations

from array import array
from collections.abc import Sequence

import torch
from torch import nn

from msda_triton_b200 import _core, _lib

_POSITION_CODE = {torch.float32: 0, torch.int32: 1, torch.int64: 2}
MAX_AXES = 4
MAX_PAIRS = 2048


def axial_frequencies(rotated: int, num_axes: int, theta: float = 100.0,
                      sections: Sequence[int] | None = None, device=None
                      ) -> tuple[torch.Tensor, torch.Tensor]:
    """(inv_freq, axis_index) for `rotated` channels on `num_axes` axes.

    By default the rotated // 2 pairs are dealt to the axes in turn (pair j on
    axis j % num_axes), so every axis has high and low frequencies; with
    `sections`, axis a has the next sections[a] pairs.  The frequencies of an
    axis with n pairs fall geometrically, theta ** (-i / n) for i = 0 ... n - 1.
    """
    if rotated < 0 or rotated % 2:
        raise ValueError(f"rotated must be an even number of channels, got {rotated}")
    if not 1 <= num_axes <= MAX_AXES:
        raise ValueError(f"num_axes must be 1 to {MAX_AXES}, got {num_axes}")
    pairs = rotated // 2
    if sections is None:
        axis = [j % num_axes for j in range(pairs)]
    else:
        if len(sections) != num_axes or sum(sections) != pairs or min(sections) < 0:
            raise ValueError(f"sections must be {num_axes} numbers of pairs with sum {pairs}, "
                             f"got {tuple(sections)}")
        axis = [a for a, n in enumerate(sections) for _ in range(n)]
    seen, freq = [0] * num_axes, []
    for a in axis:
        freq.append(float(theta) ** (-seen[a] / axis.count(a)))
        seen[a] += 1
    return (torch.tensor(freq, dtype=torch.float32, device=device),
            torch.tensor(axis, dtype=torch.int32, device=device))


def pyramid_positions(spatial_shapes, device=None) -> torch.Tensor:
    """(1, K, d) positions (x, y[, z]) of a flattened pyramid's cells, all in
    cells of the first level: a cell of a coarser level lies at its centre."""
    sizes = [tuple(int(n) for n in s) for s in spatial_shapes]
    levels = []
    for size in sizes:
        axes = [(torch.arange(n, device=device, dtype=torch.float32) + 0.5) * (n0 / n) - 0.5
                for n, n0 in zip(size, sizes[0])]
        grid = torch.meshgrid(*axes, indexing="ij")
        levels.append(torch.stack(grid[::-1], -1).reshape(-1, len(size)))
    return torch.cat(levels)[None]


def _check(xs, positions, inv_freq, axis_index):
    """positions as (1 or B, Q, A)."""
    first = xs[0]
    if not first.is_cuda:
        raise ValueError("rotary requires CUDA tensors. Got CPU tensors instead.")
    dtype, device, shape = first.dtype, first.device, first.shape
    if dtype not in _core._DTYPE_CODE:
        raise NotImplementedError(f"rotary only supports fp32, fp16, and bf16. Got {dtype}.")
    if len(shape) != 4:
        raise ValueError(f"expected (B, Q, H, C), got {tuple(shape)}")
    B, Q, _, C = shape
    for x in xs[1:]:
        other = x.shape
        if (x.device != device or x.dtype != dtype or len(other) != 4 or other[0] != B
                or other[1] != Q or other[3] != C):
            raise ValueError("queries and keys must share their device, dtype, batch, tokens and "
                             f"channels; got {tuple(other)} {x.dtype} beside {tuple(shape)} "
                             f"{dtype}")
    if positions.dim() == 2:
        positions = positions[None]
    where = positions.shape
    if len(where) != 3 or where[0] not in (1, B) or where[1] != Q:
        raise ValueError(f"positions must be (Q, A) or (1 or B, Q, A) with B={B}, Q={Q}; "
                         f"got {tuple(where)}")
    if not 1 <= where[2] <= MAX_AXES:
        raise ValueError(f"positions must have 1 to {MAX_AXES} axes, got {where[2]}")
    if positions.dtype == torch.bool or positions.is_complex():
        raise ValueError(f"positions must be numbers, got {positions.dtype}")
    pairs = inv_freq.shape
    if (len(pairs) != 1 or inv_freq.dtype != torch.float32 or axis_index.shape != pairs
            or axis_index.dtype != torch.int32):
        raise ValueError("inv_freq must be (pairs,) fp32 and axis_index (pairs,) int32, got "
                         f"{tuple(pairs)} {inv_freq.dtype} and "
                         f"{tuple(axis_index.shape)} {axis_index.dtype}")
    if 2 * pairs[0] > C or pairs[0] > MAX_PAIRS:
        raise ValueError(f"{pairs[0]} pairs do not fit {C} channels (and at most {MAX_PAIRS})")
    if positions.device != device or inv_freq.device != device or axis_index.device != device:
        raise ValueError(f"positions, inv_freq and axis_index must be on {device}, got "
                         f"{positions.device}, {inv_freq.device} and {axis_index.device}")
    return positions


def _positions(positions):
    """In a dtype and layout that the kernel reads."""
    if positions.dtype not in _POSITION_CODE:
        p = positions.detach()
        positions = p.float() if p.dtype.is_floating_point else p.long()
    return positions if positions.is_contiguous() else positions.detach().contiguous()


def _dense_channels(x):
    return x if x.stride(3) == 1 or x.shape[3] <= 1 else x.detach().contiguous()


def _address(values) -> tuple[array, int]:
    """A host table of 64-bit values (to be kept alive), and where it lies."""
    table = array("q", values)
    return table, table.buffer_info()[0]


def _tables(ts):
    """Host tables of the tensors' addresses and of their (batch, token, head) strides."""
    strides = []
    for t in ts:
        strides += t.stride()[:3]
    return _address([t.data_ptr() for t in ts]), _address(strides)


def turn(xs, ys, positions, inv_freq, axis_index, interleaved, inverse, inputs=None, gpos=None):
    """Launch on prepared tensors: ys are the xs turned (or turned back)."""
    first = xs[0]
    B, Q, _, C = first.shape
    batch, _, axes = positions.shape
    heads = _address([x.shape[2] for x in xs])
    (px, sx), (py, sy) = _tables(xs), _tables(ys)
    pi, si = _tables(inputs) if inputs is not None else ((None, None), (None, None))
    _core.launch(
        _lib.lib().msda_rotary, first.get_device(),
        _core._DTYPE_CODE[first.dtype], B, Q, C, len(xs), heads[1], px[1], sx[1], py[1], sy[1],
        positions.data_ptr(), _POSITION_CODE[positions.dtype], 0 if batch == 1 else Q * axes, axes,
        inv_freq.data_ptr(), axis_index.data_ptr(), inv_freq.shape[0], interleaved, inverse,
        pi[1], si[1], None if gpos is None else gpos.data_ptr())


def _new(x):
    return (torch.empty_like(x) if x.is_contiguous()
            else torch.empty(x.shape, device=x.device, dtype=x.dtype))


def rotary_forward(positions, inv_freq, axis_index, interleaved, xs):
    ys = [_new(x) for x in xs]
    turn([_dense_channels(x) for x in xs], ys, _positions(positions), inv_freq.contiguous(),
         axis_index.contiguous(), interleaved, False)
    return ys


def rotary_backward(positions, inv_freq, axis_index, interleaved, grads, inputs=None):
    """(gradients of the inputs, of the positions or None without `inputs`)."""
    grads = [_dense_channels(g) for g in grads]
    gxs, pos, gpos = [_new(g) for g in grads], _positions(positions), None
    if inputs is not None:
        B, Q = grads[0].shape[:2]
        gpos = torch.empty((B, Q, pos.shape[2]), device=pos.device, dtype=torch.float32)
        inputs = [_dense_channels(x) for x in inputs]
    turn(grads, gxs, pos, inv_freq.contiguous(), axis_index.contiguous(), interleaved, True,
         inputs, gpos)
    if gpos is not None:
        if pos.shape[0] != gpos.shape[0]:  # one set of positions for the whole batch
            gpos = gpos.sum(0, keepdim=True)
        gpos = gpos.to(positions.dtype)
    return gxs, gpos


class RotaryFn(torch.autograd.Function):
    """Autograd Function of rotary / rotary_qk; gradients flow to the tensors and, where they
    require one, to the positions."""

    @staticmethod
    def forward(ctx, positions, inv_freq, axis_index, interleaved, *xs):
        ys = rotary_forward(positions, inv_freq, axis_index, interleaved, xs)
        ctx.interleaved = interleaved
        ctx.save_for_backward(positions, inv_freq, axis_index,
                              *(xs if ctx.needs_input_grad[0] else ()))
        return tuple(ys)

    @staticmethod
    def backward(ctx, *grads):
        positions, inv_freq, axis_index, *inputs = ctx.saved_tensors
        gxs, gpos = rotary_backward(positions, inv_freq, axis_index, ctx.interleaved, grads,
                                    inputs or None)
        return (gpos, None, None, None, *gxs)


def _apply(xs, positions, inv_freq, axis_index, interleaved):
    if torch.compiler.is_compiling():
        from msda_triton_b200 import ops

        if positions.dim() == 2:
            positions = positions[None]
        return tuple(ops.rotary_forward(list(xs), positions, inv_freq, axis_index, interleaved))
    positions = _check(xs, positions, inv_freq, axis_index)
    if torch.is_grad_enabled() and (positions.requires_grad or any(x.requires_grad for x in xs)):
        return RotaryFn.apply(positions, inv_freq, axis_index, bool(interleaved), *xs)
    return tuple(rotary_forward(positions, inv_freq, axis_index, bool(interleaved), xs))


def rotary(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
           axis_index: torch.Tensor, interleaved: bool = False) -> torch.Tensor:
    """x (B, Q, H, C) with the first 2 * pairs channels of each head turned.

    Args:
        x: fp32, fp16 or bf16; any strides with dense channels are read in place.
        positions: (Q, A) or (1 or B, Q, A), A = 1 to 4 axes; fp32, or integers
            (exact up to 2^24); other floating types are converted to fp32.
        inv_freq: (pairs,) fp32 angle per unit of position.
        axis_index: (pairs,) int32, each in [0, A) (not checked: it stays on the
            device).
        interleaved: pairs are channels (2j, 2j + 1) instead of (j, j + pairs).

    Returns:
        a tensor of x's shape and dtype, with autograd for x and positions.

    Raises:
        ValueError: CPU tensors, shapes that do not fit.
        NotImplementedError: dtype other than fp32/fp16/bf16.
    """
    return _apply((x,), positions, inv_freq, axis_index, interleaved)[0]


def rotary_qk(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
              axis_index: torch.Tensor, interleaved: bool = False
              ) -> tuple[torch.Tensor, torch.Tensor]:
    """rotary of queries and keys of the same tokens in one launch; they may
    differ in their number of heads."""
    return _apply((q, k), positions, inv_freq, axis_index, interleaved)


def rotary_qk_(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
               axis_index: torch.Tensor, interleaved: bool = False
               ) -> tuple[torch.Tensor, torch.Tensor]:
    """rotary_qk in place, for inference: q and k are overwritten and returned."""
    positions = _check((q, k), positions, inv_freq, axis_index)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad
                                    or positions.requires_grad):
        raise RuntimeError("rotary_qk_ has no gradient: use rotary_qk, or torch.no_grad()")
    for x in (q, k):
        if x.stride(3) != 1 and x.shape[3] > 1:
            raise ValueError("rotary_qk_ needs dense channels")
        if any(s == 0 and n > 1 for s, n in zip(x.stride(), x.shape)):
            raise ValueError("rotary_qk_ cannot write to an expanded tensor")
    turn((q, k), (q, k), _positions(positions), inv_freq.contiguous(), axis_index.contiguous(),
         bool(interleaved), False)
    torch.autograd.graph.increment_version((q, k))
    return q, k


class AxialRotary(nn.Module):
    """rotary_qk with its frequencies as buffers.

    head_dim channels per head, of which the first `rotated` (default: all)
    turn with the position on num_axes axes (see axial_frequencies)."""

    def __init__(self, head_dim: int, num_axes: int, theta: float = 100.0,
                 rotated: int | None = None, sections: Sequence[int] | None = None,
                 interleaved: bool = False, device=None) -> None:
        super().__init__()
        rotated = head_dim - head_dim % 2 if rotated is None else rotated
        if rotated > head_dim:
            raise ValueError(f"rotated ({rotated}) exceeds head_dim ({head_dim})")
        inv_freq, axis_index = axial_frequencies(rotated, num_axes, theta, sections, device)
        self.register_buffer("inv_freq", inv_freq, persistent=False)
        self.register_buffer("axis_index", axis_index, persistent=False)
        self.num_axes, self.interleaved = num_axes, interleaved

    def forward(self, q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor
                ) -> tuple[torch.Tensor, torch.Tensor]:
        if positions.shape[-1] != self.num_axes:
            raise ValueError(f"positions must have {self.num_axes} axes, "
                             f"got {tuple(positions.shape)}")
        return rotary_qk(q, k, positions, self.inv_freq, self.axis_index, self.interleaved)

    def _apply(self, fn, recurse=True):
        # moving the module to a 16-bit dtype must not round the frequencies
        freq = self.inv_freq
        super()._apply(fn, recurse)
        if self.inv_freq.dtype != torch.float32:
            self.inv_freq = freq.to(self.inv_freq.device)
        return self


__all__ = ["rotary", "rotary_qk", "rotary_qk_", "AxialRotary", "RotaryFn", "axial_frequencies",
           "pyramid_positions"]
