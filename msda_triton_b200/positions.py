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

from collections.abc import Sequence

import torch
from torch import nn

from msda_triton_b200 import _lib

MAX_AXES = 4


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


def _traced(xs, positions, inv_freq, axis_index, interleaved):
    """As one opaque op (msda_b200::rotary_forward) under torch.compile."""
    from msda_triton_b200 import ops

    if positions.dim() == 2:
        positions = positions[None]
    return tuple(ops.rotary_forward(list(xs), positions, inv_freq, axis_index, interleaved))


def rotary(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
           axis_index: torch.Tensor, interleaved: bool = False) -> torch.Tensor:
    """x (B, Q, H, C) with the first 2 * pairs channels of each head turned.

    Args:
        x: fp32, fp16 or bf16; any strides with dense channels are read in place.
        positions: (Q, A) or (1 or B, Q, A), A = 1 to 4 axes; fp32, or integers
            (exact up to 2^24); other floating types are converted to fp32.
        inv_freq: (pairs,) fp32 angle per unit of position; a constant.
        axis_index: (pairs,) int32, each in [0, A); it stays on the device, so
            a pair with another index is no error but becomes NaN.
        interleaved: pairs are channels (2j, 2j + 1) instead of (j, j + pairs).

    Returns:
        a tensor of x's shape and dtype, with autograd for x and positions.

    Raises:
        ValueError: CPU tensors, shapes that do not fit.
        NotImplementedError: dtype other than fp32/fp16/bf16; a forward-mode tangent.
        RuntimeError: an inv_freq that requires a gradient.
    """
    if torch.compiler.is_compiling():
        return _traced((x,), positions, inv_freq, axis_index, interleaved)[0]
    return _lib.binding().rotary(x, positions, inv_freq, axis_index, interleaved)


def rotary_qk(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
              axis_index: torch.Tensor, interleaved: bool = False
              ) -> tuple[torch.Tensor, torch.Tensor]:
    """rotary of queries and keys of the same tokens in one launch; they may
    differ in their number of heads."""
    if torch.compiler.is_compiling():
        return _traced((q, k), positions, inv_freq, axis_index, interleaved)
    return _lib.binding().rotary_qk(q, k, positions, inv_freq, axis_index, interleaved)


def rotary_qk_(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
               axis_index: torch.Tensor, interleaved: bool = False
               ) -> tuple[torch.Tensor, torch.Tensor]:
    """rotary_qk in place, for inference: q and k are overwritten and returned.

    They may be slices of one tensor, but no element may lie in both, or twice
    in one: ValueError."""
    _lib.binding().rotary_in_place([q, k], positions, inv_freq, axis_index, interleaved)
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
        self._table = rotated, num_axes, theta, sections
        inv_freq, axis_index = axial_frequencies(*self._table, device)
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
        # moving the module to a 16-bit dtype must not round the frequencies, and no state_dict
        # fills them where a module made on the meta device gets its memory
        freq = self.inv_freq
        super()._apply(fn, recurse)
        if freq.is_meta and not self.inv_freq.is_meta:
            self.inv_freq, self.axis_index = axial_frequencies(*self._table, self.inv_freq.device)
        elif self.inv_freq.dtype != torch.float32:
            self.inv_freq = freq.to(self.inv_freq.device)
        return self


__all__ = ["rotary", "rotary_qk", "rotary_qk_", "AxialRotary", "axial_frequencies",
           "pyramid_positions"]
