"""Group norm with an affine map and an activation over a feature pyramid.

Deformable attention reads its values from a pyramid of feature levels
flattened to (B, K, C), and a model normalises each level by itself before
that.  `pyramid_group_norm` does so in the flattened, channels-last layout, or
reads the L maps (B, *spatial, C) and writes the flattened pyramid in the same
pass:

    h = (x - mean) / sqrt(var + eps)      over one level of one batch entry and
                                          the channels of one group
    y = activation(h * weight + bias)

Statistics are fp32 for every dtype.  Runs in the sm_100a kernels of
libmsda_b200.so (msda_group_norm_fwd / _bwd); there is no CPU fallback.
"""

from __future__ import annotations

from collections.abc import Sequence

import torch
from torch import nn

from msda_triton_b200 import _lib

ACTIVATIONS = ("none", "relu", "silu", "gelu")


def pyramid_group_norm(x: torch.Tensor | Sequence[torch.Tensor],
                       spatial_shapes: torch.Tensor | Sequence[Sequence[int]] | None,
                       num_groups: int, weight: torch.Tensor | None = None,
                       bias: torch.Tensor | None = None, eps: float = 1e-5,
                       activation: str = "none") -> torch.Tensor:
    """Group norm, affine map and activation over each level of a pyramid.

    Args:
        x: the flattened pyramid (B, K, C), K = the sum of the level sizes,
            level after level; or a sequence of channels-last levels
            (B, *spatial, C), which are flattened on the way (for maps of
            torch's channels_last memory format, `m.movedim(1, -1)` is that
            view without a copy).
        spatial_shapes: (L, d) integer level sizes, as for msda2d / msda3d; kept
            on the CPU they cost nothing, on the GPU they are copied to the host,
            which waits for the device.  None is allowed for a sequence of levels.
        num_groups: groups of neighbouring channels; divides C.
        weight, bias: (C,), or (L, C) for a map per level; None: ones / zeros.
        eps: added to the variance.
        activation: "none", "relu", "silu" or "gelu" (the error function's).

    Returns:
        (B, K, C) in x's dtype, with autograd.

    Raises:
        ValueError: CPU tensors, shapes that do not fit, more than 16 levels.
        NotImplementedError: dtype other than fp32/fp16/bf16.
    """
    if torch.compiler.is_compiling():
        from msda_triton_b200 import ops

        maps = not isinstance(x, torch.Tensor)
        if spatial_shapes is not None and not isinstance(spatial_shapes, torch.Tensor):
            spatial_shapes = torch.tensor(spatial_shapes, dtype=torch.int64)
        y, _ = ops.group_norm_forward(list(x) if maps else [x], maps, spatial_shapes, num_groups,
                                      weight, bias, eps, activation)
        return y
    return _lib.binding().pyramid_group_norm(x, spatial_shapes, num_groups, weight, bias, eps,
                                             activation)


class PyramidGroupNorm(nn.Module):
    """pyramid_group_norm with its parameters: weight and bias of (num_channels,),
    or (num_levels, num_channels) with num_levels given."""

    def __init__(self, num_groups: int, num_channels: int, num_levels: int | None = None,
                 eps: float = 1e-5, affine: bool = True, activation: str = "none",
                 device=None, dtype=None) -> None:
        super().__init__()
        if num_channels % num_groups:
            raise ValueError(f"num_channels ({num_channels}) must be a multiple of num_groups "
                             f"({num_groups})")
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {ACTIVATIONS}, "
                             f"got {activation!r}")
        self.num_groups, self.num_channels, self.num_levels = num_groups, num_channels, num_levels
        self.eps, self.activation = eps, activation
        shape = (num_channels,) if num_levels is None else (num_levels, num_channels)
        for name, fill in (("weight", torch.ones), ("bias", torch.zeros)):
            self.register_parameter(
                name, nn.Parameter(fill(shape, device=device, dtype=dtype)) if affine else None)

    def forward(self, x, spatial_shapes=None) -> torch.Tensor:
        return pyramid_group_norm(x, spatial_shapes, self.num_groups, self.weight, self.bias,
                                  self.eps, self.activation)

    def extra_repr(self) -> str:
        return (f"{self.num_groups}, {self.num_channels}, num_levels={self.num_levels}, "
                f"eps={self.eps}, activation={self.activation!r}")


__all__ = ["pyramid_group_norm", "PyramidGroupNorm"]
