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

import functools
import math
from array import array
from collections.abc import Sequence

import torch
from torch import nn

from msda_triton_b200 import _core, _lib

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}


def _sizes(spatial_shapes) -> list[tuple[int, ...]]:
    """Level sizes on the host (a CUDA tensor of shapes is copied, which waits for the device)."""
    if isinstance(spatial_shapes, torch.Tensor):
        if spatial_shapes.dtype.is_floating_point or spatial_shapes.dtype == torch.bool:
            raise ValueError("spatial_shapes must be an integer tensor, "
                             f"got {spatial_shapes.dtype}")
        if spatial_shapes.dim() != 2:
            raise ValueError(f"spatial_shapes must be (L, d), got {tuple(spatial_shapes.shape)}")
        return spatial_shapes.tolist()
    return [tuple(int(n) for n in s) for s in spatial_shapes]


def _check(x, spatial_shapes, num_groups, weight, bias, activation):
    """(maps, list of inputs, rows per level) of checked arguments."""
    maps = not isinstance(x, torch.Tensor)
    xs = list(x) if maps else [x]
    if not xs:
        raise ValueError("pyramid_group_norm needs at least one level")
    first = xs[0]
    device, dtype, shape = first.device, first.dtype, first.shape
    if not first.is_cuda:
        raise ValueError("pyramid_group_norm requires CUDA tensors. Got CPU tensors instead.")
    if dtype not in _core._DTYPE_CODE:
        raise NotImplementedError("pyramid_group_norm only supports fp32, fp16, and bf16. "
                                  f"Got {dtype}.")
    for t in xs:
        if t.dim() < 3 or (not maps and t.dim() != 3):
            raise ValueError("x must be (B, K, C), or levels of (B, *spatial, C); "
                             f"got {tuple(t.shape)}")
        if t is not first and (t.device != device or t.dtype != dtype
                               or t.shape[0] != shape[0] or t.shape[-1] != shape[-1]):
            raise ValueError("levels must share their device, dtype, batch and channels; got "
                             f"{tuple(t.shape)} {t.dtype} beside {tuple(shape)} {dtype}")
    if maps:
        if spatial_shapes is not None:
            sizes = [list(s) for s in _sizes(spatial_shapes)]
            if sizes != [list(t.shape[1:-1]) for t in xs]:
                raise ValueError(f"spatial_shapes {sizes} do not match the levels' "
                                 f"{[list(t.shape[1:-1]) for t in xs]}")
        rows = [math.prod(t.shape[1:-1]) for t in xs]
    else:
        if spatial_shapes is None:
            raise ValueError("spatial_shapes is required for a flattened pyramid")
        sizes = _sizes(spatial_shapes)
        rows = [math.prod(s) for s in sizes]
        if any(min(s, default=0) < 0 for s in sizes):
            raise ValueError(f"negative spatial shape: {sizes}")
        if sum(rows) != shape[1]:
            raise ValueError(f"K={shape[1]} does not match sum of spatial shapes {sum(rows)}")
    channels = shape[-1]
    if num_groups < 1 or channels < 1 or channels % num_groups:
        raise ValueError(f"channels ({channels}) must be a positive multiple of num_groups "
                         f"({num_groups})")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.device != device:
            raise ValueError(f"{name} must be on {device}, got {t.device}")
        if t.dtype not in _core._DTYPE_CODE:
            raise NotImplementedError(f"{name} must be fp32, fp16, or bf16. Got {t.dtype}.")
        if t.shape not in ((channels,), (len(rows), channels)):
            raise ValueError(f"{name} must be ({channels},) or ({len(rows)}, {channels}), "
                             f"got {tuple(t.shape)}")
    if weight is not None and bias is not None and weight.shape != bias.shape:
        raise ValueError(f"weight {tuple(weight.shape)} and bias {tuple(bias.shape)} differ in "
                         "shape")
    return maps, xs, rows


def _row_stride(t: torch.Tensor) -> int | None:
    """Elements between neighbouring rows of (B, *spatial, C), if one step serves them all."""
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        return None
    step, rows = t.stride(-2), t.shape[-2]
    for n, s in zip(t.shape[-3:0:-1], t.stride()[-3:0:-1]):
        if n > 1 and s != step * rows:
            if rows > 1:
                return None
            step = s
        rows *= n
    return step


def _dense_rows(t: torch.Tensor) -> torch.Tensor:
    """t, copied if its rows are not evenly spaced rows of dense channels."""
    return t if t.numel() == 0 or _row_stride(t) is not None else t.contiguous()


def _table(values) -> tuple[array, int]:
    """A host table of 64-bit values (to be kept alive), and where it lies."""
    table = array("q", values)
    return table, table.buffer_info()[0]


def _levels(maps, xs, rows):
    """Host tables of the levels' addresses and (batch, row) strides."""
    if maps:
        ptrs = [t.data_ptr() for t in xs]
        strides = [s for t in xs for s in (t.stride(0), _row_stride(t) or 0)]
    else:
        (x,) = xs
        batch, step, _ = x.stride()
        ptrs, at, size = [], x.data_ptr(), x.element_size() * step
        for n in rows:
            ptrs.append(at)
            at += n * size
        strides = [batch, step] * len(rows)
    return _table(ptrs), _table(strides)


def _affine(weight, bias):
    """(weight, bias, dtype code, per_level) as the kernels take them."""
    one = weight if weight is not None else bias
    if one is None:
        return None, None, _lib.FLOAT32, 0
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        weight, bias = weight.float(), bias.float()
        one = weight
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    return weight, bias, _core._DTYPE_CODE[one.dtype], int(one.dim() == 2)


def _ptr(t):
    return None if t is None else t.data_ptr()


@functools.lru_cache(maxsize=256)
def _workspace_bytes(dtype, batch, channels, groups, rows, backward):
    """A function of sizes alone."""
    table = _table(rows)
    return _lib.lib().msda_group_norm_workspace_bytes(dtype, batch, channels, groups, len(rows),
                                                      table[1], backward)


def norm_forward(maps, xs, rows, groups, weight, bias, eps, activation):
    """(y, statistics) of checked arguments."""
    xs = [_dense_rows(t) for t in xs]
    first = xs[0]
    batch, channels, code = first.shape[0], first.shape[-1], _core._DTYPE_CODE[first.dtype]
    y = torch.empty((batch, sum(rows), channels), device=first.device, dtype=first.dtype)
    # the statistics, and behind them (on a boundary of 256 bytes) the workspace
    n_stats = -(-batch * len(rows) * groups * 2 // 64) * 64
    ws_bytes = _workspace_bytes(code, batch, channels, groups, tuple(rows), 0)
    stats = torch.empty((n_stats + ws_bytes // 4,), device=first.device, dtype=torch.float32)
    w, b, affine, per_level = _affine(weight, bias)
    c_rows = _table(rows)
    ptrs, strides = _levels(maps, xs, rows)
    at = stats.data_ptr()
    _core.launch(
        _lib.lib().msda_group_norm_fwd, first.get_device(),
        code, batch, channels, groups, len(rows), c_rows[1], ptrs[1], strides[1], _ptr(w), _ptr(b),
        affine, per_level, eps, ACTIVATIONS[activation], y.data_ptr(), at, at + 4 * n_stats,
        ws_bytes)
    return y, stats


def norm_backward(maps, xs, rows, groups, weight, bias, activation, stats, grad_y):
    """(gradients of xs, of weight, of bias); the last two None where the input is."""
    shapes = [t.shape for t in xs]
    xs = [_dense_rows(t) for t in xs]
    first = xs[0]
    batch, channels, code = first.shape[0], first.shape[-1], _core._DTYPE_CODE[first.dtype]
    grad_y = grad_y.to(first.dtype).contiguous()
    gxs = [torch.empty(s, device=first.device, dtype=first.dtype) for s in shapes]
    w, b, affine, per_level = _affine(weight, bias)
    gw = None if w is None else torch.empty_like(w)
    gb = None if b is None else torch.empty_like(b)
    c_rows = _table(rows)
    ptrs, strides = _levels(maps, xs, rows)
    gptrs, gstrides = _levels(maps, gxs, rows)
    ws_bytes = _workspace_bytes(code, batch, channels, groups, tuple(rows), 1)
    ws = torch.empty((ws_bytes,), device=first.device, dtype=torch.uint8)
    _core.launch(
        _lib.lib().msda_group_norm_bwd, first.get_device(),
        code, batch, channels, groups, len(rows), c_rows[1], ptrs[1], strides[1], _ptr(w), _ptr(b),
        affine, per_level, ACTIVATIONS[activation], stats.data_ptr(), grad_y.data_ptr(),
        gptrs[1], gstrides[1], _ptr(gw), _ptr(gb), ws.data_ptr(), ws_bytes)
    return (gxs, None if gw is None else gw.to(weight.dtype),
            None if gb is None else gb.to(bias.dtype))


class PyramidGroupNormFn(torch.autograd.Function):
    """Autograd Function of pyramid_group_norm; gradients flow to the features, weight and bias."""

    @staticmethod
    def forward(ctx, maps, rows, groups, eps, activation, weight, bias, *xs):
        y, stats = norm_forward(maps, xs, rows, groups, weight, bias, eps, activation)
        ctx.save_for_backward(stats, weight, bias, *xs)
        ctx.meta = maps, rows, groups, activation
        return y

    @staticmethod
    def backward(ctx, grad_y):
        stats, weight, bias, *xs = ctx.saved_tensors
        maps, rows, groups, activation = ctx.meta
        gxs, gw, gb = norm_backward(maps, xs, rows, groups, weight, bias, activation, stats,
                                    grad_y)
        return (None, None, None, None, None, gw, gb, *gxs)


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
    maps, xs, rows = _check(x, spatial_shapes, num_groups, weight, bias, activation)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                       for t in (weight, bias, *xs)):
        return PyramidGroupNormFn.apply(maps, rows, num_groups, float(eps), activation, weight,
                                        bias, *xs)
    return norm_forward(maps, xs, rows, num_groups, weight, bias, float(eps), activation)[0]


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
            raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, "
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


__all__ = ["pyramid_group_norm", "PyramidGroupNorm", "PyramidGroupNormFn"]
