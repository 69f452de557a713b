"""torch.library registration of the MSDA ops.

The reference hides its kernels from torch.compile (`@torch.compiler.disable`,
src/msda_triton/triton/msda_3d.py:729,797), which costs a graph break at
every call.  Here the forward and backward are registered as custom ops with
fake (meta) implementations and an autograd formula, so torch.compile traces
through them (Dynamo sees an opaque op with known output shapes) and CUDA
graphs capture them like any other kernel launch:

    torch.ops.msda_b200.msda_forward(value, shapes, loc, attn, ndim, clamp, eps)
    torch.ops.msda_b200.msda_backward(grad_out, value, shapes, loc, attn, ndim, clamp, eps)

`msda2d`/`msda3d`/`msda2d_fwd`/`msda3d_fwd` route through these ops while
torch.compile is tracing, and call the autograd Functions directly in eager
mode (no dispatcher overhead).  Both paths run the same C ABI entry points.
"""

from __future__ import annotations

import torch
from torch import Tensor

from msda_triton_b200 import _core, _lib


@torch.library.custom_op("msda_b200::msda_forward", mutates_args=())
def msda_forward(value: Tensor, spatial_shapes: Tensor, sampling_locations: Tensor,
                 attention_weights: Tensor, ndim: int, clamp_grid: bool,
                 clamp_eps: float) -> Tensor:
    """(B, Q, H*C) output of MSDA in value's dtype (same checks and errors as msda2d/msda3d)."""
    return _core.fwd_entry(ndim, value, spatial_shapes, sampling_locations, attention_weights,
                           clamp_grid, clamp_eps)


@msda_forward.register_fake
def _msda_forward_fake(value, spatial_shapes, sampling_locations, attention_weights, ndim,
                       clamp_grid, clamp_eps):
    B, _, H, C = value.shape
    return value.new_empty((B, sampling_locations.shape[1], H * C))


@torch.library.custom_op("msda_b200::msda_backward", mutates_args=())
def msda_backward(grad_output: Tensor, value: Tensor, spatial_shapes: Tensor,
                  sampling_locations: Tensor, attention_weights: Tensor, ndim: int,
                  clamp_grid: bool, clamp_eps: float) -> tuple[Tensor, Tensor, Tensor]:
    """(grad_value, grad_sampling_locations, grad_attention_weights), each in the
    dtype of its input."""
    shapes, on_dev = _core.prepare_spatial(spatial_shapes)
    loc, attn = _core.sampling_pair(value, sampling_locations, attention_weights)
    gv, gl, ga = _core.backward(ndim, value.contiguous(), shapes, on_dev, loc, attn, clamp_grid,
                                clamp_eps, grad_output)
    return gv, gl.to(sampling_locations.dtype), ga.to(attention_weights.dtype)


@msda_backward.register_fake
def _msda_backward_fake(grad_output, value, spatial_shapes, sampling_locations,
                        attention_weights, ndim, clamp_grid, clamp_eps):
    fmt = torch.contiguous_format
    return (torch.empty_like(value, memory_format=fmt),
            torch.empty_like(sampling_locations, memory_format=fmt),
            torch.empty_like(attention_weights, memory_format=fmt))


def _setup_context(ctx, inputs, output):
    value, spatial_shapes, loc, attn, ndim, clamp_grid, clamp_eps = inputs
    ctx.save_for_backward(value, spatial_shapes, loc, attn)
    ctx.ndim = ndim
    ctx.clamp_grid = clamp_grid
    ctx.clamp_eps = clamp_eps


def _backward(ctx, grad_output):
    value, spatial_shapes, loc, attn = ctx.saved_tensors
    gv, gl, ga = msda_backward(grad_output.contiguous(), value, spatial_shapes, loc, attn,
                               ctx.ndim, ctx.clamp_grid, ctx.clamp_eps)
    return gv, None, gl, ga, None, None, None


msda_forward.register_autograd(_backward, setup_context=_setup_context)


__all__ = ["msda_forward", "msda_backward"]


# ---------------------------------------------------------------- fused prologue
@torch.library.custom_op("msda_b200::msda_fused_forward", mutates_args=())
def msda_fused_forward(value: Tensor, spatial_shapes: Tensor, reference_points: Tensor,
                       sampling_offsets: Tensor, attention_logits: Tensor, ndim: int,
                       clamp_grid: bool, clamp_eps: float) -> Tensor:
    """(B, Q, H*C) output of msda{2,3}d_fused (locations and weights formed in the kernels)."""
    from msda_triton_b200 import fused

    with torch.no_grad():
        return fused.MSDAFusedFn.apply(ndim, value, spatial_shapes, reference_points,
                                       sampling_offsets, attention_logits, clamp_grid, clamp_eps)


@msda_fused_forward.register_fake
def _msda_fused_forward_fake(value, spatial_shapes, reference_points, sampling_offsets,
                             attention_logits, ndim, clamp_grid, clamp_eps):
    B, _, H, C = value.shape
    return value.new_empty((B, sampling_offsets.shape[1], H * C))


@torch.library.custom_op("msda_b200::msda_fused_backward", mutates_args=())
def msda_fused_backward(grad_output: Tensor, value: Tensor, spatial_shapes: Tensor,
                        reference_points: Tensor, sampling_offsets: Tensor,
                        attention_logits: Tensor, ndim: int, clamp_grid: bool,
                        clamp_eps: float) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """(grad_value, grad_reference_points, grad_sampling_offsets,
    grad_attention_logits), each in the dtype and shape of its input."""
    from msda_triton_b200 import fused

    return fused.fused_backward(ndim, grad_output, value, spatial_shapes, reference_points,
                                sampling_offsets, attention_logits, clamp_grid, clamp_eps)


@msda_fused_backward.register_fake
def _msda_fused_backward_fake(grad_output, value, spatial_shapes, reference_points,
                              sampling_offsets, attention_logits, ndim, clamp_grid, clamp_eps):
    fmt = torch.contiguous_format
    return tuple(torch.empty_like(t, memory_format=fmt)
                 for t in (value, reference_points, sampling_offsets, attention_logits))


def _fused_setup_context(ctx, inputs, output):
    value, spatial_shapes, ref, off, logits, ndim, clamp_grid, clamp_eps = inputs
    ctx.save_for_backward(value, spatial_shapes, ref, off, logits)
    ctx.ndim = ndim
    ctx.clamp_grid = clamp_grid
    ctx.clamp_eps = clamp_eps


def _fused_backward(ctx, grad_output):
    value, spatial_shapes, ref, off, logits = ctx.saved_tensors
    gv, gr, go, gl = msda_fused_backward(grad_output.contiguous(), value, spatial_shapes, ref,
                                         off, logits, ctx.ndim, ctx.clamp_grid, ctx.clamp_eps)
    return gv, None, gr, go, gl, None, None, None


msda_fused_forward.register_autograd(_fused_backward, setup_context=_fused_setup_context)

__all__ += ["msda_fused_forward", "msda_fused_backward"]


# ---------------------------------------------------------------- pyramid group norm
@torch.library.custom_op("msda_b200::group_norm_forward", mutates_args=())
def group_norm_forward(x: list[Tensor], maps: bool, spatial_shapes: Tensor | None,
                       num_groups: int, weight: Tensor | None, bias: Tensor | None, eps: float,
                       activation: str) -> tuple[Tensor, Tensor]:
    """(y, statistics) of pyramid_group_norm; x holds the levels (maps) or the flattened pyramid."""
    return _lib.binding().pyramid_group_norm_forward(x, maps, spatial_shapes, num_groups, weight,
                                                     bias, eps, activation)


@group_norm_forward.register_fake
def _group_norm_forward_fake(x, maps, spatial_shapes, num_groups, weight, bias, eps, activation):
    first = x[0]
    keys = sum(t.shape[1:-1].numel() for t in x)
    levels = len(x) if maps else spatial_shapes.shape[0]
    return (first.new_empty((first.shape[0], keys, first.shape[-1])),
            first.new_empty((first.shape[0] * levels * num_groups * 2,), dtype=torch.float32))


@torch.library.custom_op("msda_b200::group_norm_backward", mutates_args=())
def group_norm_backward(grad_y: Tensor, stats: Tensor, x: list[Tensor], maps: bool,
                        spatial_shapes: Tensor | None, num_groups: int, weight: Tensor | None,
                        bias: Tensor | None, activation: str) -> list[Tensor]:
    """Gradients of x, then of weight and bias where they are given."""
    grads = _lib.binding().pyramid_group_norm_backward(grad_y, stats, x, maps, spatial_shapes,
                                                       num_groups, weight, bias, activation)
    return [g for g in grads if g is not None]


@group_norm_backward.register_fake
def _group_norm_backward_fake(grad_y, stats, x, maps, spatial_shapes, num_groups, weight, bias,
                              activation):
    return [torch.empty_like(t, memory_format=torch.contiguous_format)
            for t in (*x, weight, bias) if t is not None]


def _group_norm_setup(ctx, inputs, output):
    x, maps, spatial_shapes, num_groups, weight, bias, _, activation = inputs
    ctx.save_for_backward(output[1], spatial_shapes, weight, bias, *x)
    ctx.meta = maps, num_groups, activation


def _group_norm_backward(ctx, grad_y, grad_stats):
    stats, spatial_shapes, weight, bias, *x = ctx.saved_tensors
    maps, num_groups, activation = ctx.meta
    grads = group_norm_backward(grad_y.contiguous(), stats, x, maps, spatial_shapes, num_groups,
                                weight, bias, activation)
    gxs, rest = grads[:len(x)], iter(grads[len(x):])
    return (gxs, None, None, None, None if weight is None else next(rest),
            None if bias is None else next(rest), None, None)


group_norm_forward.register_autograd(_group_norm_backward, setup_context=_group_norm_setup)


# ---------------------------------------------------------------- rotary positions
@torch.library.custom_op("msda_b200::rotary_forward", mutates_args=())
def rotary_forward(xs: list[Tensor], positions: Tensor, inv_freq: Tensor, axis_index: Tensor,
                   interleaved: bool) -> list[Tensor]:
    """One or two tensors of heads turned by their positions (1 or B, Q, A)."""
    return _lib.binding().rotary_forward(xs, positions, inv_freq, axis_index, interleaved)


@rotary_forward.register_fake
def _rotary_forward_fake(xs, positions, inv_freq, axis_index, interleaved):
    return [torch.empty_like(x, memory_format=torch.contiguous_format) for x in xs]


@torch.library.custom_op("msda_b200::rotary_backward", mutates_args=())
def rotary_backward(grads: list[Tensor], inputs: list[Tensor], positions: Tensor,
                    inv_freq: Tensor, axis_index: Tensor, interleaved: bool) -> list[Tensor]:
    """Gradients of the tensors and, where `inputs` are given, of the positions."""
    return _lib.binding().rotary_backward(grads, inputs, positions, inv_freq, axis_index,
                                          interleaved)


@rotary_backward.register_fake
def _rotary_backward_fake(grads, inputs, positions, inv_freq, axis_index, interleaved):
    return [torch.empty_like(t, memory_format=torch.contiguous_format)
            for t in (*grads, *([positions] if inputs else []))]


def _rotary_setup(ctx, inputs, output):
    xs, positions, inv_freq, axis_index, interleaved = inputs
    if inv_freq.requires_grad:
        raise RuntimeError("rotary forms no gradient for inv_freq: detach it")
    ctx.count, ctx.interleaved = len(xs), interleaved
    ctx.save_for_backward(positions, inv_freq, axis_index,
                          *(xs if positions.requires_grad else ()))


def _rotary_backward(ctx, grads):
    positions, inv_freq, axis_index, *inputs = ctx.saved_tensors
    got = rotary_backward([g.contiguous() for g in grads], inputs, positions, inv_freq,
                          axis_index, ctx.interleaved)
    gpos = got[ctx.count] if inputs else None
    return got[:ctx.count], gpos, None, None, None


rotary_forward.register_autograd(_rotary_backward, setup_context=_rotary_setup)

__all__ += ["group_norm_forward", "group_norm_backward", "rotary_forward", "rotary_backward"]
