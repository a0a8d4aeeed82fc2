"""Rows of numbers around the memory over decisions, on the MI355X library (include/flyguy_memory.h): layer norm and dropout.
An addition: the reference norms nothing and drops nothing.

    y = layer_norm(x, weight, bias)           # each row centred, divided by its deviation, scaled and shifted
    y = dropout(x, share, counter)            # a share of the numbers dropped; the mask is made again for the gradient

float32, bfloat16 or binary16 on the GPU; rows are the last dimension.  Gradients are backwards and of the first order.  Work
goes to the current stream; nothing synchronises, and calls may be captured in a graph.
"""
from __future__ import annotations

import struct

import torch

from ._lib import lib
from .memory_hip import _TYPES, _call, _floats, _no_tangents, _once, _ptr, _wants_grad, _workspaces

_NORM = struct.Struct("=17qd")
_DROP = struct.Struct("=7qd")


def _of_rows(what: str, x) -> None:
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError(f"{what}: x must be a tensor on the GPU")
    if x.dtype not in _TYPES or x.dim() < 1:
        raise ValueError(f"{what}: x must be float32, bfloat16 or float16 of at least one dimension")


def _as_rows(x: torch.Tensor) -> torch.Tensor:
    """x as [rows, width], a row's values side by side; a copy only where no strides do."""
    width = x.shape[-1]
    if x.dim() != 2:
        rows = x.numel() // width if width else 0
        x = x.view(rows, width) if x.is_contiguous() else x.reshape(rows, width)
    return x if x.stride(1) == 1 or width == 1 else x.contiguous()


# ------------------------------------------------------------------------------------------------ layer norm
def _pack_norm(x, y, g, gx, weight, bias, gweight, gbias, stats, partial, eps) -> bytes:
    rows, width = x.shape
    return _NORM.pack(x.data_ptr(), _ptr(y), _ptr(g), _ptr(gx), x.stride(0), 0 if y is None else y.stride(0),
                      0 if g is None else g.stride(0), 0 if gx is None else gx.stride(0), _ptr(weight), _ptr(bias),
                      _ptr(gweight), _ptr(gbias), _ptr(stats), _ptr(partial), rows, width, _TYPES[x.dtype], eps)


def _partial(rows, like) -> torch.Tensor:
    """Room for the workgroups' sums."""
    sizes = ("norm", *rows.shape, rows.dtype)
    n = _workspaces.get(sizes)
    if n is None:
        if len(_workspaces) >= 4096:
            _workspaces.clear()
        n = _workspaces[sizes] = lib().fm_norm_partial(_pack_norm(rows, *[None] * 9, 0.0))
    return like.new_empty(n)


class LayerNormHip(torch.autograd.Function):
    """layer_norm with gradients: apply(x, weight, bias, eps) (weight and bias may be None)."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        rows = _as_rows(x)
        stats = torch.empty(rows.shape[0], 2, dtype=torch.float32, device=x.device)
        y = x.new_empty(x.shape)
        _call("fm_norm", x, _pack_norm(rows, y.view(rows.shape), None, None, weight, bias, None, None, stats, None, eps))
        ctx.eps = eps
        ctx.save_for_backward(x, weight, bias, stats)
        return y

    @staticmethod
    def backward(ctx, gy):
        _once("layer_norm")
        x, weight, bias, stats = ctx.saved_tensors
        rows, g = _as_rows(x), _as_rows(gy)
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        gx = x.new_empty(x.shape) if want_x else None
        gw = torch.empty_like(weight) if want_w else None
        gb = torch.empty_like(bias) if want_b else None
        partial = _partial(rows, stats) if want_w or want_b else None
        _call("fm_norm_bwd", x, _pack_norm(rows, None, g, None if gx is None else gx.view(rows.shape), weight, bias, gw, gb, stats,
                                           partial, ctx.eps))
        return gx, gw, gb, None


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """Each row (the last dimension, 1 to 2^24 values) less its mean, over the root of its mean square deviation plus eps, times
    weight, plus bias (float32 [width] each, or None).  Means and deviations are taken in float32 about the mean (a row whose
    squares add up past float32's largest number, as two numbers 1e20 apart do, is all bias); y is dense, of x's type.  Gradients of x, weight and bias; the weights' are summed in a fixed order."""
    what = "layer_norm"
    _no_tangents(what, x, weight, bias)
    _of_rows(what, x)
    width, eps = x.shape[-1], float(eps)
    if not 1 <= width <= 1 << 24:
        raise ValueError(f"{what}: rows of 1 to 2^24 values")
    if not eps >= 0:
        raise ValueError(f"{what}: eps below 0")
    weight = None if weight is None else _floats(what, "weight", weight, (width,), x.device)
    bias = None if bias is None else _floats(what, "bias", bias, (width,), x.device)
    if _wants_grad(x, weight, bias):
        return LayerNormHip.apply(x, weight, bias, eps)
    rows, y = _as_rows(x), x.new_empty(x.shape)
    _call("fm_norm", x, _pack_norm(rows, y.view(rows.shape), None, None, weight, bias, None, None, None, None, eps))
    return y


# ------------------------------------------------------------------------------------------------ dropout
def _drop(x, share, counter):
    y = x.new_empty(x.shape)
    if x.numel():
        rows = x.view(1, -1) if x.is_contiguous() else _as_rows(x)
        _call("fm_drop", x, _DROP.pack(rows.data_ptr(), y.data_ptr(), counter.data_ptr(), rows.stride(0), *rows.shape,
                                       _TYPES[x.dtype], share))
    return y


class DropoutHip(torch.autograd.Function):
    """dropout with its gradient: apply(x, share, counter)."""

    @staticmethod
    def forward(ctx, x, share, counter):
        ctx.share = share
        ctx.save_for_backward(counter)        # (one that is changed before the gradient is found out)
        return _drop(x, share, counter)

    @staticmethod
    def backward(ctx, gy):
        _once("dropout")
        return _drop(gy, ctx.share, ctx.saved_tensors[0]), None, None


def dropout(x, share: float, counter):
    """x with a share of its numbers set to 0, the others divided by what is left: number i (in x's order, whatever its strides)
    is dropped where its 16-bit draw is below t = round(65536 share), and multiplied by 65536 / (65536 - t) elsewhere, so that
    the mean stays exactly; share 1 drops all.  counter: int64 [2] on the same GPU, (seed, offset), read when the work runs: the
    draws are those of Philox4x32 of 10 rounds, of key seed and counter (i // 8, offset).  The same counter gives the same mask;
    it may not be changed in place before the gradient is taken.  y is dense."""
    what = "dropout"
    _no_tangents(what, x)
    _of_rows(what, x)
    share = float(share)
    if not 0 <= share <= 1:
        raise ValueError(f"{what}: a share from 0 to 1")
    if not isinstance(counter, torch.Tensor) or counter.dtype != torch.int64 or counter.device != x.device or \
            tuple(counter.shape) != (2,):
        raise ValueError(f"{what}: counter must be int64 [2] on the same GPU")
    counter = counter.contiguous()
    if _wants_grad(x):
        return DropoutHip.apply(x, share, counter)
    return _drop(x, share, counter)
