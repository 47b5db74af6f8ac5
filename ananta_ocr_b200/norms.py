"""The residual sum behind a block and the norm before the next one, as one kernel
(``dash_add_norm`` and ``dash_add_norm_bwd`` of libdash_b200.so).

  rms_norm                x / sqrt(mean(x^2) + eps) * weight
  add_rms_norm            residual + scale * gate * (norm of) y, and its norm
  add_rms_norm_backward   the gradients of both, as a plain call

``rms_norm`` and ``add_rms_norm`` can be differentiated (once, in reverse; tensors with tangents
are refused).  A backward pass that is
captured into a CUDA graph should be a call of ``add_rms_norm_backward``: torch's own
differentiation of leaves whose accumulation nodes were made outside of the capture
(by an earlier graph that still lives) ends the process.
CUDA tensors only; every non-zero library status raises.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L
from .ops import _DT, _need_cuda, _no_tangents
from .page_pool import _call

_NORM = L.packer(L.DashNormArgs)
_BWD = L.packer(L.DashNormBwdArgs)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension, in fp32, rounded
    once to x's type (bf16, fp16 or fp32; weight [hidden] fp32 or of x's type)."""
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        return _AddNorm.apply(x, None, weight, None, None, float(eps), 1.0)
    return _forward(x, None, weight, None, None, eps, 1.0)[1]


def add_rms_norm(y: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float, *,
                 gate: Optional[torch.Tensor] = None, post_weight: Optional[torch.Tensor] = None,
                 scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """The stream behind a block and its norm, (stream, normed):

        z = rms_norm(y, post_weight) if post_weight is given else y
        stream = residual + scale * gate * z
        normed = rms_norm(stream, weight)

    y, residual [..., hidden] of one type (bf16, fp16, fp32), hidden <= 8192; weight and
    post_weight [hidden]; gate [hidden], or [groups, hidden] with a row for each group of
    rows / groups consecutive rows (a sequence's); the three are fp32 or of y's type.
    Everything is fp32 inside; the norm is that of the unrounded stream."""
    if torch.is_grad_enabled() and (y.requires_grad or residual.requires_grad or weight.requires_grad or
                                    (gate is not None and gate.requires_grad) or
                                    (post_weight is not None and post_weight.requires_grad)):
        return _AddNorm.apply(y, residual, weight, gate, post_weight, float(eps), float(scale))
    return _forward(y, residual, weight, gate, post_weight, eps, scale)


class NormGrads(NamedTuple):
    """Gradients of ``add_rms_norm``'s inputs; None where there is no such input.  Without
    gate, post_weight and scale those of y and residual are one tensor."""
    y: torch.Tensor
    residual: torch.Tensor
    weight: torch.Tensor
    gate: Optional[torch.Tensor]
    post_weight: Optional[torch.Tensor]


def add_rms_norm_backward(dstream: Optional[torch.Tensor], dnormed: torch.Tensor, y: torch.Tensor,
                          residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float, *,
                          gate: Optional[torch.Tensor] = None, post_weight: Optional[torch.Tensor] = None,
                          scale: float = 1.0) -> NormGrads:
    """The gradients of ``add_rms_norm``'s inputs from those of its outputs (dstream None: 0;
    residual None: the gradients of ``rms_norm``).  Those of the weights are fp32 sums in
    a fixed order, in their weight's type."""
    return NormGrads(*_backward(dstream, dnormed, y, residual, weight, gate, post_weight, eps, scale))


def _rows(t: torch.Tensor, name: str, like: torch.Tensor) -> torch.Tensor:
    """[rows, hidden] with a unit inner stride."""
    if t.shape != like.shape or t.dtype is not like.dtype or t.get_device() != like.get_device():
        _need_cuda(t)
        raise ValueError(f"{name} must be {tuple(like.shape)} {like.dtype} on {like.device}")
    if t.ndim != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _weight(w: torch.Tensor, name: str, y: torch.Tensor, shape) -> torch.Tensor:
    if w.shape != shape or (w.dtype is not torch.float32 and w.dtype is not y.dtype) or w.get_device() != y.get_device():
        _need_cuda(w)
        raise ValueError(f"{name} must be {tuple(shape)} in fp32 or {y.dtype} on {y.device}")
    return w if w.stride(-1) == 1 else w.contiguous()


def _fields(y, residual, weight, gate, post, eps, scale, stream=0, normed=0):
    """(tensors to be kept alive, the fields of DashNormArgs in order)."""
    _no_tangents("the norm", y, residual, weight, gate, post)
    shape, dt = y.shape, y.dtype
    if y.get_device() < 0 or dt not in _DT or not shape:
        _need_cuda(y)
        raise ValueError("y must be [..., hidden] in fp32, bf16 or fp16")
    hidden = shape[-1]
    y2 = _rows(y, "y", y)
    rows, f32 = y2.shape[0], torch.float32
    w = _weight(weight, "weight", y, (hidden,))
    keep = [y2, w]
    res = res_stride = post_at = post_f32 = gate_at = gate_f32 = 0
    gate_stride, group = hidden, rows
    if residual is not None:
        r2 = _rows(residual, "residual", y)
        keep.append(r2)
        res, res_stride = r2.data_ptr(), r2.stride(0)
    if post is not None:
        p = _weight(post, "post_weight", y, (hidden,))
        keep.append(p)
        post_at, post_f32 = p.data_ptr(), int(p.dtype is f32)
    if gate is not None:
        if gate.ndim not in (1, 2):
            raise ValueError("gate must be [hidden] or [groups, hidden]")
        groups = 1 if gate.ndim == 1 else gate.shape[0]
        g = _weight(gate, "gate", y, (hidden,) if gate.ndim == 1 else (groups, hidden))
        if rows and (groups == 0 or rows % groups):
            raise ValueError(f"{rows} rows do not divide into {groups} groups")
        keep.append(g)
        gate_at, gate_f32 = g.data_ptr(), int(g.dtype is f32)
        if g.ndim == 2:
            gate_stride, group = g.stride(0), rows // max(1, groups)
    return keep, (y2.data_ptr(), y2.stride(0), res, res_stride, w.data_ptr(), post_at, gate_at, gate_stride, stream, hidden,
                  normed, hidden, rows, max(1, group), hidden, _DT[dt], int(w.dtype is f32), post_f32, gate_f32, eps, scale, 0)


def _new(t: torch.Tensor) -> torch.Tensor:
    """A packed tensor like t (a third of the time of torch.empty)."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _forward(y, residual, weight, gate, post, eps, scale):
    normed = _new(y)
    stream = None if residual is None else _new(y)
    keep, values = _fields(y, residual, weight, gate, post, eps, scale, 0 if stream is None else stream.data_ptr(),
                           normed.data_ptr())
    if values[12]:
        _call("dash_add_norm", _NORM(*values), y.get_device())
    return stream, normed


def _backward(dstream, dnormed, y, residual, weight, gate, post, eps, scale, need=(True,) * 5):
    _no_tangents("the norm", dstream, dnormed)
    keep, values = _fields(y, residual, weight, gate, post, eps, scale)
    dh = _rows(dnormed, "dnormed", y)
    ds = None if dstream is None else _rows(dstream, "dstream", y)
    # of a plain sum both gradients are the same, and one tensor
    same = residual is not None and gate is None and post is None and scale == 1.0
    dy = _new(y) if need[0] and not same else None
    dr = _new(y) if residual is not None and (need[1] or (same and need[0])) else None
    dw = _new(weight) if need[2] else None
    dg = _new(gate) if need[3] and gate is not None else None
    dp = _new(post) if need[4] and post is not None else None
    rows, hidden = values[12], values[14]
    out = dr if same else dy, dr, dw, dg, dp
    if not rows:
        for t in (dw, dg, dp):
            if t is not None:
                t.zero_()
        return out
    at = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    # the workspace depends on sizes and on which weights there are
    key = (rows, hidden, values[13], values[15], post is None, gate is None)
    size = _SIZES.get(key)
    if size is None:
        if len(_SIZES) >= 1024:                   # (a training loop with other numbers of rows in each step)
            _SIZES.clear()
        size = _SIZES[key] = L.load().dash_add_norm_bwd_workspace_size(_BWD(*values, *(0,) * 13))
    ws = y.new_empty(size, dtype=torch.uint8)
    _call("dash_add_norm_bwd", _BWD(*values, at(ds), 0 if ds is None else ds.stride(0), dh.data_ptr(), dh.stride(0), at(dy),
                                    hidden, at(dr), hidden, at(dw), at(dp), at(dg), ws.data_ptr(), size), y.get_device())
    return out


_SIZES = {}


class _AddNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, residual, weight, gate, post, eps, scale):
        stream, normed = _forward(y, residual, weight, gate, post, eps, scale)
        ctx.save_for_backward(y, residual, weight, gate, post)
        ctx.cfg = eps, scale
        ctx.set_materialize_grads(False)
        return normed if residual is None else (stream, normed)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        y, residual, weight, gate, post = ctx.saved_tensors
        dstream, dnormed = (None, grads[0]) if residual is None else grads
        if dnormed is None:
            dnormed = torch.zeros_like(y)
        out = _backward(dstream, dnormed, y, residual, weight, gate, post, *ctx.cfg, need=ctx.needs_input_grad)
        return (*out, None, None)
