"""The residual sum behind a block and the norm before the next one, as one kernel
(``dash_add_norm`` and ``dash_add_norm_bwd`` of libdash_b200.so).

  rms_norm                x / sqrt(mean(x^2) + eps) * weight
  add_rms_norm            residual + scale * gate * (norm of) y, and its norm
  add_rms_norm_backward   the gradients of both, as a plain call

``rms_norm`` and ``add_rms_norm`` can be differentiated.  To capture a backward pass
into a CUDA graph, call ``add_rms_norm_backward``, or make sure that no graph that was
recorded outside of the capture still holds the leaves: torch's own accumulation
nodes belong to the stream that they were made on, and ends the process otherwise.
CUDA tensors only; every non-zero library status raises.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib as L
from .ops import _DT, _need_cuda
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
    """Gradients of ``add_rms_norm``'s inputs; None where there is no such input."""
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


def _rows(t: torch.Tensor, name: str, like: Optional[torch.Tensor] = None) -> torch.Tensor:
    """[rows, hidden] with a unit inner stride."""
    if like is not None and (t.shape != like.shape or t.dtype is not like.dtype or t.device != like.device):
        _need_cuda(t)
        raise ValueError(f"{name} must be {tuple(like.shape)} {like.dtype} on {like.device}")
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _weight(w: Optional[torch.Tensor], name: str, y: torch.Tensor, shape) -> Tuple[Optional[torch.Tensor], int, int]:
    """The tensor, its address and whether it is fp32."""
    if w is None:
        return None, 0, 0
    if w.shape != shape or (w.dtype is not torch.float32 and w.dtype is not y.dtype) or w.device != y.device:
        _need_cuda(w)
        raise ValueError(f"{name} must be {tuple(shape)} in fp32 or {y.dtype} on {y.device}")
    if w.stride(-1) != 1:
        w = w.contiguous()
    return w, w.data_ptr(), 1 if w.dtype is torch.float32 else 0


def _inputs(y, residual, weight, gate, post):
    """Checked rows and weights: (y2, residual2, w, p, g, rows, hidden, group_rows)."""
    _need_cuda(y)
    if y.dtype not in _DT or y.dim() < 1:
        raise ValueError("y must be [..., hidden] in fp32, bf16 or fp16")
    hidden = y.shape[-1]
    y2 = _rows(y, "y")
    r2 = None if residual is None else _rows(residual, "residual", y)
    rows = y2.shape[0]
    w, p = _weight(weight, "weight", y, (hidden,)), _weight(post, "post_weight", y, (hidden,))
    if gate is not None and gate.dim() not in (1, 2):
        raise ValueError("gate must be [hidden] or [groups, hidden]")
    groups = 1 if gate is None or gate.dim() == 1 else gate.shape[0]
    g = _weight(gate, "gate", y, (hidden,) if gate is None or gate.dim() == 1 else (groups, hidden))
    if rows and (groups == 0 or rows % groups):
        raise ValueError(f"{rows} rows do not divide into {groups} groups")
    return y2, r2, w, p, g, rows, hidden, max(1, rows // max(1, groups))


def _values(y2, r2, w, p, g, rows, hidden, group_rows, eps, scale, stream, normed):
    """The fields of DashNormArgs in order."""
    return (y2.data_ptr(), y2.stride(0), 0 if r2 is None else r2.data_ptr(), 0 if r2 is None else r2.stride(0),
            w[1], p[1], g[1], g[0].stride(0) if g[0] is not None and g[0].dim() == 2 else hidden,
            0 if stream is None else stream.data_ptr(), hidden, 0 if normed is None else normed.data_ptr(), hidden,
            rows, group_rows, hidden, _DT[y2.dtype], w[2], p[2], g[2], eps, scale, 0)


def _forward(y, residual, weight, gate, post, eps, scale):
    y2, r2, w, p, g, rows, hidden, group_rows = _inputs(y, residual, weight, gate, post)
    stream = None if r2 is None else torch.empty(y.shape, dtype=y.dtype, device=y.device)
    normed = torch.empty(y.shape, dtype=y.dtype, device=y.device)
    if rows:
        _call("dash_add_norm", _NORM(*_values(y2, r2, w, p, g, rows, hidden, group_rows, eps, scale, stream, normed)),
              y.get_device())
    return stream, normed


def _backward(dstream, dnormed, y, residual, weight, gate, post, eps, scale, need=(True,) * 5):
    y2, r2, w, p, g, rows, hidden, group_rows = _inputs(y, residual, weight, gate, post)
    ds = None if dstream is None else _rows(dstream, "dstream", y)
    dh = _rows(dnormed, "dnormed", y)
    empty = lambda t, on: torch.empty(t.shape, dtype=t.dtype, device=t.device) if on else None  # noqa: E731
    dy, dr = empty(y, need[0]), empty(y, need[1] and residual is not None)
    dw = empty(weight, need[2])
    dg, dp = empty(gate, need[3] and gate is not None), empty(post, need[4] and post is not None)
    if not rows:
        for t in (dw, dg, dp):
            if t is not None:
                t.zero_()
        return dy, dr, dw, dg, dp
    at = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    values = _values(y2, r2, w, p, g, rows, hidden, group_rows, eps, scale, None, None) + (
        at(ds), 0 if ds is None else ds.stride(0), dh.data_ptr(), dh.stride(0), at(dy), hidden, at(dr), hidden,
        at(dw), at(dp), at(dg))
    size = L.load().dash_add_norm_bwd_workspace_size(_BWD(*values, 0, 0))
    ws = torch.empty(size, dtype=torch.uint8, device=y.device)
    _call("dash_add_norm_bwd", _BWD(*values, ws.data_ptr(), size), y.get_device())
    return dy, dr, dw, dg, dp


class _AddNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, residual, weight, gate, post, eps, scale):
        stream, normed = _forward(y, residual, weight, gate, post, eps, scale)
        ctx.save_for_backward(y, residual, weight, gate, post)
        ctx.cfg = eps, scale
        ctx.set_materialize_grads(False)
        return normed if residual is None else (stream, normed)

    @staticmethod
    def backward(ctx, *grads):
        y, residual, weight, gate, post = ctx.saved_tensors
        dstream, dnormed = (None, grads[0]) if residual is None else grads
        if dnormed is None:
            dnormed = torch.zeros_like(y)
        out = _backward(dstream, dnormed, y, residual, weight, gate, post, *ctx.cfg, need=ctx.needs_input_grad)
        return (*out, None, None)
