"""A whole mixture-of-experts layer for a few tokens (``dash_moe`` of libdash_b200.so):
a decoding step's, or a tree's of drafted tokens.

  MoeWeights   the layer's weights, named once
  moe_layer    router, top-k, the picked experts, the shared expert, the residual

Only the experts that some token picked are read.  Nothing waits for the GPU; a call
can be captured into a CUDA graph.  CUDA tensors only; every non-zero library status
raises.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib as L
from .ops import _DT, DeviceErrorWord, _need_cuda, _no_tangents
from .page_pool import _call

MAX_TOKENS = 256                  # of a call
_ARGS = L.packer(L.DashMoeArgs)


class MoeWeights:
    """Weights of a layer: gate [experts, hidden] (fp32 or the experts' type); gate_up
    [experts, 2 * ffn, hidden] (a first half of gate rows, then the up rows) and down
    [experts, hidden, ffn], bf16 or fp16, contiguous; optionally one shared expert of its
    own width, [2 * shared_ffn, hidden] and [hidden, shared_ffn].  hidden and the widths
    are multiples of 8.  The handle keeps the tensors alive; it holds no copies, so that
    weights updated in place are the ones that are read, and so is other memory that a tensor
    was given (``.data``, a module's ``to``), which is looked over as at first."""

    def __init__(self, gate: torch.Tensor, gate_up: torch.Tensor, down: torch.Tensor,
                 shared_gate_up: Optional[torch.Tensor] = None, shared_down: Optional[torch.Tensor] = None):
        self.tensors = [gate, gate_up, down, shared_gate_up, shared_down]
        self._check()

    def _check(self):
        self.seen = None
        gate, gate_up, down, shared_gate_up, shared_down = self.tensors
        _need_cuda(*self.tensors)
        if gate_up.dim() != 3 or down.dim() != 3 or gate.dim() != 2:
            raise ValueError("gate must be [experts, hidden], gate_up [experts, 2 * ffn, hidden], down [experts, hidden, ffn]")
        E, two, H = gate_up.shape
        F = two // 2
        if (shared_gate_up is None) != (shared_down is None):
            raise ValueError("a shared expert has both gate_up and down")
        S = 0 if shared_down is None else shared_down.shape[-1]
        want = [(E, H), (E, 2 * F, H), (E, H, F), (2 * S, H), (H, S)]
        for name, t, shape in zip(("gate", "gate_up", "down", "shared_gate_up", "shared_down"), self.tensors, want):
            if t is None:
                continue
            if tuple(t.shape) != shape or t.device != gate_up.device or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous {list(shape)} on {gate_up.device}, got {list(t.shape)}")
            if t.dtype is not gate_up.dtype and not (name == "gate" and t.dtype is torch.float32):
                raise ValueError(f"{name} must be of gate_up's type {gate_up.dtype}")
        if gate_up.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("the experts must be bf16 or fp16")
        self.index, self.device, self.dtype = gate_up.get_device(), gate_up.device, gate_up.dtype
        self.experts, self.hidden, self.ffn, self.shared_ffn = E, H, F, S
        self.gate_f32 = 1 if gate.dtype is torch.float32 else 0
        self._sizes = {}
        self.given = [t for t in self.tensors if t is not None]
        self.seen = [t.data_ptr() for t in self.given], [t.dtype for t in self.given]

    def addresses(self):
        """Of the tensors as they are now (0: none)."""
        if self.seen is None or self.seen[0] != [t.data_ptr() for t in self.given] or \
                self.seen[1] != [t.dtype for t in self.given]:
            self._check()
        at = self.seen[0]
        return at if len(at) == 5 else [*at, 0, 0]

    def workspace_bytes(self, tokens: int, topk: int) -> int:
        n = self._sizes.get((tokens, topk))
        if n is None:
            a = L.DashMoeArgs()
            a.tokens, a.hidden, a.ffn, a.experts, a.topk = tokens, self.hidden, self.ffn, self.experts, topk
            a.shared_ffn, a.dtype = self.shared_ffn, _DT[self.dtype]
            n = self._sizes[tokens, topk] = L.load().dash_moe_workspace_size(a)
        return n


class MoeOut(NamedTuple):
    """``out`` [tokens, hidden]; ``ids`` int32 and ``weights`` fp32 [tokens, topk], the
    best expert first."""
    out: torch.Tensor
    ids: torch.Tensor
    weights: torch.Tensor


def moe_layer(x: torch.Tensor, weights: MoeWeights, topk: int, *, renormalize: bool = False, scale: float = 1.0,
              residual: Optional[torch.Tensor] = None, device_error: Optional[DeviceErrorWord] = None) -> MoeOut:
    """out = residual + sum_j w_j FFN_{ids_j}(x) + FFN_shared(x), with FFN(x) = down (silu(g) *
    u), (g, u) = gate_up x; ids are the topk experts of the largest gate scores (lowest
    index among equals), w their softmax over all experts (``renormalize``: over the
    picked ones) times ``scale``.

    x, residual [tokens, hidden] of the weights' type, at most 256 tokens; no gradients (inputs and
    weights that ask for them, or carry tangents, are refused).  Scores are 64-bit sums, everything
    else in fp32 (the FFN's inner values as the sum of two numbers of the weights' type), and
    rounded once."""
    at = weights.addresses()
    if x.dim() != 2 or x.shape[1] != weights.hidden or x.dtype is not weights.dtype or x.get_device() != weights.index:
        _need_cuda(x)
        raise ValueError(f"x must be [tokens, {weights.hidden}] {weights.dtype} on {weights.device}")
    if residual is not None and (residual.shape != x.shape or residual.dtype is not x.dtype or
                                 residual.get_device() != weights.index):
        raise ValueError("residual must have x's shape, type and device")
    if torch.is_grad_enabled():
        for v in (x, *weights.given) if residual is None else (x, residual, *weights.given):
            if v.requires_grad:
                raise NotImplementedError("moe_layer has no gradients")
    _no_tangents("moe_layer", x, residual, *weights.tensors)
    T = x.shape[0]
    x = _aligned(x)
    res = None if residual is None else _aligned(residual)
    out = x.new_empty(x.shape)
    ids = x.new_empty((T, topk), dtype=torch.int32)
    w = x.new_empty((T, topk), dtype=torch.float32)
    if T:
        size = weights.workspace_bytes(T, topk)
        ws = x.new_empty(size, dtype=torch.uint8)
        _call("dash_moe", _ARGS(
            x.data_ptr(), x.stride(0), *at,
            0 if res is None else res.data_ptr(), 0 if res is None else res.stride(0), out.data_ptr(), weights.hidden,
            ids.data_ptr(), w.data_ptr(), T, weights.hidden, weights.ffn, weights.experts, topk, weights.shared_ffn,
            _DT[x.dtype], weights.gate_f32, 1 if renormalize else 0, scale, ws.data_ptr(), size,
            device_error.ptr if device_error is not None else 0), weights.index)
    return MoeOut(out, ids, w)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """Rows of unit inner stride that start at 16-byte boundaries."""
    if t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1] and t.data_ptr() % 16 == 0:
        return t
    # (clone and contiguous keep the stride of a dimension of one)
    return t.new_empty(t.shape).copy_(t)
