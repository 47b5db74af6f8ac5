"""The next token of a batch of rows from logits and given random numbers
(``dash_sample`` of libdash_b200.so).

  sample   a token per row
  probs    the distribution that ``sample`` draws from (a target for
           ``drafts.verify_drafts``)

Both take logits [rows, vocab] (fp32, bf16, fp16) and four settings, each a number
or a tensor of one per row:

  temperature   logits are divided by it; 0 or less: the largest logit alone
  top_k         that many of the largest are kept (0 or less: all)
  top_p         of those the shortest head, in descending order, that holds this share of
                their probability (1 or more: all; the first is always kept)
  min_p         of those the ones with at least this share of the largest's probability

Among equal logits the lowest index comes first.  -inf and NaN are never kept.
Nothing waits for the GPU; a call can be captured into a CUDA graph.  CUDA tensors
only; every non-zero library status raises.
"""
from __future__ import annotations

from typing import Union

import torch

from . import _lib as L
from .ops import _DT, _need_cuda, _no_tangents
from .page_pool import _call, _ints

Setting = Union[float, torch.Tensor]
_ARGS = L.packer(L.DashSampleArgs)


def sample(logits: torch.Tensor, u: torch.Tensor, *, temperature: Setting = 1.0, top_k: Union[int, torch.Tensor] = 0,
           top_p: Setting = 1.0, min_p: Setting = 0.0) -> torch.Tensor:
    """int64 [rows]: the first kept token whose running sum of probabilities, in the
    vocabulary's order, exceeds u (fp32 [rows], in [0, 1)); -1 where nothing is kept."""
    rows = _check(logits)
    if u.shape != (rows,) or u.dtype is not torch.float32 or u.get_device() != logits.get_device():
        _need_cuda(u)
        raise ValueError(f"u must be fp32 [{rows}] on {logits.device}")
    tokens = logits.new_empty(rows, dtype=torch.int64)
    _run(logits, rows, u.contiguous(), temperature, top_k, top_p, min_p, tokens, None)
    return tokens


def probs(logits: torch.Tensor, *, temperature: Setting = 1.0, top_k: Union[int, torch.Tensor] = 0, top_p: Setting = 1.0,
          min_p: Setting = 0.0) -> torch.Tensor:
    """fp32 [rows, vocab]: the kept tokens' probabilities, 0 for the others and for those below 2^-44
    of the largest's (a row that keeps nothing is all 0).  No gradients: logits and settings that ask for them, or
    carry tangents, are refused."""
    rows = _check(logits)
    if torch.is_grad_enabled():
        for t in (logits, temperature, top_p, min_p):
            if torch.is_tensor(t) and t.requires_grad:
                raise NotImplementedError("probs has no gradients")
    _no_tangents("probs", logits, temperature, top_p, min_p)
    out = logits.new_empty(logits.shape, dtype=torch.float32)
    _run(logits, rows, None, temperature, top_k, top_p, min_p, None, out)
    return out


def _check(logits: torch.Tensor) -> int:
    if logits.dim() != 2 or logits.dtype not in _DT or logits.get_device() < 0:
        _need_cuda(logits)
        raise ValueError("logits must be [rows, vocab] in fp32, bf16 or fp16")
    return logits.shape[0]


def _run(logits, rows, u, temperature, top_k, top_p, min_p, tokens, out):
    if rows == 0:
        return
    index, V = logits.get_device(), logits.shape[1]
    if logits.stride(1) != 1 and V > 1:
        logits = logits.contiguous()
    keep = []

    def floats(v, name):
        """(address, number for all rows)"""
        if not torch.is_tensor(v):
            return 0, float(v)
        if v.shape != (rows,) or v.dtype is not torch.float32 or v.get_device() != index:
            raise ValueError(f"{name} must be a number or fp32 [{rows}] on cuda:{index}")
        keep.append(v.contiguous())
        return keep[-1].data_ptr(), 0.0

    t, ta = floats(temperature, "temperature")
    p, pa = floats(top_p, "top_p")
    m, ma = floats(min_p, "min_p")
    if torch.is_tensor(top_k):
        # (64-bit numbers do not wrap: those beyond the vocabulary keep all, as they are)
        keep.append(_ints(top_k.clamp(0, V) if top_k.dtype is torch.int64 else top_k, "top_k", index, rows))
        k, ka = keep[-1].data_ptr(), 0
    else:
        k, ka = 0, max(0, min(int(top_k), V))
    _call("dash_sample", _ARGS(
        logits.data_ptr(), logits.stride(0) if rows > 1 else V, 0 if u is None else u.data_ptr(), t, k, p, m, ta, ka, pa,
        ma, rows, V, _DT[logits.dtype], 0, 0 if tokens is None else tokens.data_ptr(),
        0 if out is None else out.data_ptr(), V), index)
