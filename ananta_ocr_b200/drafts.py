"""Speculative decoding on the paged DASH cache (``dash_tree_*`` and
``dash_draft_*`` of libdash_b200.so).

A step checks a tree of drafted tokens per sequence: token 0 is the last
sampled token (the root), every other token follows its parent, parents come
before their children.  Token i of a sequence with ``ctx`` committed tokens has
its K/V (and index key) at token ``ctx + i`` of the sequence's pages.

  tree_plan             parents -> depths, positions, masks, cache slots
  dash_sparse_attn_tree DASH attention of all drafted tokens
  verify_drafts         which tokens are kept, and the next token
  commit_drafts         the kept tokens' cache entries moved together

``e2e_decoder.DashDecoder.draft_step`` runs them as one step.  CUDA tensors only;
every non-zero library status raises.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib as L
from . import ops
from .ops import DeviceErrorWord, _need_cuda, _ptr
from .page_pool import Layers, _call, _ints, _layers
from .unlimited_dash_ops.attend_triton import _paged_kv, _routes_from


@dataclass
class TreePlan:
    """``depth``, ``row_pos``, ``row_seq`` int32 [rows]; ``mask`` int32 [rows,
    words] (bit j of the words: token j is the row's ancestor or itself);
    ``slots`` int64 [rows] (-1: no page) or None."""
    depth: torch.Tensor
    row_pos: torch.Tensor
    row_seq: torch.Tensor
    mask: torch.Tensor
    slots: Optional[torch.Tensor]


def tree_plan(parents: Optional[torch.Tensor], cu_seqlens_q: torch.Tensor, ctx_lens: torch.Tensor, *,
              rows: int, max_nodes: int, block_table: Optional[torch.Tensor] = None, block_size: int = 0,
              num_pages: int = 0, device_error: Optional[DeviceErrorWord] = None) -> TreePlan:
    """Positions, masks and cache slots of ``rows`` packed drafted tokens
    (``dash_tree_plan``).  ``parents`` [rows] int32: index of a token's parent
    within its sequence (-1: none); None: every sequence drafts a chain.
    ``slots`` are filled when a ``block_table`` [n_seq, W] is given."""
    _need_cuda(cu_seqlens_q, parents, block_table)
    dev = cu_seqlens_q.device
    cu = _ints(cu_seqlens_q, "cu_seqlens_q", dev)
    n_seq = cu.shape[0] - 1
    ctx = _ints(ctx_lens, "ctx_lens", dev, n_seq)
    par = _ints(parents, "parents", dev, rows)
    words = (max_nodes + 31) // 32
    # rows behind the last sequence keep these values
    buf = torch.zeros((3 + words) * rows, dtype=torch.int32, device=dev)
    depth, pos, seq = buf[:3 * rows].view(3, rows).unbind(0)
    mask = buf[3 * rows:].view(rows, words)
    a = L.DashTreePlanArgs()
    a.parents, a.q_start, a.ctx_len = _ptr(par), cu.data_ptr(), ctx.data_ptr()
    a.n_seq, a.rows, a.max_nodes, a.mask_words = n_seq, rows, int(max_nodes), words
    a.depth, a.row_pos, a.row_seq, a.mask = depth.data_ptr(), pos.data_ptr(), seq.data_ptr(), mask.data_ptr()
    slots = None
    if block_table is not None:
        bt = block_table if block_table.dtype == torch.int32 and block_table.stride(1) == 1 else \
            block_table.to(torch.int32).contiguous()
        if bt.shape[0] != n_seq:
            raise ValueError(f"block_table has {bt.shape[0]} rows for {n_seq} sequences")
        slots = torch.full((rows,), -1, dtype=torch.int64, device=dev)
        a.block_table, a.bt_stride, a.bt_width = bt.data_ptr(), bt.stride(0), bt.shape[1]
        a.block_size, a.num_pages, a.slots = int(block_size), int(num_pages), slots.data_ptr()
    a.device_error = device_error.ptr if device_error is not None else None
    _call("dash_tree_plan", a, dev)
    return TreePlan(depth, pos, seq, mask, slots)


@torch.no_grad()
def dash_sparse_attn_tree(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                          topk_idx: torch.Tensor, blk_bias: Optional[torch.Tensor],
                          block_table: torch.Tensor, cu_seqlens_q: torch.Tensor, ctx_lens: torch.Tensor,
                          row_pos: torch.Tensor, tree_mask: torch.Tensor, max_nodes: int,
                          num_kv_heads: int, sm_scale: float, output: torch.Tensor,
                          local_blocks: int = 0, sparse_block_size: int = 128, num_splits: int = 0,
                          lse: Optional[torch.Tensor] = None,
                          device_error: Optional[DeviceErrorWord] = None) -> None:
    """Bias-aware block-sparse attention of drafted tokens over the paged cache
    (in place; ``dash_tree_attn``), with the conventions of
    ``attend_triton.dash_sparse_attn``.

    q, output [rows, H, 128]; k/v cache [num_pages, block, Hkv, 128] (bf16 or
    fp16, block == ``sparse_block_size``); topk_idx / blk_bias [Hkv, rows, K]
    (usually one router head, expanded); block_table [n_seq, W]; cu_seqlens_q
    [n_seq + 1]; ctx_lens [n_seq] committed tokens; row_pos [rows] and tree_mask
    [rows, words] as ``tree_plan`` makes them.  A row attends its window of
    ``local_blocks * sparse_block_size`` committed tokens, its routed blocks
    (with their biases) before it, and the drafted tokens of its mask.  Rows
    from ``cu_seqlens_q[-1]`` on are left as they were.  lse [rows, H] fp32:
    natural-log sums.  num_splits: CTAs per sequence and kv head (0 = automatic)."""
    _need_cuda(q, k_cache, v_cache, topk_idx, block_table, tree_mask, output, lse)
    dev, dt = q.device, k_cache.dtype
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache), ("topk_idx", topk_idx), ("blk_bias", blk_bias),
                    ("block_table", block_table), ("tree_mask", tree_mask), ("output", output), ("lse", lse)):
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, not {dev}")
    if q.dim() != 3 or output.shape != q.shape:
        raise ValueError("q and output must be [rows, heads, head_dim]")
    rows, H, hd = q.shape
    if q.dtype != dt or v_cache.dtype != dt or output.dtype != dt:
        raise ValueError("q, k_cache, v_cache and output must have one dtype")
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.stride() != v_cache.stride() or \
            k_cache.shape[1:] != (sparse_block_size, num_kv_heads, hd):
        raise ValueError(f"caches must be [pages, {sparse_block_size}, {num_kv_heads}, {hd}] with common strides")
    for name, t in (("q", q), ("output", output), ("k_cache", k_cache)):
        if t.stride(-1) != 1:
            raise ValueError(f"{name} must have a unit inner stride")
    if topk_idx.dim() != 3 or topk_idx.shape[:2] != (num_kv_heads, rows):
        raise ValueError(f"topk_idx must be [{num_kv_heads}, {rows}, K]")
    if blk_bias is not None and (blk_bias.shape != topk_idx.shape or blk_bias.dtype != torch.float32):
        raise ValueError("blk_bias must be fp32 of topk_idx's shape")
    cu = _ints(cu_seqlens_q, "cu_seqlens_q", dev)
    n_seq = cu.shape[0] - 1
    ctx = _ints(ctx_lens, "ctx_lens", dev, n_seq)
    pos = _ints(row_pos, "row_pos", dev, rows)
    if tree_mask.dtype != torch.int32 or tree_mask.dim() != 2 or tree_mask.shape[0] != rows or \
            (tree_mask.shape[1] > 1 and tree_mask.stride(1) != 1):
        raise ValueError(f"tree_mask must be int32 [{rows}, words]")
    if block_table.dim() != 2 or block_table.shape[0] != n_seq:
        raise ValueError(f"block_table must be [{n_seq}, W]")
    bt = block_table if block_table.dtype == torch.int32 and block_table.stride(1) == 1 else \
        block_table.to(torch.int32).contiguous()
    if rows == 0 or n_seq == 0:
        return
    if topk_idx.shape[2]:
        routes, idx_keep, bias_keep = _routes_from(topk_idx, blk_bias, num_kv_heads)
    else:
        routes, idx_keep, bias_keep = ops._routes(None, None, 0, 0, 1), None, None
    a = L.DashTreeAttnArgs()
    a.seqs = ops.Seqs(n_seq=n_seq, q_start=cu, total_rows=rows, max_q_len=int(max_nodes)).c()
    a.kv = _paged_kv(k_cache, v_cache, bt, num_kv_heads)
    a.routes = routes
    lse_strides = (0, 0, 0)
    if lse is not None:
        if lse.shape != (rows, H) or lse.dtype != torch.float32:
            raise ValueError(f"lse must be fp32 [{rows}, {H}]")
        lse_strides = (0, lse.stride(0), lse.stride(1))
    a.qo = ops._qo(q, output, (0, q.stride(0), q.stride(1)), (0, output.stride(0), output.stride(1)), H,
                   lse, lse_strides)
    a.ctx_len, a.row_pos = ctx.data_ptr(), pos.data_ptr()
    a.mask, a.mask_stride, a.mask_words = tree_mask.data_ptr(), tree_mask.stride(0), tree_mask.shape[1]
    a.bt_width = bt.shape[1]
    a.scale, a.block_size = float(sm_scale), int(sparse_block_size)
    a.local_window = int(local_blocks) * int(sparse_block_size)
    a.num_splits = int(num_splits)
    a.device_error = device_error.ptr if device_error is not None else None
    _call("dash_tree_attn", a, dev)
    del idx_keep, bias_keep


@dataclass
class Verified:
    """``n_accept`` int32 [n_seq] (drafts kept, the root not counted); ``path``
    int32 [n_seq, max_nodes] (kept tokens' indices, the root's 0 first, -1
    behind); ``next_token`` int64 [n_seq]; ``tokens`` int64 [n_seq, max_nodes]
    (the kept drafts, then next_token, -1 behind)."""
    n_accept: torch.Tensor
    path: torch.Tensor
    next_token: torch.Tensor
    tokens: torch.Tensor


def verify_drafts(tokens: torch.Tensor, parents: Optional[torch.Tensor], cu_seqlens_q: torch.Tensor,
                  target: torch.Tensor, *, max_nodes: int, draft: Optional[torch.Tensor] = None,
                  u_accept: Optional[torch.Tensor] = None, u_sample: Optional[torch.Tensor] = None,
                  greedy: bool = False, device_error: Optional[DeviceErrorWord] = None) -> Verified:
    """Keeps a path of each sequence's drafted tokens and picks the next token
    (``dash_draft_verify``).

    tokens [rows] int64; parents as in ``tree_plan``; target [rows, vocab] (fp32,
    bf16 or fp16): the target's probabilities behind each row.  ``draft`` [rows,
    vocab]: the distributions that each row's children were drawn from (each
    child on its own); without it the drafts count as certain (each child named
    once).  ``u_accept`` [rows] and ``u_sample`` [n_seq]: fp32 numbers, uniform in
    [0, 1).  The kept tokens and the next one then follow the target's
    distribution.  ``greedy``: target are logits (or probabilities), a draft is kept
    where it is the row's argmax (lowest index among equals), and no random
    numbers are read."""
    _need_cuda(tokens, target, draft, u_accept, u_sample)
    dev = target.device
    cu = _ints(cu_seqlens_q, "cu_seqlens_q", dev)
    n_seq = cu.shape[0] - 1
    if target.dim() != 2 or target.dtype not in ops._DT:
        raise ValueError("target must be [rows, vocab] in fp32, bf16 or fp16")
    rows, V = target.shape
    par = _ints(parents, "parents", dev, rows)
    if tokens.shape != (rows,) or tokens.dtype != torch.int64 or tokens.device != dev:
        raise ValueError(f"tokens must be int64 [{rows}] on {dev}")
    if target.stride(1) != 1 and V > 1:
        target = target.contiguous()
    if greedy and (draft is not None or u_accept is not None or u_sample is not None):
        raise ValueError("greedy verification takes neither draft probabilities nor random numbers")
    if not greedy and (u_accept is None or u_sample is None):
        raise ValueError("u_accept and u_sample are needed unless greedy")
    if draft is not None:
        if draft.shape != target.shape or draft.dtype != target.dtype or draft.device != dev:
            raise ValueError("draft must have target's shape, dtype and device")
        if draft.stride(1) != 1 and V > 1:
            draft = draft.contiguous()
    for name, u, n in (("u_accept", u_accept, rows), ("u_sample", u_sample, n_seq)):
        if u is not None and (u.shape != (n,) or u.dtype != torch.float32 or u.device != dev):
            raise ValueError(f"{name} must be fp32 [{n}] on {dev}")
    tokens = tokens.contiguous()
    u_accept = None if u_accept is None else u_accept.contiguous()
    u_sample = None if u_sample is None else u_sample.contiguous()
    max_nodes = int(max_nodes)
    i64 = torch.empty(n_seq * (max_nodes + 1), dtype=torch.int64, device=dev)
    i32 = torch.empty(n_seq * (max_nodes + 1), dtype=torch.int32, device=dev)
    r = Verified(i32[:n_seq], i32[n_seq:].view(n_seq, max_nodes), i64[:n_seq],
                 i64[n_seq:].view(n_seq, max_nodes))
    a = L.DashVerifyArgs()
    a.tokens, a.parents, a.q_start = tokens.data_ptr(), _ptr(par), cu.data_ptr()
    a.target, a.target_stride = target.data_ptr(), target.stride(0) if rows > 1 else V
    if draft is not None:
        a.draft, a.draft_stride = draft.data_ptr(), draft.stride(0) if rows > 1 else V
    a.u_accept, a.u_sample = _ptr(u_accept), _ptr(u_sample)
    a.n_seq, a.rows, a.max_nodes, a.vocab = n_seq, rows, max_nodes, V
    a.dtype, a.mode = ops._DT[target.dtype], 2 if greedy else 0 if draft is not None else 1
    a.n_accept, a.path = r.n_accept.data_ptr(), r.path.data_ptr()
    a.next_token, a.out_tokens = r.next_token.data_ptr(), r.tokens.data_ptr()
    a.device_error = device_error.ptr if device_error is not None else None
    _call("dash_draft_verify", a, dev)
    return r


def commit_drafts(caches: Layers, path: torch.Tensor, n_accept: torch.Tensor, ctx_lens: torch.Tensor,
                  block_table: torch.Tensor, device_error: Optional[DeviceErrorWord] = None) -> None:
    """Moves the kept tokens' entries together, in every tensor of ``caches`` ([pages,
    block, ...] each): token ``ctx + path[s, i]`` -> ``ctx + i`` for 0 < i <=
    ``n_accept[s]`` (``dash_draft_commit``; path and n_accept as ``verify_drafts``
    returns them).  ``ctx_lens + 1 + n_accept`` tokens are committed afterwards;
    summaries of the touched pages (k-bar) have to be refreshed."""
    layers = _layers(caches)
    dev = layers.device
    if layers.page_tokens is None:
        raise ValueError("commit_drafts takes tensors with one entry per token")
    _need_cuda(path, block_table)
    if path.dim() != 2 or path.dtype != torch.int32 or path.device != dev or \
            (path.shape[1] > 1 and path.stride(1) != 1):
        raise ValueError(f"path must be int32 [n_seq, max_nodes] on {dev}")
    n_seq, max_nodes = path.shape
    acc = _ints(n_accept, "n_accept", dev, n_seq)
    ctx = _ints(ctx_lens, "ctx_lens", dev, n_seq)
    if block_table.dim() != 2 or block_table.shape[0] != n_seq or block_table.device != dev:
        raise ValueError(f"block_table must be [{n_seq}, W] on {dev}")
    bt = block_table if block_table.dtype == torch.int32 and block_table.stride(1) == 1 else \
        block_table.to(torch.int32).contiguous()
    a = L.DashCommitArgs()
    a.tensors, a.n_tensors = ctypes.addressof(layers.c), len(layers.c)
    a.n_seq, a.max_nodes, a.block_size = n_seq, max_nodes, layers.page_tokens
    a.bt_width, a.num_pages = bt.shape[1], layers.num_pages
    a.path, a.path_stride = path.data_ptr(), path.stride(0) if n_seq > 1 else max_nodes
    a.n_accept, a.ctx_len = acc.data_ptr(), ctx.data_ptr()
    a.block_table, a.bt_stride = bt.data_ptr(), bt.stride(0) if n_seq > 1 else bt.shape[1]
    a.device_error = device_error.ptr if device_error is not None else None
    _call("dash_draft_commit", a, dev)
