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

from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib as L
from . import ops
from .ops import DeviceErrorWord, _need_cuda, _ptr
from .page_pool import Layers, _call, _ints, _layers


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
    dev, index = cu_seqlens_q.device, cu_seqlens_q.get_device()
    cu = _ints(cu_seqlens_q, "cu_seqlens_q", index)
    n_seq = cu.shape[0] - 1
    ctx = _ints(ctx_lens, "ctx_lens", index, n_seq)
    par = _ints(parents, "parents", index, rows)
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
        bt = _table(block_table, index, n_seq)
        slots = torch.full((rows,), -1, dtype=torch.int64, device=dev)
        a.block_table, a.bt_stride, a.bt_width = bt.data_ptr(), bt.stride(0), bt.shape[1]
        a.block_size, a.num_pages, a.slots = int(block_size), int(num_pages), slots.data_ptr()
    a.device_error = device_error.ptr if device_error is not None else None
    _call("dash_tree_plan", a, index)
    return TreePlan(depth, pos, seq, mask, slots)


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
    (usually one router head, both expanded: anything else is copied first); block_table [n_seq, W]; cu_seqlens_q
    [n_seq + 1]; ctx_lens [n_seq] committed tokens; row_pos [rows] and tree_mask
    [rows, words] as ``tree_plan`` makes them.  A row attends its window of
    ``local_blocks * sparse_block_size`` committed tokens, its routed blocks
    (with their biases) before it, and the drafted tokens of its mask, however far
    back: the keys are those of decoding the path token by token as long as no
    token lies ``local_blocks * sparse_block_size`` or more below the root.  Rows
    from ``cu_seqlens_q[-1]`` on are left as they were.  output may be q itself.
    lse [rows, H] fp32: natural-log sums.  num_splits: CTAs per sequence and kv head
    (0 = automatic)."""
    index, dt = q.get_device(), q.dtype
    qs, ks, ts, ms = q.shape, k_cache.shape, topk_idx.shape, tree_mask.shape
    qst, kst, ist = q.stride(), k_cache.stride(), topk_idx.stride()
    # the usual call passes one test; what is wrong with any other is said below
    if not (len(qs) == 3 == len(ts) and len(ks) == 4 and output.shape == qs and
            ks == v_cache.shape and kst == v_cache.stride() and
            ks[1] == sparse_block_size and ks[2] == num_kv_heads and ks[3] == qs[2] and
            dt is k_cache.dtype is v_cache.dtype is output.dtype and
            index == k_cache.get_device() == v_cache.get_device() == output.get_device() ==
            topk_idx.get_device() == tree_mask.get_device() and index >= 0):
        _refuse_tree(q, k_cache, v_cache, output, topk_idx, tree_mask, sparse_block_size, num_kv_heads)
    rows, H, D = qs
    if rows == 0:
        return
    ost = output.stride()
    if qst[2] != 1 or ost[2] != 1 or kst[3] != 1:
        raise ValueError("q, output and the caches must have a unit inner stride")
    HI, trows, K = ts
    if HI != num_kv_heads or trows != rows:
        raise ValueError(f"topk_idx must be [{num_kv_heads}, {rows}, K]")
    mst = tree_mask.stride()
    if tree_mask.dtype is not torch.int32 or len(ms) != 2 or ms[0] != rows or (ms[1] > 1 and mst[1] != 1):
        raise ValueError(f"tree_mask must be int32 [{rows}, words]")
    cu = _ints(cu_seqlens_q, "cu_seqlens_q", index)
    n_seq = cu.numel() - 1
    ctx = _ints(ctx_lens, "ctx_lens", index, n_seq)
    pos = _ints(row_pos, "row_pos", index, rows)
    bt = _table(block_table, index, n_seq)
    if n_seq == 0:
        return
    idx = bias = 0
    bst = ist
    if blk_bias is not None:
        if blk_bias.shape != ts or blk_bias.dtype is not torch.float32 or blk_bias.get_device() != index:
            raise ValueError(f"blk_bias must be fp32 of topk_idx's shape on cuda:{index}")
        bst = blk_bias.stride()
    # a router head that all kv heads share: ids and biases both
    one = ist[0] == 0 == bst[0] or num_kv_heads == 1
    if K:
        if topk_idx.dtype is not torch.int32 or ist[2] != 1 or bst != ist:
            # one layout for both; a shared router head is kept once
            topk_idx = (topk_idx[:1] if one else topk_idx).to(torch.int32).contiguous()
            if blk_bias is not None:
                blk_bias = (blk_bias[:1] if one else blk_bias).contiguous()
            ist = topk_idx.stride()
        idx = topk_idx.data_ptr()
        if blk_bias is not None:
            bias = blk_bias.data_ptr()
    z, zst = 0, (0, 0)
    if lse is not None:
        if lse.shape != (rows, H) or lse.dtype is not torch.float32 or lse.get_device() != index:
            raise ValueError(f"lse must be fp32 [{rows}, {H}] on cuda:{index}")
        z, zst = lse.data_ptr(), lse.stride()
    _call("dash_tree_attn", _TREE(
        # seqs: n_seq, q_len_fixed (all rows), kv_len_fixed, max_q_len, q_start, pos0, kv_len
        n_seq, rows, 0, max_nodes, cu.data_ptr(), 0, 0,
        # kv: k, v, dtype, n_kv_heads, head_dim, pad, strides of a page, a token, a head, table, its stride, num_pages
        k_cache.data_ptr(), v_cache.data_ptr(), ops._DT.get(dt, -1), num_kv_heads, D, 0, kst[0], kst[1], kst[2],
        bt.data_ptr(), bt.stride(0), ks[0],
        # routes: idx, bias, row_stride, ihead_stride, K, n_index_heads
        idx, bias, ist[1], 0 if one else ist[0], K, 1 if one else num_kv_heads,
        # qo: q, out, q strides, out strides (sequence, token, head), n_heads, pad, lse, its strides
        q.data_ptr(), output.data_ptr(), 0, qst[0], qst[1], 0, ost[0], ost[1], H, 0, z, 0, zst[0], zst[1],
        # ctx_len, row_pos, mask, mask_stride, mask_words, bt_width, scale
        ctx.data_ptr(), pos.data_ptr(), tree_mask.data_ptr(), mst[0], ms[1], bt.shape[1], sm_scale,
        # block_size, local_window, num_splits, device_error
        sparse_block_size, local_blocks * sparse_block_size, num_splits,
        device_error.ptr if device_error is not None else 0), index)


_TREE = L.packer(L.DashTreeAttnArgs)


def _table(block_table: torch.Tensor, index: int, n_seq: int) -> torch.Tensor:
    """The block table as int32 rows of unit inner stride."""
    shape = block_table.shape
    if len(shape) != 2 or shape[0] != n_seq or block_table.get_device() != index:
        _need_cuda(block_table)
        raise ValueError(f"block_table must be [{n_seq}, W] on cuda:{index}")
    return block_table if block_table.dtype is torch.int32 and block_table.stride(1) == 1 else \
        block_table.to(torch.int32).contiguous()


def _refuse_tree(q, k_cache, v_cache, output, topk_idx, tree_mask, block, n_kv):
    _need_cuda(q, k_cache, v_cache, output, topk_idx, tree_mask)
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache), ("output", output), ("topk_idx", topk_idx),
                    ("tree_mask", tree_mask)):
        if t.device != q.device:
            raise ValueError(f"{name} is on {t.device}, not {q.device}")
    if q.dim() != 3 or output.shape != q.shape:
        raise ValueError("q and output must be [rows, heads, head_dim]")
    if not q.dtype == k_cache.dtype == v_cache.dtype == output.dtype:
        raise ValueError("q, k_cache, v_cache and output must have one dtype")
    if topk_idx.dim() != 3:
        raise ValueError("topk_idx must be [kv heads, rows, K]")
    raise ValueError(f"caches must be [pages, {block}, {n_kv}, {q.shape[2]}] with common strides")


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
    index = target.get_device()
    if index < 0:
        _need_cuda(target)
    cu = _ints(cu_seqlens_q, "cu_seqlens_q", index)
    n_seq = cu.numel() - 1
    if target.ndim != 2 or target.dtype not in ops._DT:
        raise ValueError("target must be [rows, vocab] in fp32, bf16 or fp16")
    rows, V = target.shape
    par = _ints(parents, "parents", index, rows)
    if tokens.ndim != 1 or tokens.numel() != rows or tokens.dtype is not torch.int64 or tokens.get_device() != index:
        raise ValueError(f"tokens must be int64 [{rows}] on cuda:{index}")
    if greedy:
        if draft is not None or u_accept is not None or u_sample is not None:
            raise ValueError("greedy verification takes neither draft probabilities nor random numbers")
    else:
        if u_accept is None or u_sample is None:
            raise ValueError("u_accept and u_sample are needed unless greedy")
        for name, u, n in (("u_accept", u_accept, rows), ("u_sample", u_sample, n_seq)):
            if u.ndim != 1 or u.numel() != n or u.dtype is not torch.float32 or u.get_device() != index:
                raise ValueError(f"{name} must be fp32 [{n}] on cuda:{index}")
        u_accept, u_sample = u_accept.contiguous(), u_sample.contiguous()
    tst = target.stride()
    if tst[1] != 1 and V > 1:
        target = target.contiguous()
        tst = target.stride()
    tokens = tokens.contiguous()
    dev, i32, i64 = target.device, torch.int32, torch.int64
    r = Verified(torch.empty(n_seq, dtype=i32, device=dev), torch.empty(n_seq, max_nodes, dtype=i32, device=dev),
                 torch.empty(n_seq, dtype=i64, device=dev), torch.empty(n_seq, max_nodes, dtype=i64, device=dev))
    q = q_stride = 0
    if draft is not None:
        if draft.shape != target.shape or draft.dtype is not target.dtype or draft.get_device() != index:
            raise ValueError("draft must have target's shape, dtype and device")
        if draft.stride(1) != 1 and V > 1:
            draft = draft.contiguous()
        q, q_stride = draft.data_ptr(), draft.stride(0) if rows > 1 else V
    _call("dash_draft_verify", _VERIFY(
        # tokens, parents, q_start, target, target_stride, draft, draft_stride
        tokens.data_ptr(), 0 if par is None else par.data_ptr(), cu.data_ptr(), target.data_ptr(),
        tst[0] if rows > 1 else V, q, q_stride,
        # u_accept, u_sample, n_seq, rows, max_nodes, vocab, dtype, mode
        0 if greedy else u_accept.data_ptr(), 0 if greedy else u_sample.data_ptr(), n_seq, rows, max_nodes, V,
        ops._DT[target.dtype], 2 if greedy else 1 if draft is None else 0,
        # n_accept, path, next_token, out_tokens, device_error
        r.n_accept.data_ptr(), r.path.data_ptr(), r.next_token.data_ptr(), r.tokens.data_ptr(),
        device_error.ptr if device_error is not None else 0), index)
    return r


_VERIFY = L.packer(L.DashVerifyArgs)


def commit_drafts(caches: Layers, path: torch.Tensor, n_accept: torch.Tensor, ctx_lens: torch.Tensor,
                  block_table: torch.Tensor, device_error: Optional[DeviceErrorWord] = None) -> None:
    """Moves the kept tokens' entries together, in every tensor of ``caches`` ([pages,
    block, ...] each): token ``ctx + path[s, i]`` -> ``ctx + i`` for 0 < i <=
    ``n_accept[s]`` (``dash_draft_commit``; path and n_accept as ``verify_drafts``
    returns them).  ``ctx_lens + 1 + n_accept`` tokens are committed afterwards;
    summaries of the touched pages (k-bar) have to be refreshed."""
    layers = _layers(caches)
    index = layers.index
    if layers.page_tokens is None:
        raise ValueError("commit_drafts takes tensors with one entry per token")
    shape = path.shape
    if len(shape) != 2 or path.dtype is not torch.int32 or path.get_device() != index or \
            (shape[1] > 1 and path.stride(1) != 1):
        raise ValueError(f"path must be int32 [n_seq, max_nodes] on cuda:{index}")
    n_seq, max_nodes = shape
    acc = _ints(n_accept, "n_accept", index, n_seq)
    ctx = _ints(ctx_lens, "ctx_lens", index, n_seq)
    bt = _table(block_table, index, n_seq)
    many = n_seq > 1
    _call("dash_draft_commit", _COMMIT(
        # tensors, n_tensors, n_seq, max_nodes, block_size, bt_width, pad, num_pages, path, path_stride
        layers.address, layers.n, n_seq, max_nodes, layers.page_tokens, bt.shape[1], 0, layers.num_pages,
        path.data_ptr(), path.stride(0) if many else max_nodes,
        # n_accept, ctx_len, block_table, bt_stride, device_error
        acc.data_ptr(), ctx.data_ptr(), bt.data_ptr(), bt.stride(0) if many else bt.shape[1],
        device_error.ptr if device_error is not None else 0), index)


_COMMIT = L.packer(L.DashCommitArgs)
