"""End-to-end DeepSeek-V2-style decoder with the DASH kernels as its attention.

The decoder of ANANTA_OCR (modeling_deepseekv2.py / the sglang
unlimited_ocr_v2.py model) around this library's serving path, used to measure
the attention kernels inside a whole model and to check
that a paged prefill followed by decode steps reproduces a longer prefill.
Weights are random (the trained checkpoint is not available); the layer
structure is the model's: RMSNorm, q/k/v/o projections (10 x 128 heads),
the DASH router's index branch, a dense SwiGLU FFN in the first layer and a
64-expert top-6 MoE with 2 shared experts after it (softmax gate, no top-k
renormalisation, routing scale 1), final norm, LM head on the last token.

Attention per layer, all through libdash_b200:
  rope_and_store_kv   rotate q in place; rotated k and v into the paged cache
  index_qk_fused      index projections + RMSNorm + RoPE; idx_k into the paged
                      index cache
  kbar refresh        k-bar summaries of the pages written this step
  route_*_triton      scores + 1.5-entmax + top-K over the paged k-bar, with
                      page-aware candidates when the token ids are given
                      (PageIsolationState, once per forward for all layers)
  dash_sparse_attn*   paged prefill (tcgen05) / decode (split-KV) attention
The GEMMs and the MoE are PyTorch (cuBLAS).  ``decode_step`` allocates nothing
that changes between steps and is captured in a CUDA graph by the caller.

``draft_step`` checks a tree of drafted tokens per sequence in one pass over the
layers (speculative decoding, drafts.py), keeps a path of it and commits its cache
entries.  With ``pool_pages`` the sequences draw their pages from a page_pool.PagePool
instead of owning a fixed part of the cache; ``fork`` continues one sequence in
another row, sharing its full pages when there is a pool.  Nothing waits for the
GPU: a token without a page (the pool is empty, the row is full) or a malformed
tree is recorded in ``errors``.  A draft without a page is passed over, as if it
had not been drafted.  A row whose next token has no page stays as long as its
pages allow and its tokens mean nothing from there on; other rows are not touched.

With ``fused_steps`` the steps take the residual sums with their norms and the MoE
layers as kernels of this library (norms.py, moe.py: only the picked experts are
read, gate scores are not rounded to bf16 as the default's are).  ``decode_step`` and
``draft_step`` can draw tokens with top-k, top-p and min-p (sampling.py).
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import List, Optional, Sequence

import torch
import torch.nn.functional as F

from . import drafts, moe, norms, sampling
from .ops import DeviceErrorWord
from .page_pool import CacheLayers, PagePool, copy_pages
from .unlimited_dash_ops import attend_triton as AT
from .unlimited_dash_ops import decode_meta_triton as DM
from .unlimited_dash_ops import index_frontend as IF
from .unlimited_dash_ops import page_state as PS
from .unlimited_dash_ops import route_triton as RT


@dataclass
class DecoderConfig:
    hidden: int = 1280
    heads: int = 10
    kv_heads: int = 10
    head_dim: int = 128
    layers: int = 12
    vocab: int = 129280
    dense_ffn: int = 6848
    moe_ffn: int = 896
    experts: int = 64
    topk: int = 6
    shared: int = 2
    first_dense: int = 1
    eps: float = 1e-6
    rope_theta: float = 500000.0
    # the checkpoint's DASH settings (config.json: sparse_block_size 32,
    # sparse_local_block 4, dash_topk_blocks 12) and the serving router's
    # defaults (WHL dash_router.py:16,101-105: entmax window 16, 16 output
    # slots, the last 4 of them -1)
    block_size: int = 32
    local_blocks: int = 4
    K: int = 12
    topm: int = 16
    slots: int = 16
    index_dim: int = 128
    scaling: float = 128.0
    prior_floor: float = 1e-4
    sigma: float = 1.0


def rmsnorm(x, w, eps):
    x32 = x.float()
    x32 = x32 * torch.rsqrt(x32.pow(2).mean(-1, keepdim=True) + eps)
    return (x32 * w).to(x.dtype)


class DashDecoder:
    """Random-init bf16 decoder with paged caches for ``batch`` sequences of
    up to ``max_len`` tokens.  ``pool_pages``: that many pages shared by the
    sequences through a page pool (default: a fixed set for each).  ``fused_steps``:
    decode and draft steps of up to 256 tokens with fused norms and MoE layers."""

    def __init__(self, cfg: DecoderConfig, batch: int, max_len: int, device, seed: int = 0,
                 page_cfg=None, page_mask: bool = False, pool_pages: int = 0, fused_steps: bool = False):
        self.cfg = c = cfg
        self.B = batch
        self.dev = device
        g = torch.Generator(device=device).manual_seed(seed)
        bf = torch.bfloat16

        def rnd(*shape, std):
            return (torch.randn(*shape, generator=g, device=device) * std).to(bf)

        H = c.hidden
        self.embed = rnd(c.vocab, H, std=0.02)
        self.lm_head = rnd(c.vocab, H, std=1.0 / math.sqrt(H))
        self.final_norm = torch.ones(H, device=device)
        self.layers: List[dict] = []
        for li in range(c.layers):
            L = dict(ln1=torch.ones(H, device=device), ln2=torch.ones(H, device=device),
                     wqkv=rnd(3 * H, H, std=1.0 / math.sqrt(H)),
                     wo=rnd(H, H, std=1.0 / math.sqrt(H)),
                     wiq=rnd(c.index_dim, H, std=1.0 / math.sqrt(H)),
                     wik=rnd(c.index_dim, H, std=1.0 / math.sqrt(H)),
                     niq=torch.zeros(c.index_dim, device=device),
                     nik=torch.zeros(c.index_dim, device=device),
                     head_cls=torch.zeros(c.index_dim, device=device))
            if li < c.first_dense:
                L["dense_gu"] = rnd(2 * c.dense_ffn, H, std=1.0 / math.sqrt(H))
                L["dense_d"] = rnd(H, c.dense_ffn, std=1.0 / math.sqrt(c.dense_ffn))
            else:
                L["gate"] = rnd(c.experts, H, std=1.0 / math.sqrt(H))
                L["exp_gu"] = rnd(c.experts, 2 * c.moe_ffn, H, std=1.0 / math.sqrt(H))
                L["exp_d"] = rnd(c.experts, H, c.moe_ffn, std=1.0 / math.sqrt(c.moe_ffn))
                sf = c.shared * c.moe_ffn
                L["sh_gu"] = rnd(2 * sf, H, std=1.0 / math.sqrt(H))
                L["sh_d"] = rnd(H, sf, std=1.0 / math.sqrt(sf))
            self.layers.append(L)
        self.fused_steps = fused_steps
        # paged caches: one block of block_size tokens per page, random block table
        bs = c.block_size
        self.pps = -(-max_len // bs)
        self.capacity = self.pps * bs                                   # tokens that a row's table holds
        P = batch * self.pps
        self.num_pages = P
        self.block_table = torch.randperm(P, generator=g, device=device).to(torch.int32).view(batch, self.pps).contiguous()
        self.pool = None
        self.errors = DeviceErrorWord(device)
        self.rows = torch.arange(batch, dtype=torch.int32, device=device)
        self.one_each = torch.arange(batch + 1, dtype=torch.int32, device=device)
        if pool_pages:
            self.num_pages = P = pool_pages
            self.pool = PagePool(P, batch, self.pps, bs, device)
            self.block_table = self.pool.block_table
        self.kc = [torch.zeros(P, bs, c.kv_heads, c.head_dim, dtype=bf, device=device) for _ in range(c.layers)]
        self.vc = [torch.zeros_like(self.kc[0]) for _ in range(c.layers)]
        self.ic = [torch.zeros(P, bs, c.index_dim, device=device) for _ in range(c.layers)]
        self.kbar = [torch.zeros(P, c.index_dim, device=device) for _ in range(c.layers)]
        # the caches of all layers: per token (commits), and with the k-bar rows (page copies)
        self.token_caches = CacheLayers(self.kc + self.vc + self.ic)
        self.page_caches = CacheLayers(self.kc + self.vc + self.ic + [k[:, None] for k in self.kbar])
        self.seq_lens = torch.zeros(batch, dtype=torch.int32, device=device)
        inv = 1.0 / (c.rope_theta ** (torch.arange(0, c.head_dim // 2, device=device).float() / (c.head_dim // 2)))
        self.inv_freq = inv
        # decode-step buffers (fixed addresses for graph replay)
        self.tok = torch.zeros(batch, dtype=torch.int64, device=device)
        self.oi = torch.empty(batch, c.slots, dtype=torch.int32, device=device)
        self.ob = torch.empty(batch, c.slots, dtype=torch.float32, device=device)
        self.attn_out = torch.empty(batch, c.heads, c.head_dim, dtype=bf, device=device)
        self.dec_ws = torch.empty(16 << 20, dtype=torch.uint8, device=device)
        self.idx_scale = c.scaling / math.sqrt(c.index_dim)
        # page-aware candidates (image_token_id / page_token_id / per_page_image_tokens)
        self.pst = PS.PageIsolationState(page_cfg, bs) if page_cfg is not None else None
        # page_mask: pass the reference's dense [rows, max_block] allow mask
        # (build_query_allow / decode_allow_fused) instead of the compact domain
        self.page_mask = page_mask
        self.qpage = torch.empty(batch, dtype=torch.int32, device=device)

    # ---------------------------------------------------------------- pieces
    def rope_tables(self, pos):
        ang = pos.float()[:, None] * self.inv_freq[None, :]
        emb = torch.cat([ang, ang], -1)
        return emb.cos().to(torch.bfloat16), emb.sin().to(torch.bfloat16)

    def slots_of(self, pos, req):
        bs = self.cfg.block_size
        page = self.block_table[req, (pos // bs)].long()
        return page * bs + pos % bs

    def ffn_prefill(self, L, h):
        c = self.cfg
        if "dense_gu" in L:
            g, u = F.linear(h, L["dense_gu"]).chunk(2, -1)
            return F.linear(F.silu(g) * u, L["dense_d"])
        out = torch.zeros(h.shape, dtype=torch.float32, device=h.device)
        g, u = F.linear(h, L["sh_gu"]).chunk(2, -1)
        out += F.linear(F.silu(g) * u, L["sh_d"]).float()
        probs = F.linear(h, L["gate"]).float().softmax(-1)
        w, idx = probs.topk(c.topk, dim=-1)
        flat = idx.reshape(-1)
        order = torch.argsort(flat, stable=True)
        counts = torch.bincount(flat, minlength=c.experts).tolist()
        tok = order // c.topk
        wt = w.reshape(-1)[order]
        xs = h[tok]
        start = 0
        for e in range(c.experts):
            n = counts[e]
            if n == 0:
                continue
            seg = slice(start, start + n)
            gg, uu = F.linear(xs[seg], L["exp_gu"][e]).chunk(2, -1)
            y = F.linear(F.silu(gg) * uu, L["exp_d"][e]).float() * wt[seg, None]
            out.index_add_(0, tok[seg], y)
            start += n
        return out.to(h.dtype)

    def ffn_decode(self, L, h):
        """Every expert on every decode token, weighted by the (mostly zero)
        gates: static shapes for graph replay; the expert weights are read
        once per step either way."""
        c = self.cfg
        if "dense_gu" in L:
            return self.ffn_prefill(L, h)
        g, u = F.linear(h, L["sh_gu"]).chunk(2, -1)
        out = F.linear(F.silu(g) * u, L["sh_d"]).float()
        probs = F.linear(h, L["gate"]).float().softmax(-1)
        w, idx = probs.topk(c.topk, dim=-1)
        gates = torch.zeros(h.shape[0], c.experts, device=h.device).scatter(1, idx, w)
        gu = torch.matmul(L["exp_gu"], h.t())                       # [E, 2F, B]
        gg, uu = gu.split(c.moe_ffn, dim=1)
        y = torch.matmul(L["exp_d"], F.silu(gg) * uu).float()       # [E, H, B]
        out += (y * gates.t()[:, None, :]).sum(0).t()
        return out.to(h.dtype)

    @staticmethod
    def _moe_weights(L):
        """The handle of a layer's tensors, made again when one of them is another tensor."""
        t = [L[k] for k in ("gate", "exp_gu", "exp_d", "sh_gu", "sh_d")]
        w = L.get("moe")
        if w is None or any(a is not b for a, b in zip(w.tensors, t)):
            w = L["moe"] = moe.MoeWeights(*t)
        return w

    def _step_norm(self, x, w):
        """The norm before the first layer of a decode or draft step."""
        return (norms.rms_norm if self.fused_steps else rmsnorm)(x, w, self.cfg.eps)

    def _step_layer(self, li, x, attn):
        """What a decode or draft step does between a layer's attention and the next
        layer's: (x, the normed rows that the next layer, or the LM head, takes)."""
        c, L = self.cfg, self.layers[li]
        after = self.layers[li + 1]["ln1"] if li + 1 < c.layers else self.final_norm
        out = F.linear(attn, L["wo"])
        if not self.fused_steps:
            x = x + out
            x = x + self.ffn_decode(L, rmsnorm(x, L["ln2"], c.eps))
            return x, rmsnorm(x, after, c.eps)
        x, h = norms.add_rms_norm(out, x, L["ln2"], c.eps)
        if "gate" in L and h.shape[0] <= moe.MAX_TOKENS:
            x = moe.moe_layer(h, self._moe_weights(L), c.topk, residual=x, device_error=self.errors).out
            return x, norms.rms_norm(x, after, c.eps)
        return norms.add_rms_norm(self.ffn_decode(L, h), x, after, c.eps)

    # ---------------------------------------------------------------- prefill
    @torch.no_grad()
    def prefill(self, embeds: torch.Tensor, attn_events=None, token_ids=None, gen_start=None):
        """embeds [B, S, hidden] bf16 -> logits [B, vocab] of each sequence's
        last token; fills the caches (positions 0..S-1).  With ``token_ids``
        [B, S] and a page configuration, routing is restricted to the blocks of
        each query's own image page; ``gen_start`` [B] marks the positions from
        which tokens count as generated (text pages numbered as responses, as a
        decode step numbers them)."""
        c = self.cfg
        B, S, H = embeds.shape
        T = B * S
        dev = embeds.device
        if S > self.capacity:
            raise ValueError(f"sequences of {S} tokens do not fit the tables' {self.capacity}")
        x = embeds.reshape(T, H).clone()
        req = torch.arange(B, device=dev).repeat_interleave(S)
        pos = torch.arange(S, device=dev).repeat(B)
        cos, sin = self.rope_tables(pos)
        self.seq_lens.fill_(S)
        if self.pool is not None:
            pages = -(-S // c.block_size)
            if pages > self.pps or B * pages > self.num_pages:
                raise ValueError(f"{B} sequences of {S} tokens do not fit {self.num_pages} pages, {self.pps} each")
            self.pool.free(self.rows)
            self.pool.reserve(self.rows, self.seq_lens, self.errors)
        slots = self.slots_of(pos, req)
        cu = (torch.arange(B + 1, device=dev) * S).to(torch.int32)
        ctx = torch.zeros(B, dtype=torch.int32, device=dev)
        row2req = RT.prefill_row2req(cu_seqlens_q=cu, device=dev, total_q=T)
        plan = RT.kbar_all_plan(block_table=self.block_table, seq_lens=self.seq_lens,
                                context_lens=ctx, block_size=c.block_size, max_block=self.pps,
                                max_query_len=S, device=dev)
        domain = allow = None
        if self.pst is not None and token_ids is not None:
            layout = PS.BatchLayout(num_tokens=T, num_reqs=B,
                                    q_start=torch.arange(B + 1, device=dev) * S,
                                    start_pos=torch.zeros(B, dtype=torch.int64, device=dev),
                                    block_table=self.block_table, req_of_token=req,
                                    gen_start=gen_start)
            q_page = self.pst.step(token_ids.reshape(T), layout, slots,
                                   self.num_pages * c.block_size)
            domain = self.pst.candidate_domain(q_page)
            self.last_q_page = q_page
            if self.page_mask:
                allow = self.pst.build_query_allow(layout, q_page, self.pps, self.num_pages)
                domain = None
        oi = torch.empty(T, c.slots, dtype=torch.int32, device=dev)
        ob = torch.empty(T, c.slots, dtype=torch.float32, device=dev)
        attn = torch.empty(T, c.heads, c.head_dim, dtype=torch.bfloat16, device=dev)
        for li, L in enumerate(self.layers):
            if attn_events is not None:
                attn_events[li][0].record()
            h = rmsnorm(x, L["ln1"], c.eps)
            qkv = F.linear(h, L["wqkv"])
            q, k, v = qkv[:, :H], qkv[:, H:2 * H], qkv[:, 2 * H:]
            IF.rope_and_store_kv(q, k, v, cos, sin, self.kc[li], self.vc[li], slots, c.head_dim)
            idx_q, _ = IF.index_qk_fused(h, L["wiq"], L["wik"], L["niq"], L["nik"], c.eps, cos, sin,
                                         index_cache=self.ic[li], slot_mapping=slots)
            RT.kbar_refresh_tail_triton(kv_cache=self.ic[li], k_bar=self.kbar[li],
                                        block_table=self.block_table, seq_lens=self.seq_lens,
                                        head_cls=L["head_cls"], block_size=c.block_size, plan=plan)
            RT.route_prefill_triton(idx_q=idx_q, k_bar=self.kbar[li], block_table=self.block_table,
                                    seq_lens=self.seq_lens, cu_seqlens_q=cu, context_lens=ctx,
                                    row2req=row2req, image_allow=allow, out_idx=oi, out_bias=ob,
                                    max_block=self.pps, block_size=c.block_size,
                                    local_blocks=c.local_blocks, idx_scale=self.idx_scale,
                                    prior_floor=c.prior_floor, sigma=c.sigma, topm=c.topm, budget=c.K,
                                    out_slots=c.slots, page_domain=domain)
            AT.dash_sparse_attn(q.view(T, c.heads, c.head_dim), self.kc[li], self.vc[li],
                                oi[None].expand(c.kv_heads, T, c.slots), ob[None].expand(c.kv_heads, T, c.slots),
                                self.block_table, cu, self.seq_lens, ctx, S, c.kv_heads,
                                1.0 / math.sqrt(c.head_dim), attn, local_blocks=c.local_blocks,
                                sparse_block_size=c.block_size)
            if attn_events is not None:
                attn_events[li][1].record()
            x = x + F.linear(attn.view(T, H), L["wo"])
            x = x + self.ffn_prefill(L, rmsnorm(x, L["ln2"], c.eps))
        self.last_route = (oi, ob)         # the last layer's routes (tests read them)
        last = x.view(B, S, H)[:, -1]
        return F.linear(rmsnorm(last, self.final_norm, c.eps), self.lm_head)

    # ---------------------------------------------------------------- decode
    @torch.no_grad()
    def decode_step(self, u: Optional[torch.Tensor] = None, *, temperature: sampling.Setting = 1.0, top_k=0,
                    top_p: sampling.Setting = 1.0, min_p: sampling.Setting = 0.0):
        """One token per sequence: ``self.tok`` at position ``self.seq_lens``;
        returns logits [B, vocab], writes the next token into ``self.tok`` and
        advances ``self.seq_lens``.  The next token is the greedy one, or with
        random numbers ``u`` [B] drawn as ``sampling.sample`` draws it (a setting can
        be one number or one per sequence)."""
        c = self.cfg
        B, H = self.B, c.hidden
        dev = self.tok.device
        x = self.embed[self.tok]
        cos, sin = self.rope_tables(self.seq_lens)
        sl = self.seq_lens + 1
        if self.pool is not None:
            self.pool.reserve(self.rows, sl, self.errors)
        # a token behind the table's end has no slot, and the row's keys end there
        slots = drafts.tree_plan(None, self.one_each, self.seq_lens, rows=B, max_nodes=1,
                                 block_table=self.block_table, block_size=c.block_size, num_pages=self.num_pages,
                                 device_error=self.errors).slots
        sl.clamp_(max=self.capacity)
        tail = RT.kbar_tail_plan(block_table=self.block_table, seq_lens=sl,
                                 block_size=c.block_size, tail_pages=1, device=dev)
        domain = allow = None
        if self.pst is not None:
            q_page, _ = DM.decode_meta_fused(input_ids=self.tok, block_table=self.block_table,
                                             seq_lens=sl, slot_mapping=slots, page_state=self.pst,
                                             num_slots=self.num_pages * c.block_size,
                                             block_size=c.block_size, out_q_page=self.qpage)
            domain = self.pst.candidate_domain(q_page)
            if self.page_mask:
                allow = DM.decode_allow_fused(block_table=self.block_table, page_state=self.pst,
                                              q_page=q_page, seq_lens=sl, max_block=self.pps,
                                              num_blocks=self.num_pages, block_size=c.block_size)
                domain = None
        h = self._step_norm(x, self.layers[0]["ln1"])
        for li, L in enumerate(self.layers):
            qkv = F.linear(h, L["wqkv"])
            q, k, v = qkv[:, :H], qkv[:, H:2 * H], qkv[:, 2 * H:]
            IF.rope_and_store_kv(q, k, v, cos, sin, self.kc[li], self.vc[li], slots, c.head_dim)
            # index projections + index-K write + k-bar refresh of the tail pages
            idx_q, _ = IF.index_qk_fused(h, L["wiq"], L["wik"], L["niq"], L["nik"], c.eps, cos, sin,
                                         index_cache=self.ic[li], slot_mapping=slots,
                                         kbar_refresh=(self.kbar[li], tail, L["head_cls"],
                                                       c.block_size))
            RT.route_decode_triton(idx_q=idx_q, k_bar=self.kbar[li], block_table=self.block_table,
                                   seq_lens=sl, image_allow=allow, out_idx=self.oi, out_bias=self.ob,
                                   max_block=self.pps, block_size=c.block_size,
                                   local_blocks=c.local_blocks, decode_query_len=1,
                                   idx_scale=self.idx_scale, prior_floor=c.prior_floor,
                                   sigma=c.sigma, topm=c.topm, budget=c.K, out_slots=c.slots,
                                   page_domain=domain)
            AT.dash_sparse_attn_decode(q.view(B, c.heads, c.head_dim), self.kc[li], self.vc[li],
                                       self.oi[None].expand(c.kv_heads, B, c.slots),
                                       self.ob[None].expand(c.kv_heads, B, c.slots), self.block_table,
                                       sl, c.kv_heads, 1.0 / math.sqrt(c.head_dim), self.attn_out, 1,
                                       local_blocks=c.local_blocks, sparse_block_size=c.block_size,
                                       workspace=self.dec_ws)
            x, h = self._step_layer(li, x, self.attn_out.view(B, H))
        logits = F.linear(h, self.lm_head)
        if u is None:
            self.tok.copy_(logits.argmax(-1))
        else:
            drawn = sampling.sample(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
            self.tok.copy_(drawn.clamp_(min=0))                         # (-1: logits that are no numbers)
        self.seq_lens.copy_(sl)
        return logits

    # ---------------------------------------------------------------- drafts
    @torch.no_grad()
    def draft_step(self, drafted: torch.Tensor, parents: Optional[torch.Tensor] = None, *,
                   temperature: float = 0.0, draft_probs: Optional[torch.Tensor] = None,
                   u_accept: Optional[torch.Tensor] = None, u_sample: Optional[torch.Tensor] = None,
                   top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0):
        """Checks drafted tokens [B, n - 1] (int64) behind ``self.tok`` at once.

        With the root ``self.tok`` as token 0, ``parents`` [B, n] int32 gives each
        token's parent (None: chains).  temperature 0 keeps the drafts that greedy
        decoding would have chosen; otherwise the drafts are accepted against the
        softmax of logits / temperature with the random numbers ``u_accept`` [B * n]
        and ``u_sample`` [B] (``draft_probs`` [B * n, vocab]: the distributions that the
        drafts were drawn from; ``top_k``, ``top_p``, ``min_p``: the target is what
        ``sampling.probs`` keeps of the softmax).  The kept tokens' cache entries are moved
        together, the k-bar rows of their pages refreshed, ``self.seq_lens``
        advanced by the kept tokens and the root, and ``self.tok`` becomes the
        next token.  A draft without a page (the row is full, the pool is empty) or
        with an id outside the vocabulary (-1: no draft) is not kept.  Returns (drafts.Verified, logits [B, n, vocab])."""
        c = self.cfg
        if self.pst is not None:
            raise NotImplementedError("draft_step has no page-aware candidates (page state has no rewind)")
        B, H, dev = self.B, c.hidden, self.tok.device
        n = drafted.shape[1] + 1
        if n - 1 > (c.local_blocks - 1) * c.block_size:
            # a deeper token would route among blocks that hold drafts
            raise ValueError(f"{n - 1} drafts reach past the local window's whole blocks "
                             f"({(c.local_blocks - 1) * c.block_size} tokens)")
        T = B * n
        # refused before anything is written
        if drafted.shape[0] != B or (parents is not None and parents.numel() != T):
            raise ValueError(f"drafted must be [{B}, n - 1] and parents [{B}, n]")
        if temperature > 0:
            if u_accept is None or u_sample is None or u_accept.shape != (T,) or u_sample.shape != (B,):
                raise ValueError(f"a temperature needs u_accept [{T}] and u_sample [{B}]")
            if draft_probs is not None and (draft_probs.shape != (T, c.vocab) or draft_probs.dtype != torch.float32):
                raise ValueError(f"draft_probs must be fp32 [{T}, {c.vocab}]")
        tokens = torch.cat([self.tok[:, None], drafted], 1).reshape(T)
        if parents is not None:
            parents = parents.to(torch.int32).reshape(T)
        ctx = self.seq_lens
        if self.pool is not None:
            # every root has its page before any draft, so that drafts cost no row its next token
            self.pool.reserve(self.rows, ctx + 1, self.errors)
            if n > 1:
                self.pool.reserve(self.rows, (ctx + n).clamp_(max=self.capacity), self.errors)
        cu = torch.arange(B + 1, dtype=torch.int32, device=dev) * n
        plan = drafts.tree_plan(parents, cu, ctx, rows=T, max_nodes=n, block_table=self.block_table,
                                block_size=c.block_size, num_pages=self.num_pages, device_error=self.errors)
        cos, sin = self.rope_tables(plan.row_pos)
        table = self.block_table.index_select(0, plan.row_seq)          # a row per token, for the router
        sl = (plan.row_pos + 1).clamp_(max=self.capacity)
        # (an id outside the vocabulary is no draft: the verification passes it over)
        x = self.embed[tokens.clamp(0, c.vocab - 1)]
        oi = torch.empty(T, c.slots, dtype=torch.int32, device=dev)
        ob = torch.empty(T, c.slots, dtype=torch.float32, device=dev)
        attn = torch.empty(T, c.heads, c.head_dim, dtype=torch.bfloat16, device=dev)
        h = self._step_norm(x, self.layers[0]["ln1"])
        for li, L in enumerate(self.layers):
            qkv = F.linear(h, L["wqkv"])
            q, k, v = qkv[:, :H], qkv[:, H:2 * H], qkv[:, 2 * H:]
            IF.rope_and_store_kv(q, k, v, cos, sin, self.kc[li], self.vc[li], plan.slots, c.head_dim)
            idx_q, _ = IF.index_qk_fused(h, L["wiq"], L["wik"], L["niq"], L["nik"], c.eps, cos, sin,
                                         index_cache=self.ic[li], slot_mapping=plan.slots)
            RT.route_decode_triton(idx_q=idx_q, k_bar=self.kbar[li], block_table=table, seq_lens=sl,
                                   image_allow=None, out_idx=oi, out_bias=ob, max_block=self.pps,
                                   block_size=c.block_size, local_blocks=c.local_blocks, decode_query_len=1,
                                   idx_scale=self.idx_scale, prior_floor=c.prior_floor, sigma=c.sigma,
                                   topm=c.topm, budget=c.K, out_slots=c.slots)
            drafts.dash_sparse_attn_tree(q.view(T, c.heads, c.head_dim), self.kc[li], self.vc[li],
                                         oi[None].expand(c.kv_heads, T, c.slots),
                                         ob[None].expand(c.kv_heads, T, c.slots), self.block_table, cu, ctx,
                                         plan.row_pos, plan.mask, n, c.kv_heads, 1.0 / math.sqrt(c.head_dim), attn,
                                         local_blocks=c.local_blocks, sparse_block_size=c.block_size,
                                         device_error=self.errors)
            x, h = self._step_layer(li, x, attn.view(T, H))
        logits = F.linear(h, self.lm_head)
        # a draft whose keys could not be stored is passed over
        tokens = tokens.masked_fill(plan.slots < 0, -1)
        if temperature > 0:
            if top_k > 0 or top_p < 1 or min_p > 0:
                target = sampling.probs(logits, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
            else:
                target = (logits.float() / temperature).softmax(-1)
            kept = drafts.verify_drafts(tokens, parents, cu, target, max_nodes=n, draft=draft_probs,
                                        u_accept=u_accept, u_sample=u_sample, device_error=self.errors)
        else:
            kept = drafts.verify_drafts(tokens, parents, cu, logits, max_nodes=n, greedy=True, device_error=self.errors)
        drafts.commit_drafts(self.token_caches, kept.path, kept.n_accept, ctx, self.block_table, self.errors)
        now = (ctx + kept.n_accept + 1).clamp_(max=self.capacity)
        fresh = RT.kbar_all_plan(block_table=self.block_table, seq_lens=now, context_lens=ctx,
                                 block_size=c.block_size, max_block=self.pps, max_query_len=n, device=dev)
        for li, L in enumerate(self.layers):
            RT.kbar_refresh_tail_triton(kv_cache=self.ic[li], k_bar=self.kbar[li], block_table=self.block_table,
                                        seq_lens=now, head_cls=L["head_cls"], block_size=c.block_size, plan=fresh)
        self.seq_lens.copy_(now)
        self.tok.copy_(kept.next_token)
        if self.pool is not None:
            # pages that only dropped drafts reached go back
            self.pool.free(self.rows, (now + c.block_size - 1) // c.block_size)
        return kept, logits.view(B, n, -1)

    # ---------------------------------------------------------------- sequences
    @torch.no_grad()
    def fork(self, src: Sequence[int], dst: Sequence[int]) -> None:
        """Row ``dst[i]`` becomes a copy of row ``src[i]``: with a page pool full
        pages are shared and the last one is copied, without one all pages of the
        sequence are copied into the row's own."""
        if self.pst is not None:
            raise NotImplementedError("fork has no page-aware candidates")
        dev = self.tok.device
        if len(src) != len(dst) or len(set(dst)) != len(dst) or set(src) & set(dst) or \
                not all(0 <= r < self.B for r in (*src, *dst)):
            raise ValueError("fork takes distinct rows, none of them source and destination")
        if not src:
            return
        s, d = (torch.tensor(list(x), dtype=torch.int32, device=dev) for x in (src, dst))
        lens = self.seq_lens.index_select(0, s)
        if self.pool is not None:
            self.pool.free(d)
            self.pool.fork(s, d, lens, self.page_caches, self.errors)
        else:
            used = torch.arange(self.pps, device=dev) * self.cfg.block_size < lens[:, None]
            pages = self.block_table.index_select(0, s).masked_fill(~used, -1)
            copy_pages(self.page_caches, pages.reshape(-1), self.block_table.index_select(0, d).reshape(-1))
        self.seq_lens.index_copy_(0, d.long(), lens)
        self.tok.index_copy_(0, d.long(), self.tok.index_select(0, s))

    @torch.no_grad()
    def compact(self) -> None:
        """Moves the pool's pages to the lowest ids, with all that is kept by page:
        caches, k-bar rows and the page state."""
        if self.pool is None:
            raise ValueError("compact needs a page pool (pool_pages)")
        layers = self.page_caches
        state = self.pst.page_tensors(self.num_pages) if self.pst is not None else []
        if state:
            layers = CacheLayers(layers.tensors + state)
        self.pool.compact(layers)
