"""Inputs of the speculative-decoding tests."""
import numpy as np
import torch

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def tree_parents(n, branch):
    """Token j has the children j * branch + 1 ...; branch 0: a random tree."""
    if branch:
        return [-1] + [(i - 1) // branch for i in range(1, n)]
    rng = np.random.default_rng(n)
    return [-1] + [int(rng.integers(0, i)) for i in range(1, n)]


def mask_words(vis, words):
    rows = vis.shape[0]
    b = np.zeros((rows, words * 32), np.uint64)
    b[:, :vis.shape[1]] = vis
    w = (b.reshape(rows, words, 32) << np.arange(32, dtype=np.uint64)).sum(-1)
    return torch.from_numpy(w.astype(np.uint32).view(np.int32))


def attention_tolerance(ref, A, dtype, eps=None):
    """How far an output may be off the exact one.  The output is rounded once
    (eps / 2 of it) and so is each weight p before it meets v (eps / 2 of
    A = sum p |v| / sum p at most).  Logits are 128-term fp32 sums of values
    whose products add up to some 10 at most after scaling: at 2^-24 * 128 of that
    they are off by 8e-5, and so is p by that share; exp2 and the sums add
    less than 1e-5."""
    e = torch.finfo(dtype).eps / 2
    return e * (np.abs(ref) + 1.01 * A) + 1e-4 * A + 1e-6


def make_tree(seed, nodes, ctx, *, H, Hkv, bs, window, K, dtype="bf16", branch=2, index_heads=1, pad_rows=0,
              poison=False, spread=True, shuffle=True, dup=False, scale_q=1.0):
    """A batch of trees (nodes, ctx: lists) on a shuffled page table.  poison:
    NaN and infinities wherever no drafted token may look."""
    from oracle import draft_oracle as DO
    rng = np.random.default_rng(seed)
    B, D = len(nodes), 128
    starts = np.concatenate([[0], np.cumsum(nodes)]).tolist()
    rows = starts[-1]
    W = max(1, max(-(-(c + n) // bs) for c, n in zip(ctx, nodes)) + 1)
    P = B * W + 3
    perm = rng.permutation(P)[:B * W] if shuffle else np.arange(B * W)
    bt = perm.reshape(B, W).astype(np.int32)
    par = []
    for n in nodes:
        par += tree_parents(n, branch) if n else []
    par = np.array(par, np.int32).reshape(-1)
    depth, pos, vis, slots = DO.tree_plan(par, starts, ctx, bt, bs, P)
    lw = window * bs
    idx = np.full((index_heads, rows, K), -1, np.int32)
    for s in range(B):
        for i in range(nodes[s]):
            r = starts[s] + i
            hi = max(0, -(-ctx[s] // bs))
            for ih in range(index_heads):
                k = min(K, hi) if spread else min(K, hi, 2)
                pick = rng.choice(hi, size=k, replace=False) if hi else []     # unsorted, some in the window
                idx[ih, r, :len(pick)] = pick
                if dup and k > 1:
                    idx[ih, r, k - 1] = idx[ih, r, 0]                           # repeated id, another bias
    bias = rng.standard_normal((index_heads, rows, K)).astype(np.float32)
    dt = DT[dtype]
    g = torch.Generator().manual_seed(seed)
    kc = (torch.randn(P, bs, Hkv, D, generator=g) * 0.5).to(dt)
    vc = (torch.randn(P, bs, Hkv, D, generator=g) * 0.5).to(dt)
    q = (torch.randn(rows + pad_rows, H, D, generator=g) * scale_q).to(dt)
    if poison:
        bad = torch.tensor([float("nan"), float("inf"), -float("inf")])
        live = torch.zeros(P, bs, dtype=torch.bool)
        for s in range(B):
            for t in range(ctx[s] + nodes[s]):
                live[bt[s, t // bs], t % bs] = True
        junk = bad[torch.randint(0, 3, (P, bs, Hkv, D), generator=g)].to(dt)
        kc = torch.where(live[:, :, None, None], kc, junk)
        vc = torch.where(live[:, :, None, None], vc, junk)
    words = (max(nodes + [1]) + 31) // 32
    mask = mask_words(vis, words)
    pad = lambda t, v: torch.cat([t, torch.full((pad_rows,) + tuple(t.shape[1:]), v, dtype=t.dtype)])   # noqa: E731
    return dict(B=B, rows=rows, starts=starts, ctx=list(ctx), nodes=list(nodes), P=P, bt=bt, par=par, pos=pos, vis=vis,
                depth=depth, slots=slots, idx=idx, bias=bias, q=q, kc=kc, vc=vc, bs=bs, window=lw, H=H, Hkv=Hkv,
                local_blocks=window, dtype=dt, pad_rows=pad_rows,
                t_idx=torch.cat([torch.from_numpy(idx), torch.full((index_heads, pad_rows, K), -1, dtype=torch.int32)], 1),
                t_bias=torch.cat([torch.from_numpy(bias), torch.zeros(index_heads, pad_rows, K)], 1),
                t_pos=pad(torch.from_numpy(pos.astype(np.int32)), 0), t_mask=pad(mask, 0),
                t_cu=torch.tensor(starts, dtype=torch.int32), t_ctx=torch.tensor(list(ctx), dtype=torch.int32),
                t_bt=torch.from_numpy(bt))
