"""Speculative decoding over the paged DASH cache: what is measured.

Three operators and their plain forms in elementary torch operations:

  tree    DASH attention of a tree of drafted tokens over the paged K/V cache
  verify  acceptance of drafted tokens against the target's distribution, from
          given random numbers, and the next token
  pages   commit (accepted tokens moved to the front), fork (pages shared, the
          partial last page copied) and compact (pages moved to the lowest ids)
          of a block-paged cache of several layers

``listed()`` names the measured cases, ``draw(rng)`` gives further ones of the
same ranges, ``run(state)`` makes one pass.
"""
import math

import torch

own = False

DEV = "cuda"
D = 128                                   # head dim of the decoder
VOCAB = 129280                            # the decoder's vocabulary
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _tree(name, batch, nodes, ctx, heads, kv_heads, block, window, K, dtype="bf16", branch=2, ragged=False):
    return dict(name=name, op="tree", batch=batch, nodes=nodes, ctx=ctx, heads=heads, kv_heads=kv_heads,
                block=block, window=window, K=K, dtype=dtype, branch=branch, ragged=ragged)


def _verify(name, batch, nodes, vocab, mode, dtype="fp32", branch=2):
    return dict(name=name, op="verify", batch=batch, nodes=nodes, vocab=vocab, mode=mode, dtype=dtype,
                branch=branch)


def _pages(name, op, rows, pages, layers, block, heads, tokens):
    return dict(name=name, op=op, rows=rows, pages=pages, layers=layers, block=block, heads=heads,
                tokens=tokens)


def listed():
    return [
        # one short document, a small draft tree: launch latency counts
        _tree("tree 1x8 ctx 1348", 1, 8, 1348, 10, 10, 64, 4, 8),
        # single tokens over the long document (100 pages): the plain decode step
        _tree("tree 32x1 ctx 27556", 32, 1, 27556, 10, 10, 64, 4, 32),
        # the end-to-end decoder's batch and DASH settings, ragged trees
        _tree("tree 8x17 ctx 27556 ragged", 8, 17, 27556, 10, 10, 32, 4, 12, branch=3, ragged=True),
        # the largest: many sequences, trees of 16, long documents of several lengths
        _tree("tree 16x16 ctx 27556 ragged", 16, 16, 27556, 10, 10, 64, 4, 16, branch=2, ragged=True),
        # wide trees with shared kv heads, fp16
        _tree("tree 4x64 ctx 9248 gqa fp16", 4, 64, 9248, 16, 4, 128, 2, 16, dtype="fp16", branch=4),
        # one sequence, one draft path sampled from the draft model
        _verify("verify 1x4 sampled", 1, 4, VOCAB, "sampled", branch=1),
        # a serving batch of trees
        _verify("verify 64x16 sampled", 64, 16, VOCAB, "sampled", branch=3),
        # greedy decoding on the decoder's bf16 logits
        _verify("verify 16x8 greedy", 16, 8, VOCAB, "greedy", dtype="bf16", branch=2),
        # accepted tokens of a batch moved to the front, all layers
        _pages("commit 8 rows 12 layers", "commit", 8, 512, 12, 32, 10, 17),
        # one sequence forked: its last page is copied
        _pages("fork 2 rows 2 layers", "fork", 2, 256, 2, 32, 10, 1348),
        # eight prompts continued eight ways each
        _pages("fork 64 rows 12 layers", "fork", 64, 1024, 12, 32, 10, 1348),
        # a fragmented pool brought to its lowest pages
        _pages("compact 1024 pages 12 layers", "compact", 32, 1024, 12, 32, 10, 600),
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "verify", "commit", "fork", "compact"])
    if op == "tree":
        kv = rng.choice([1, 2, 4, 10])
        heads = kv * rng.choice([1, 1, 2, 4, 5])
        block = rng.choice([16, 32, 64, 128])
        nodes = _logint(rng, 1, 64)
        ctx = _logint(rng, 1, 27556)
        batch = _logint(rng, 1, 32)
        # no dearer than the largest listed case: key rows of the plain form
        while batch * ctx * max(kv, 1) * max(1, nodes // 16) > 16 * 27556 * 10 and batch > 1:
            batch -= 1
        return dict(op=op, batch=batch, nodes=nodes, ctx=ctx, heads=heads, kv_heads=kv, block=block,
                    window=rng.choice([1, 2, 4, 8]), K=rng.choice([0, 3, 8, 12, 16, 32]),
                    dtype=rng.choice(["bf16", "fp16"]), branch=rng.choice([1, 2, 3, 4]),
                    ragged=rng.random() < 0.5)
    if op == "verify":
        mode = rng.choice(["sampled", "certain", "greedy"])
        return dict(op=op, batch=_logint(rng, 1, 64), nodes=_logint(rng, 1, 16), vocab=_logint(rng, 97, VOCAB),
                    mode=mode, dtype=rng.choice(["fp32", "bf16", "fp16"]) if mode == "greedy" else "fp32",
                    branch=rng.choice([1, 2, 3, 4]))
    layers, block = rng.randint(1, 12), rng.choice([16, 32, 64])
    pages = _logint(rng, 64, 1024) * 32 // block + 8
    if op == "commit":
        return dict(op=op, rows=_logint(rng, 1, 32), pages=pages + 128, layers=layers, block=block,
                    heads=rng.choice([1, 2, 10]), tokens=_logint(rng, 1, 64))
    rows = 2 * _logint(rng, 1, 16)
    return dict(op=op, rows=rows, pages=pages, layers=layers, block=block, heads=rng.choice([1, 2, 10]),
                tokens=max(1, min(_logint(rng, 17, 4000), (pages // rows - 2) * block)))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _parents(n, branch):
    """A tree of n tokens in which token j has the children j * branch + 1 ..."""
    return [-1] + [(i - 1) // branch for i in range(1, n)]


def _prepare_tree(c, seed):
    g = _gen(seed)
    B, bs, H, Hkv, dt = c["batch"], c["block"], c["heads"], c["kv_heads"], _DT[c["dtype"]]
    host = torch.Generator().manual_seed(int(seed))
    if c["ragged"]:
        # the trees' sizes belong to the case (they make the outputs' shape)
        n = torch.randint(1, c["nodes"] + 1, (B,), generator=torch.Generator().manual_seed(B))
        ctx = torch.randint((c["ctx"] + 1) // 2, c["ctx"] + 1, (B,), generator=host)
        n[0], ctx[0] = c["nodes"], c["ctx"]
    else:
        n = torch.full((B,), c["nodes"])
        ctx = torch.full((B,), c["ctx"])
    n, ctx = n.tolist(), ctx.tolist()
    W = -(-(c["ctx"] + c["nodes"]) // bs)
    P = B * W
    rows = sum(n)
    start = [0]
    for x in n:
        start.append(start[-1] + x)
    par, depth = [], []
    for x in n:
        p = _parents(x, c["branch"])
        d = []
        for u in p:
            d.append(0 if u < 0 else d[u] + 1)
        par += p
        depth += d
    words = (c["nodes"] + 31) // 32
    mask = torch.zeros(rows, words * 32, dtype=torch.bool)
    for s in range(B):
        for i in range(n[s]):
            r = start[s] + i
            if par[r] >= 0:
                mask[r] = mask[start[s] + par[r]]
            mask[r, i] = True
    bits = (mask.view(rows, words, 32).long() << torch.arange(32)).sum(-1)
    bits = torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).to(torch.int32)
    pos = torch.tensor([ctx[s] + depth[r] for s in range(B) for r in range(start[s], start[s + 1])],
                       dtype=torch.int32)
    # routed lists: the tokens of one tree pick K blocks out of 2K that suit
    # their sequence (ascending, -1 tail), as neighbouring tokens do
    K = c["K"]
    idx = torch.full((rows, K), -1, dtype=torch.int32)
    for s in range(B):
        for i in range(n[s]):
            r = start[s] + i
            cand = int(pos[r]) // bs - c["window"] + 1
            cand = min(cand, -(-ctx[s] // bs))
            if i == 0:
                pool = torch.randperm(max(cand, 0), generator=host)[:2 * K]
            if cand > 0 and K:
                mine = pool[torch.randperm(len(pool), generator=host)[:K]].sort().values
                idx[r, :len(mine)] = mine.to(torch.int32)
    bias = torch.rand(rows, K, generator=g, device=DEV) * 2 - 1.5
    kc = torch.randn(P, bs, Hkv, D, generator=g, device=DEV, dtype=dt).mul_(0.5)
    vc = torch.randn(P, bs, Hkv, D, generator=g, device=DEV, dtype=dt).mul_(0.5)
    q = torch.randn(rows, H, D, generator=g, device=DEV, dtype=dt)
    bt = torch.randperm(P, generator=g, device=DEV).to(torch.int32).view(B, W)
    seq = torch.repeat_interleave(torch.arange(B), torch.tensor(n))
    return dict(case=c, q=q, kc=kc, vc=vc, idx=idx.to(DEV), bias=bias, bt=bt,
                cu=torch.tensor(start, dtype=torch.int32, device=DEV),
                ctx=torch.tensor(ctx, dtype=torch.int32, device=DEV), pos=pos.to(DEV), mask=bits.to(DEV),
                seq=seq.to(DEV), node=torch.cat([torch.arange(x) for x in n]).to(DEV),
                out=torch.empty(rows, H, D, device=DEV, dtype=dt),
                lse=torch.empty(rows, H, device=DEV), scale=1.0 / math.sqrt(D))


def _prepare_verify(c, seed):
    g = _gen(seed)
    B, n, V, mode = c["batch"], c["nodes"], c["vocab"], c["mode"]
    rows = B * n
    par = torch.tensor(_parents(n, c["branch"]) * B, dtype=torch.int32, device=DEV)
    cu = torch.arange(B + 1, dtype=torch.int32, device=DEV) * n
    logits = torch.randn(rows, V, generator=g, device=DEV) * 3
    first = torch.arange(rows, device=DEV) // n * n
    parent_row = (first + par.clamp_min(0)).long()
    draft = None
    if mode == "sampled":
        target = logits.softmax(-1)
        draft = (logits + torch.randn(rows, V, generator=g, device=DEV) * 0.5).softmax(-1)
        # inverse CDF of each parent's draft distribution
        u = torch.rand(rows, 1, generator=g, device=DEV)
        tok = torch.searchsorted(draft.cumsum(-1)[parent_row], u).squeeze(1).clamp_max(V - 1)
    else:
        target = logits.softmax(-1) if mode == "certain" else logits.to(_DT[c["dtype"]])
        # each draft is its parent's likeliest token, or the second, third ... one
        k = torch.randint(0, 3, (rows,), generator=g, device=DEV)
        k = torch.where(torch.rand(rows, generator=g, device=DEV) < 0.6, torch.zeros_like(k), k).clamp_max(V - 1)
        tok = target.float().topk(3, dim=-1).indices[parent_row, k]
    return dict(case=c, tokens=tok.long(), parents=par, cu=cu, target=target, draft=draft,
                u_accept=torch.rand(rows, generator=g, device=DEV),
                u_sample=torch.rand(B, generator=g, device=DEV))


def _caches(c, g):
    """K, V (bf16), index keys and k-bar rows (fp32) of all layers."""
    shape = (c["layers"], c["pages"], c["block"])
    return [torch.randn(*shape, c["heads"], D, generator=g, device=DEV, dtype=torch.bfloat16),
            torch.randn(*shape, c["heads"], D, generator=g, device=DEV, dtype=torch.bfloat16),
            torch.randn(*shape, D, generator=g, device=DEV),
            torch.randn(*shape[:2], 1, D, generator=g, device=DEV)]


def _keep(state):
    """What a program keeps next to its caches: their layers as a list and,
    with the framework, the handles made of the tensors once."""
    state["layers"] = [t[i] for t in state["caches"] for i in range(t.shape[0])]
    if own:
        from ananta_ocr_b200.page_pool import CacheLayers, PagePool
        state["layers"] = CacheLayers(state["layers"])
        for name in ("meta", "into"):
            if name in state:
                state[name + "_pool"] = PagePool.from_tensors(block_size=state["case"]["block"], **state[name])
    return state


def _prepare_pages(c, seed):
    g = _gen(seed)
    host = torch.Generator().manual_seed(int(seed))
    caches = _caches(c, g)
    P, bs, R = c["pages"], c["block"], c["rows"]
    if c["op"] == "commit":
        # rows of accepted nodes: ascending node numbers out of `tokens` drafts
        n = c["tokens"]
        ctx = torch.randint(0, 4 * bs, (R,), generator=host)
        W = -(-(4 * bs + n) // bs)
        path = torch.full((R, n), -1, dtype=torch.int32)
        acc = torch.zeros(R, dtype=torch.int32)
        for r in range(R):
            k = int(torch.randint(0, n, (1,), generator=host)) if n > 1 else 0
            path[r, 0] = 0
            path[r, 1:k + 1] = (torch.randperm(n - 1, generator=host)[:k].sort().values + 1).to(torch.int32)
            acc[r] = k
        # distinct pages for every row
        bt = torch.randperm(P, generator=host)[:R * W].view(R, W).to(torch.int32)
        return _keep(dict(case=c, caches=caches[:3], ctx=ctx.to(torch.int32).to(DEV), bt=bt.to(DEV),
                          path=path.to(DEV), acc=acc.to(DEV)))
    W = P // 2
    ref = torch.zeros(P, dtype=torch.int32)
    table = torch.full((R, W), -1, dtype=torch.int32)
    blocks = torch.zeros(R, dtype=torch.int32)
    perm = torch.randperm(P, generator=host).to(torch.int32)
    used = 0
    lens = torch.zeros(R, dtype=torch.int32)
    if c["op"] == "fork":
        # the first rows hold prompts; the others are continuations of them,
        # dropped and forked again by every pass
        S = max(1, R // 8)
        for r in range(S):
            most = max(1, min(c["tokens"], (P - used - 2 * R) * bs // (S - r)))
            lens[r] = int(torch.randint((most + 1) // 2, most + 1, (1,), generator=host))
            nb = -(-int(lens[r]) // bs)
            table[r, :nb] = perm[used:used + nb]
            ref[perm[used:used + nb].long()] = 1
            blocks[r] = nb
            used += nb
        src = torch.arange(R - S, dtype=torch.int32) % S
        dst = torch.arange(S, R, dtype=torch.int32)
        flens = torch.stack([lens[int(s)] for s in src]).to(torch.int32)
        for s, d, n in zip(src.tolist(), dst.tolist(), flens.tolist()):
            full = n // bs
            table[d, :full] = table[s, :full]
            ref[table[s, :full].long()] += 1
            blocks[d] = full
            if n % bs and used < P:
                table[d, full] = perm[used]
                ref[perm[used].long()] = 1
                blocks[d] = full + 1
                used += 1
    else:
        # rows of several lengths on pages scattered over the whole pool, the
        # first blocks of odd rows shared with the row before
        src = dst = flens = None
        for r in range(R):
            nb = max(1, min(-(-c["tokens"] // bs) - int(torch.randint(0, 4, (1,), generator=host)),
                            (P * 6 // 10 - used) // (R - r) if P * 6 // 10 > used else 1))
            shared = min(2, nb, int(blocks[r - 1])) if r % 2 else 0
            nb = min(nb, shared + P - used)
            if shared:
                table[r, :shared] = table[r - 1, :shared]
                ref[table[r, :shared].long()] += 1
            fresh = perm[used:used + nb - shared]
            table[r, shared:nb] = fresh
            ref[fresh.long()] = 1
            used += nb - shared
            blocks[r] = nb
    stack = torch.full((P,), -1, dtype=torch.int32)
    stack[:P - used] = perm[used:]
    meta = dict(ref=ref, free_list=stack, n_free=torch.tensor([P - used], dtype=torch.int32),
                block_table=table, n_blocks=blocks)
    meta = {k: v.to(DEV) for k, v in meta.items()}
    state = dict(case=c, caches=caches, meta=meta)
    if c["op"] == "fork":
        state.update(src=src.to(DEV), dst=dst.to(DEV), lens=flens.to(DEV),
                     keep=torch.zeros(R - S, dtype=torch.int32, device=DEV))
    else:
        state["into"] = {k: torch.empty_like(v) for k, v in meta.items()}
    return _keep(state)


def prepare(case, seed):
    if case["op"] == "tree":
        return _prepare_tree(case, seed)
    if case["op"] == "verify":
        return _prepare_verify(case, seed)
    return _prepare_pages(case, seed)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _tree_plain(s):
    c = s["case"]
    B, bs, Hkv, n, K = c["batch"], c["block"], c["kv_heads"], c["nodes"], c["K"]
    G = c["heads"] // Hkv
    W = s["bt"].shape[1]
    S = W * bs
    k = s["kc"][s["bt"].long()].view(B, S, Hkv, D).float()
    v = s["vc"][s["bt"].long()].view(B, S, Hkv, D).float()
    # rows padded to n per sequence
    seq, node = s["seq"], s["node"]
    q = torch.zeros(B, n, Hkv, G, D, device=DEV)
    q[seq, node] = s["q"].view(-1, Hkv, G, D).float()
    term = torch.full((B, n, W + 1), -math.inf, device=DEV)
    if K:
        # a slot without a block (-1) goes to a column behind the last block
        at = s["idx"].long()
        at = torch.where(at < 0, W, at)
        flat = torch.full((seq.numel(), W + 1), -math.inf, device=DEV).scatter(1, at, s["bias"])
        flat[:, W] = -math.inf
        term[seq, node] = flat
    j = torch.arange(S, device=DEV)
    pos = torch.zeros(B, n, dtype=torch.int64, device=DEV)
    pos[seq, node] = s["pos"].long()
    ctx = s["ctx"].long()[:, None, None]
    window = (pos - c["window"] * bs)[:, :, None]
    add = torch.where(j > window, 0.0, term[:, :, :W].repeat_interleave(bs, dim=2))
    seen = torch.zeros(B, n, s["mask"].shape[1] * 32, dtype=torch.bool, device=DEV)
    seen[seq, node] = (s["mask"][:, :, None].long() >> torch.arange(32, device=DEV) & 1).bool().flatten(1)
    u = (j - ctx).clamp(0, seen.shape[2] - 1)
    drafted = torch.gather(seen, 2, u.expand(B, n, S)) & (j - ctx < seen.shape[2])
    add = torch.where(j < ctx, add, torch.where(drafted, 0.0, -math.inf))
    x = torch.einsum("bnhgd,bshd->bnhgs", q, k) * s["scale"] + add[:, :, None, None, :]
    del k
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(x - m)
    del x
    total = p.sum(-1, keepdim=True)
    o = torch.einsum("bnhgs,bshd->bnhgd", p, v) / torch.where(total > 0, total, 1.0)
    lse = (m + torch.log(total)).squeeze(-1)
    rows = seq.numel()
    return o[seq, node].reshape(rows, -1, D).to(s["out"].dtype), lse[seq, node].reshape(rows, -1)


def _tree_own(s):
    from ananta_ocr_b200 import drafts
    c = s["case"]
    Hkv = c["kv_heads"]
    drafts.dash_sparse_attn_tree(
        s["q"], s["kc"], s["vc"], s["idx"][None].expand(Hkv, -1, -1), s["bias"][None].expand(Hkv, -1, -1),
        s["bt"], s["cu"], s["ctx"], s["pos"], s["mask"], c["nodes"], Hkv, s["scale"], s["out"],
        local_blocks=c["window"], sparse_block_size=c["block"], lse=s["lse"])
    return s["out"], s["lse"]


def _verify_plain(s):
    c = s["case"]
    B, n, V, mode = c["batch"], c["nodes"], c["vocab"], c["mode"]
    row0 = s["cu"][:-1].long()
    every = torch.arange(B, device=DEV)
    tok, par = s["tokens"].view(B, n), s["parents"].view(B, n)
    cur = torch.zeros(B, dtype=torch.int64, device=DEV)
    acc = torch.zeros(B, dtype=torch.int64, device=DEV)
    path = torch.full((B, n + 1), -1, dtype=torch.int64, device=DEV)
    path[:, 0] = 0
    greedy = mode == "greedy"
    best = s["target"].float().argmax(-1) if greedy else None
    p = None if greedy else s["target"][row0].double()
    q = s["draft"][row0].double() if mode == "sampled" else None
    less = torch.zeros(B, dtype=torch.float64, device=DEV)
    mass = torch.ones(B, dtype=torch.float64, device=DEV)
    for i in range(1, n):                                 # a token's fate hangs on those before it
        mine = par[:, i] == cur
        x = tok[:, i]
        if greedy:
            take = mine & (best[row0 + cur] == x)
        else:
            px = p[every, x]
            u = s["u_accept"][row0 + i].double()
            if q is not None:
                qx = q[every, x]
                take = mine & (u * mass * qx < px - less * qx)
            else:
                take = mine & (u * mass < px)
        drop = mine & ~take
        acc = acc + take
        path.scatter_(1, torch.where(take, acc, n)[:, None], i)
        cur = torch.where(take, i, cur)
        if greedy:
            continue
        new = s["target"][row0 + cur].double()
        if q is not None:
            less = torch.where(take, 0.0, torch.where(drop, less + mass, less))
            p = torch.where(take[:, None], new, p)
            q = torch.where(take[:, None], s["draft"][row0 + cur].double(), q)
            left = (p - less[:, None] * q).clamp_min(0).sum(-1)
            mass = torch.where(take, 1.0, torch.where(drop, left, mass))
        else:
            mass = torch.where(take, 1.0, torch.where(drop, mass - px, mass))
            p = torch.where(take[:, None], new, p.scatter(1, x[:, None], torch.where(drop, 0.0, px)[:, None]))
    if greedy:
        nxt = best[row0 + cur]
    else:
        r = (p - less[:, None] * q).clamp_min(0) if q is not None else p
        r = torch.where(r.sum(-1, keepdim=True) > 0, r, s["target"][row0 + cur].double())
        run_sum = r.cumsum(-1)
        at = s["u_sample"].double()[:, None] * run_sum[:, -1:]
        nxt = ((run_sum > at) & (r > 0)).to(torch.uint8).argmax(-1)
    path = path[:, :n]
    step = torch.arange(n, device=DEV)
    after = torch.gather(tok, 1, path.roll(-1, 1).clamp_min(0))
    toks = torch.where(step < acc[:, None], after, torch.where(step == acc[:, None], nxt[:, None], -1))
    return acc.to(torch.int32), path.to(torch.int32), nxt, toks


def _verify_own(s):
    from ananta_ocr_b200 import drafts
    c = s["case"]
    greedy = c["mode"] == "greedy"
    r = drafts.verify_drafts(s["tokens"], s["parents"], s["cu"], s["target"], max_nodes=c["nodes"],
                             draft=s["draft"], u_accept=None if greedy else s["u_accept"],
                             u_sample=None if greedy else s["u_sample"], greedy=greedy)
    return r.n_accept, r.path, r.next_token, r.tokens


def _commit_plain(s):
    bs = s["case"]["block"]
    R, n = s["path"].shape
    i = torch.arange(n, device=DEV)
    on = (i > 0) & (i <= s["acc"][:, None])
    row = torch.arange(R, device=DEV)[:, None].expand(R, n)[on]
    src = (s["ctx"].long()[:, None] + s["path"].long())[on]
    dst = (s["ctx"].long()[:, None] + i)[on]
    bt = s["bt"].long()
    sp, dp = bt[row, src // bs], bt[row, dst // bs]
    for t in s["caches"]:
        t[:, dp, dst % bs] = t[:, sp, src % bs]
    return _data(s)


def _commit_own(s):
    from ananta_ocr_b200 import drafts
    drafts.commit_drafts(s["layers"], s["path"], s["acc"], s["ctx"], s["bt"])
    return _data(s)


def _data(s):
    """The caches' contents as whole numbers: a move changes no bit of them."""
    return [t.view(torch.int16) if t.dtype == torch.bfloat16 else t.view(torch.int32) for t in s["caches"]]


def _free_plain(m, rows, keep):
    P = m["ref"].numel()
    rows = rows.long()
    b = torch.arange(m["block_table"].shape[1], device=DEV)
    had = m["n_blocks"][rows]
    gone = (b >= keep[:, None]) & (b < had[:, None])
    table = m["block_table"][rows]
    was = m["ref"].clone()
    m["ref"].index_add_(0, table[gone].long(), torch.full_like(table[gone], -1))
    freed = torch.nonzero((was > 0) & (m["ref"] == 0)).flatten().to(torch.int32)
    at = m["n_free"].long() + torch.arange(freed.numel(), device=DEV)
    m["free_list"][at] = freed
    m["n_free"] += freed.numel()
    m["block_table"][rows] = torch.where(gone, -1, table)
    m["n_blocks"][rows] = torch.minimum(had, keep)


def _fork_plain(s):
    m, bs = s["meta"], s["case"]["block"]
    _free_plain(m, s["dst"], s["keep"])
    src, dst, lens = s["src"].long(), s["dst"].long(), s["lens"]
    W = m["block_table"].shape[1]
    b = torch.arange(W, device=DEV)
    full, part = lens // bs, (lens % bs > 0)
    order = torch.cumsum(part, 0) - 1
    part = part & (order < m["n_free"])
    ok = part | (lens % bs == 0)
    at = (m["n_free"] - 1 - order).clamp_min(0)
    page = torch.where(part, m["free_list"][at.long()], -1)
    table = m["block_table"][src]
    old = torch.gather(table, 1, full.long().clamp_max(W - 1)[:, None]).squeeze(1)
    shared = (b < full[:, None]) & ok[:, None]
    m["ref"].index_add_(0, table[shared].long(), torch.ones_like(table[shared]))
    m["ref"][page[part].long()] = 1
    m["free_list"][at[part].long()] = -1
    m["n_free"] -= part.sum().to(torch.int32)
    m["block_table"][dst] = torch.where(shared, table, torch.where((b == full[:, None]) & part[:, None],
                                                                   page[:, None], -1))
    m["n_blocks"][dst] = torch.where(ok, full + part, 0).to(torch.int32)
    for t in s["caches"]:
        t[:, page[part].long()] = t[:, old[part].long()]
    return [m[k] for k in sorted(m)] + _data(s)


def _fork_own(s):
    m, pool = s["meta"], s["meta_pool"]
    pool.free(s["dst"], s["keep"])
    pool.fork(s["src"], s["dst"], s["lens"], s["layers"])
    return [m[k] for k in sorted(m)] + _data(s)


def _compact_plain(s):
    m, to = s["meta"], s["into"]
    P = m["ref"].numel()
    live = m["ref"] > 0
    L = live.sum()
    ids = torch.arange(P, device=DEV)
    movers = torch.nonzero(live & (ids >= L)).flatten()
    holes = torch.nonzero(~live & (ids < L)).flatten()
    new = ids.clone()
    new[movers] = holes
    to["ref"].copy_(m["ref"])
    to["ref"][holes] = m["ref"][movers]
    to["ref"][movers] = 0
    # the lowest free page is on top of the stack
    to["free_list"].copy_(torch.where(ids < P - L, P - 1 - ids, -1))
    to["n_free"].copy_((P - L)[None])
    table = m["block_table"].long()
    to["block_table"].copy_(torch.where(table >= 0, new[table.clamp_min(0)], -1))
    to["n_blocks"].copy_(m["n_blocks"])
    for t in s["caches"]:
        t[:, holes] = t[:, movers]
    return [to[k] for k in sorted(to)] + _data(s)


def _compact_own(s):
    to = s["into"]
    s["meta_pool"].compact(s["layers"], into=s["into_pool"])
    return [to[k] for k in sorted(to)] + _data(s)


_RUN = {"tree": (_tree_plain, _tree_own), "verify": (_verify_plain, _verify_own),
        "commit": (_commit_plain, _commit_own), "fork": (_fork_plain, _fork_own),
        "compact": (_compact_plain, _compact_own)}


def run(state):
    plain, kernels = _RUN[state["case"]["op"]]
    return kernels(state) if own else plain(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def _page_bytes(c, tokens):
    """Bytes of `tokens` tokens in all layers: K, V (bf16) and the index keys."""
    return c["layers"] * tokens * (2 * c["heads"] * D * 2 + D * 4)


def work(case):
    c = case
    if c["op"] == "tree":
        share = 0.75 if c["ragged"] else 1.0
        n = 1 + (c["nodes"] - 1) * (0.5 if c["ragged"] else 1.0)
        rows, ctx = c["batch"] * n, c["ctx"] * share
        win = min(ctx, c["window"] * c["block"])
        far = max(0.0, ctx - win)
        pool = min(2 * c["K"], far / c["block"])
        mine = min(c["K"], pool)
        # blocks that some token of the tree picked, of the sequence's pool
        union = pool * (1 - (1 - mine / pool) ** n) if pool else 0.0
        keys = c["batch"] * (union * c["block"] + win + n)
        per_row = mine * c["block"] + win + 1 + math.log2(n + 1)
        return dict(bytes=keys * c["kv_heads"] * D * 2 * 2 + rows * c["heads"] * (D * 2 * 2 + 4)
                    + rows * c["K"] * 8, flops=4.0 * D * c["heads"] * rows * per_row)
    if c["op"] == "verify":
        size = 2 if c["dtype"] in ("bf16", "fp16") else 4
        depth = math.log(max(2, c["nodes"]), max(2, c["branch"])) if c["branch"] > 1 else c["nodes"] - 1
        # greedy decoding reads a row for each accepted token and one more; with
        # random numbers the last row of the target and of the draft are read
        reads = 1 + sum(0.7 ** k for k in range(1, int(depth) + 1)) if c["mode"] == "greedy" else 1
        reads *= 2 if c["mode"] == "sampled" else 1
        return dict(bytes=c["batch"] * (reads * c["vocab"] * size + c["nodes"] * 24),
                    flops=c["batch"] * reads * c["vocab"] * 2.0)
    if c["op"] == "commit":
        tokens = c["rows"] * (c["tokens"] - 1) / 2
        return dict(bytes=2 * _page_bytes(c, tokens) + c["rows"] * c["tokens"] * 4 + 64, flops=0)
    bar = c["layers"] * D * 4
    if c["op"] == "fork":
        n = c["rows"] - max(1, c["rows"] // 8)
        return dict(bytes=2 * n * (_page_bytes(c, c["block"]) + bar) + n * 0.75 * c["tokens"] / c["block"] * 16,
                    flops=0)
    blocks = max(1, -(-c["tokens"] // c["block"]) - 1.5)
    live = min(0.6 * c["pages"], c["rows"] * (blocks - 1))
    moves = live * (1 - live / c["pages"])
    return dict(bytes=2 * moves * (_page_bytes(c, c["block"]) + bar) + c["pages"] * 16
                + c["rows"] * c["pages"] * 4, flops=0)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _tree_exact(s):
    c = s["case"]
    bs, H, Hkv = c["block"], c["heads"], c["kv_heads"]
    G = H // Hkv
    cu, ctx, pos = s["cu"].tolist(), s["ctx"].tolist(), s["pos"].tolist()
    routed, bias, mask = s["idx"].tolist(), s["bias"].double().cpu(), s["mask"].tolist()
    outs, lses = [], []
    for b in range(c["batch"]):
        n = cu[b + 1] - cu[b]
        total = ctx[b] + n
        pages = s["bt"][b, :-(-total // bs)].long()
        k = s["kc"][pages].reshape(-1, Hkv, D)[:total].double()
        v = s["vc"][pages].reshape(-1, Hkv, D)[:total].double()
        term = torch.full((n, total), -math.inf, dtype=torch.float64)
        for i in range(n):
            r = cu[b] + i
            edge = min(max(pos[r] - c["window"] * bs + 1, 0), ctx[b])      # first key of the window
            for a, blk in enumerate(routed[r]):
                if blk >= 0:
                    term[i, blk * bs:min(blk * bs + bs, edge)] = bias[r, a]
            term[i, edge:ctx[b]] = 0.0
            for u in range(n):
                if mask[r][u // 32] >> (u % 32) & 1:
                    term[i, ctx[b] + u] = 0.0
        term = term.to(DEV)
        q = s["q"][cu[b]:cu[b + 1]].double().view(n, Hkv, G, D)
        for h in range(Hkv):
            x = q[:, h].reshape(n * G, D) @ k[:, h].T * s["scale"] + term.repeat_interleave(G, 0)
            lse = torch.logsumexp(x, -1)
            p = torch.where(lse[:, None] > -math.inf, (x - lse[:, None]).exp(), 0.0)
            lses.append(lse.view(n, G))
            outs.append((p @ v[:, h]).view(n, G, D))
    o = torch.cat([torch.stack(outs[b * Hkv:(b + 1) * Hkv], 1).flatten(1, 2) for b in range(c["batch"])])
    z = torch.cat([torch.stack(lses[b * Hkv:(b + 1) * Hkv], 1).flatten(1, 2) for b in range(c["batch"])])
    return o, z


def _verify_exact(s):
    import numpy as np
    c = s["case"]
    B, n, mode = c["batch"], c["nodes"], c["mode"]
    tok = s["tokens"].view(B, n).tolist()
    par = s["parents"].view(B, n).tolist()
    ua = s["u_accept"].double().view(B, n).tolist()
    us = s["u_sample"].double().tolist()
    row = lambda t, r: t[r].double().cpu().numpy()                # noqa: E731
    accs, paths, nexts, toks = [], [], [], []
    for b in range(B):
        way, out, cur = [0], [], 0
        while True:
            kids = [i for i in range(cur + 1, n) if par[b][i] == cur]
            p = row(s["target"], b * n + cur)
            if mode == "greedy":
                nxt = int(np.argmax(p))
                hit = next((i for i in kids if tok[b][i] == nxt), None)
            else:
                res, hit, whole = p.copy(), None, 1.0
                q = row(s["draft"], b * n + cur) if mode == "sampled" else None
                for i in kids:
                    x = tok[b][i]
                    # the residual, normalised at each rejection
                    if ua[b][i] * (q[x] if q is not None else 1.0) < res[x] / whole:
                        hit = i
                        break
                    if q is not None:
                        res = np.maximum(res / whole - q, 0.0)
                        whole = res.sum()
                        if whole <= 0:
                            break
                    else:
                        whole -= res[x]
                        res[x] = 0.0
                if hit is None:
                    if res.sum() <= 0:
                        res = p
                    cum = np.cumsum(res)
                    nxt = int(np.argmax((cum > us[b] * cum[-1]) & (res > 0)))
            if hit is None:
                break
            way.append(hit)
            out.append(tok[b][hit])
            cur = hit
        accs.append(len(out))
        nexts.append(nxt)
        paths.append(way + [-1] * (n - len(way)))
        toks.append(out + [nxt] + [-1] * (n - 1 - len(out)))
    return (torch.tensor(accs, dtype=torch.int32), torch.tensor(paths, dtype=torch.int32), torch.tensor(nexts),
            torch.tensor(toks))


def exact(case, seed):
    if case["op"] == "tree":
        return _tree_exact(_prepare_tree(case, seed))
    if case["op"] == "verify":
        return _verify_exact(_prepare_verify(case, seed))
    return None              # pages are moved, not computed
