"""Oracle of speculative decoding on the paged cache, in numpy and 64 bits:
draft-tree plan and attention, verification, and the page pool.  Written from
the definitions in include/dash_b200.h; test infrastructure only."""
from __future__ import annotations

import numpy as np


# ---------------------------------------------------------------------------
# draft trees
# ---------------------------------------------------------------------------
def tree_plan(parents, starts, ctx, bt, bs, num_pages):
    """depth, pos, visible [rows, most] bool, slots of packed drafted tokens."""
    rows = starts[-1]
    most = max([b - a for a, b in zip(starts, starts[1:])] + [1])
    depth, pos = np.zeros(rows, np.int64), np.zeros(rows, np.int64)
    vis, slots = np.zeros((rows, most), bool), np.full(rows, -1, np.int64)
    for s in range(len(starts) - 1):
        for i in range(starts[s + 1] - starts[s]):
            r = starts[s] + i
            p = -1 if i == 0 else (i - 1 if parents is None else int(parents[r]))
            if 0 <= p < i:
                depth[r] = depth[starts[s] + p] + 1
                vis[r] = vis[starts[s] + p]
            vis[r, i] = True
            pos[r] = ctx[s] + depth[r]
            t = int(ctx[s]) + i
            page = int(bt[s, t // bs]) if t // bs < bt.shape[1] else -1
            if 0 <= page < num_pages:
                slots[r] = page * bs + t % bs
    return depth, pos, vis, slots


def tree_attend(q, kc, vc, idx, bias, bt, starts, ctx, pos, vis, bs, window, scale):
    """q [rows, H, D], caches [P, bs, Hkv, D], idx [HI, rows, K] -> (out, lse,
    A) with A = sum p |v| / sum p, the scale of an error of the weights."""
    rows, H, D = q.shape
    Hkv, HI = kc.shape[2], idx.shape[0]
    out, lse = np.zeros((rows, H, D)), np.full((rows, H), -np.inf)
    A = np.zeros((rows, H, D))
    for s in range(len(starts) - 1):
        n, c = starts[s + 1] - starts[s], int(ctx[s])
        for i in range(n):
            r = starts[s] + i
            edge = min(max(int(pos[r]) - window + 1, 0), c)
            tail = [(t, 0.0) for t in range(edge, c)] + [(c + u, 0.0) for u in range(n) if vis[r, u]]
            for ih in range(HI):
                keys, seen = [], set()
                for a, b in enumerate(idx[ih, r]):
                    b = int(b)
                    if b < 0 or b * bs >= c + n or b in seen:
                        continue
                    seen.add(b)
                    w = 0.0 if bias is None else float(bias[ih, r, a])
                    keys += [(t, w) for t in range(b * bs, min(b * bs + bs, edge))]
                keys += tail
                keys = [(t, w) for t, w in keys if 0 <= bt[s, t // bs] < kc.shape[0]]
                if not keys:
                    continue
                t = np.array([x[0] for x in keys])
                w = np.array([x[1] for x in keys])
                page = bt[s, t // bs]
                for h in range(ih * H // HI, (ih + 1) * H // HI):
                    g = h * Hkv // H
                    k = kc[page, t % bs, g].astype(np.float64)
                    v = vc[page, t % bs, g].astype(np.float64)
                    x = k @ q[r, h].astype(np.float64) * scale + w
                    m = x.max()
                    if m == -np.inf:
                        continue
                    p = np.exp(x - m)
                    z = p.sum()
                    out[r, h] = p @ v / z
                    A[r, h] = p @ np.abs(v) / z
                    lse[r, h] = m + np.log(z)
    return out, lse, A


# ---------------------------------------------------------------------------
# verification
# ---------------------------------------------------------------------------
def _pick(res, u):
    cum = np.cumsum(res)
    hit = np.nonzero((cum > u * cum[-1]) & (res > 0))[0]
    return int(hit[0]) if len(hit) else -1


def verify(tokens, parents, starts, target, draft, u_accept, u_sample, mode, max_nodes):
    """mode 'drawn' | 'certain' | 'greedy' -> n_accept, path, next, tokens."""
    n_seq, V = len(starts) - 1, target.shape[1]
    acc, nxt = np.zeros(n_seq, np.int64), np.full(n_seq, -1, np.int64)
    path, toks = np.full((n_seq, max_nodes), -1, np.int64), np.full((n_seq, max_nodes), -1, np.int64)
    for s in range(n_seq):
        r0, n = starts[s], starts[s + 1] - starts[s]
        if n == 0:
            continue
        cur, way = 0, [0]
        while True:
            par = [(-1 if i == 0 else i - 1) if parents is None else int(parents[r0 + i]) for i in range(n)]
            kids = [i for i in range(cur + 1, n) if par[i] == cur and 0 <= tokens[r0 + i] < V]
            p = target[r0 + cur].astype(np.float64)
            hit = None
            if mode == "greedy":
                best = int(np.argmax(p))          # numpy: NaN is the largest, first of equals
                hit = next((i for i in kids if tokens[r0 + i] == best), None)
            else:
                res, mass = p.copy(), 1.0
                for i in kids:
                    x = int(tokens[r0 + i])
                    q = draft[r0 + cur].astype(np.float64) if mode == "drawn" else None
                    if float(u_accept[r0 + i]) * mass * (q[x] if q is not None else 1.0) < res[x]:
                        hit = i
                        break
                    if q is not None:
                        # the normalised residual less the draft's distribution
                        if mass > 0:
                            res = np.maximum(res / mass - q, 0.0)
                            mass = res.sum()
                    else:
                        mass -= res[x]
                        res[x] = 0.0
                if hit is None:
                    res = np.maximum(res, 0.0)
                    if not res.sum() > 0:
                        res = np.maximum(p, 0.0)
                    best = _pick(res, float(u_sample[s])) if res.sum() > 0 else -1
            if hit is None:
                break
            way.append(hit)
            cur = hit
        k = len(way) - 1
        acc[s], nxt[s] = k, best
        path[s, :k + 1] = way
        toks[s, :k] = [tokens[r0 + i] for i in way[1:]]
        toks[s, k] = best
    return acc, path, nxt, toks


# ---------------------------------------------------------------------------
# pages
# ---------------------------------------------------------------------------
class Pool:
    """The page pool as plain Python lists."""

    def __init__(self, pages, rows, width, bs):
        self.ref, self.free = [0] * pages, list(range(pages - 1, -1, -1))
        self.table, self.width, self.bs = [[] for _ in range(rows)], width, bs
        self.errors = 0

    def _first(self, rows):
        seen, ok = set(), []
        for r in rows:
            ok.append(0 <= r < len(self.table) and r not in seen)
            seen.add(r)
        return ok

    def reserve(self, rows, lens):
        full = False
        asked, avail = 0, len(self.free)
        for r, n, ok in zip(rows, lens, self._first(rows)):
            need = -(-n // self.bs)
            if not ok or n < 0 or need > self.width:
                self.errors += 1
                continue
            add = max(0, need - len(self.table[r]))
            asked += add
            full = asked > avail
            if add and full:
                self.errors += 1
                continue
            for _ in range(add):
                p = self.free.pop()
                self.ref[p] = 1
                self.table[r].append(p)

    def release(self, rows, keep):
        freed = []
        for r, k, ok in zip(rows, keep, self._first(rows)):
            if not ok or k < 0:
                self.errors += 1
                continue
            for p in self.table[r][k:]:
                self.ref[p] -= 1
                if self.ref[p] == 0:
                    freed.append(p)
            self.table[r] = self.table[r][:k]
        self.free += sorted(freed)

    def fork(self, src, dst, lens):
        """Pairs of pages to copy ((-1, -1): none)."""
        pairs, asked, avail = [], 0, len(self.free)
        before = [len(t) for t in self.table]
        for s, d, n, ok in zip(src, dst, lens, self._first(dst)):
            pairs.append((-1, -1))
            if not ok or not 0 <= s < len(self.table) or s in dst or n < 0 or before[d] or \
                    -(-n // self.bs) > before[s]:
                self.errors += 1
                continue
            part = n % self.bs > 0
            asked += part
            if part and asked > avail:
                self.errors += 1
                continue
            full = n // self.bs
            self.table[d] = self.table[s][:full]
            for p in self.table[d]:
                self.ref[p] += 1
            if part:
                p = self.free.pop()
                self.ref[p] = 1
                pairs[-1] = (self.table[s][full], p)
                self.table[d].append(p)
        return pairs

    def compact(self):
        """Moves (source, target)."""
        live = [p for p, r in enumerate(self.ref) if r > 0]
        L = len(live)
        movers = [p for p in live if p >= L]
        holes = [p for p in range(L) if self.ref[p] == 0]
        new = dict(zip(movers, holes))
        for s, d in new.items():
            self.ref[d], self.ref[s] = self.ref[s], 0
        self.table = [[new.get(p, p) for p in t] for t in self.table]
        self.free = list(range(len(self.ref) - 1, L - 1, -1))
        return list(new.items())

    def arrays(self):
        """ref, free_list, n_free, block_table, n_blocks as the GPU keeps them."""
        P = len(self.ref)
        return (self.ref, self.free + [-1] * (P - len(self.free)), [len(self.free)],
                [t + [-1] * (self.width - len(t)) for t in self.table], [len(t) for t in self.table])
