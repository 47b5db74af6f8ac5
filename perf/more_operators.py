"""What a decoding step does around its attention: what is measured.

Four operators and their plain forms in elementary torch operations:

  moe      a whole mixture-of-experts layer for a few tokens: router, top-k, the
           picked experts, the shared experts, the residual
  norm     the residual sum behind a block with the block's norm, gate and scale,
           and the norm before the next block; ``train``: with its gradients
  sample   the next token from logits and given random numbers, with temperature,
           top-k, top-p and min-p
  probs    the distribution that ``sample`` draws from (a target for the
           verification of drafted tokens)

``listed()`` names the measured cases, ``draw(rng)`` gives further ones of the
same ranges, ``run(state)`` makes one pass.
"""
import math

import torch

own = False

DEV = "cuda"
VOCAB = 129280                            # the decoder's vocabulary
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _moe(name, tokens, hidden, ffn, experts, topk, shared, dtype="bf16", renorm=False, scale=1.0):
    return dict(name=name, op="moe", tokens=tokens, hidden=hidden, ffn=ffn, experts=experts, topk=topk,
                shared=shared, dtype=dtype, renorm=renorm, scale=scale)


def _norm(name, rows, hidden, dtype="bf16", train=False, gates=0, post=False, scale=1.0):
    return dict(name=name, op="norm", rows=rows, hidden=hidden, dtype=dtype, train=train, gates=gates,
                post=post, scale=scale)


def _pick(name, op, rows, vocab, dtype="bf16", settings="same", masked=False):
    return dict(name=name, op=op, rows=rows, vocab=vocab, dtype=dtype, settings=settings, masked=masked)


def listed():
    return [
        # one sequence: the decoder's layer (64 experts of 896, 6 picked, 2 shared)
        _moe("moe 1 token", 1, 1280, 896, 64, 6, 2),
        # the end-to-end decoder's batch
        _moe("moe 8 tokens", 8, 1280, 896, 64, 6, 2),
        # a serving batch, or 8 sequences with 8 drafted tokens each: every expert is picked
        _moe("moe 64 tokens", 64, 1280, 896, 64, 6, 2),
        # a small model, an odd number of tokens, renormalised weights
        _moe("moe 19 tokens small fp16", 19, 256, 136, 8, 2, 1, dtype="fp16", renorm=True, scale=2.5),
        # between attention and FFN of a decoding step
        _norm("norm 8 x 1280", 8, 1280),
        # the same in a prefill of 4 pages of 9,248 tokens
        _norm("norm 36992 x 1280", 36992, 1280),
        # training: plain residual norm
        _norm("norm train 9248 x 1280", 9248, 1280, train=True),
        # training: a block with a norm behind it and a gate for each sequence
        _norm("norm train 36992 x 1280 gate post", 36992, 1280, train=True, gates=4, post=True, scale=0.5),
        # one sequence, one setting
        _pick("sample 1 row", "sample", 1, VOCAB),
        # a serving batch: every request with settings of its own, some greedy, some masked
        _pick("sample 64 rows mixed", "sample", 64, VOCAB, dtype="fp32", settings="mixed", masked=True),
        # targets for the verification of 8 trees of 16
        _pick("probs 128 rows", "probs", 128, VOCAB),
        # a small vocabulary of odd size
        _pick("probs 5 rows small fp16", "probs", 5, 1003, dtype="fp16", settings="mixed"),
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["moe", "moe", "norm", "norm", "sample", "probs"])
    if op == "moe":
        tokens, experts = _logint(rng, 1, 200), _logint(rng, 2, 96)
        hidden, ffn = 8 * _logint(rng, 4, 256), 8 * _logint(rng, 2, 176)
        topk = rng.randint(1, min(8, experts))
        # no dearer than the largest listed case: the experts' weights, the plain form's products
        while experts * hidden * ffn > 64 * 1280 * 896:
            ffn = max(8, ffn // 16 * 8)
        while tokens * experts * hidden * ffn > 64 * 64 * 1280 * 896:
            tokens //= 2
        return dict(op=op, tokens=max(1, tokens), hidden=hidden, ffn=ffn, experts=experts, topk=topk,
                    shared=rng.choice([0, 1, 2]), dtype=rng.choice(["bf16", "bf16", "fp16"]),
                    renorm=rng.random() < 0.5, scale=rng.choice([1.0, 1.0, 2.5]))
    if op == "norm":
        hidden, train = _logint(rng, 16, 8192), rng.random() < 0.6
        groups = rng.choice([0, 0, 1, 2, 5])
        rows = _logint(rng, 1, min(40000, 36992 * 1280 // hidden))
        if groups:
            rows = max(1, rows // groups) * groups
        return dict(op=op, rows=rows, hidden=hidden, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), train=train,
                    gates=groups, post=rng.random() < 0.4, scale=rng.choice([1.0, 1.0, 0.5, 0.22]))
    return dict(op=op, rows=_logint(rng, 1, 64 if op == "sample" else 128), vocab=_logint(rng, 5, VOCAB),
                dtype=rng.choice(["bf16", "fp16", "fp32"]), settings=rng.choice(["same", "mixed"]),
                masked=rng.random() < 0.4)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _prepare_moe(c, seed):
    g, dt = _gen(seed), _DT[c["dtype"]]
    T, H, F, E = c["tokens"], c["hidden"], c["ffn"], c["experts"]

    def rnd(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device=DEV, dtype=dt).mul_(std)

    s = dict(case=c, x=rnd(T, H), residual=rnd(T, H), gate=rnd(E, H, std=H ** -0.5),
             gu=rnd(E, 2 * F, H, std=H ** -0.5), d=rnd(E, H, F, std=F ** -0.5), sgu=None, sd=None)
    if c["shared"]:
        sf = c["shared"] * F
        s["sgu"], s["sd"] = rnd(2 * sf, H, std=H ** -0.5), rnd(H, sf, std=sf ** -0.5)
    if own:
        from ananta_ocr_b200 import moe
        s["weights"] = moe.MoeWeights(s["gate"], s["gu"], s["d"], s["sgu"], s["sd"])
    return s


def _prepare_norm(c, seed):
    g, dt = _gen(seed), _DT[c["dtype"]]
    R, H, train = c["rows"], c["hidden"], c["train"]

    def rnd(*shape, std=1.0, mean=0.0, dtype=dt, grad=train):
        t = torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).mul_(std).add_(mean).to(dtype)
        return t.requires_grad_(grad)

    s = dict(case=c, y=rnd(R, H), residual=rnd(R, H, std=3.0),
             weight=rnd(H, std=0.2, mean=1.0, dtype=torch.float32), gate=None, post=None, eps=1e-6)
    if c["gates"]:
        s["gate"] = rnd(c["gates"], H, std=0.5, mean=0.5)
    if c["post"]:
        s["post"] = rnd(H, std=0.2, mean=1.0, dtype=torch.float32)
    if train:
        # what comes back from the layers behind: through the stream and through the normed rows
        s["dstream"], s["dnormed"] = rnd(R, H, grad=False), rnd(R, H, grad=False)
    return s


def _prepare_pick(c, seed):
    g = _gen(seed)
    R, V = c["rows"], c["vocab"]
    z = torch.randn(R, V, generator=g, device=DEV) * 2
    # some tokens that the text calls for stand above the rest
    hot = torch.randint(0, V, (R, 48), generator=g, device=DEV)
    z.scatter_add_(1, hot, torch.rand(R, 48, generator=g, device=DEV) * 12)
    if c["masked"]:
        # a grammar leaves a third of the vocabulary, at another place in each row
        at = torch.randint(0, V, (R, 1), generator=g, device=DEV)
        z.masked_fill_((torch.arange(V, device=DEV) + at) % V >= max(1, V // 3), float("-inf"))
    s = dict(case=c, logits=z.to(_DT[c["dtype"]]), u=torch.rand(R, generator=g, device=DEV))
    if c["settings"] == "same":
        s.update(temperature=0.8, top_k=50, top_p=0.95, min_p=0.02)
    else:
        pick = lambda values, dt: torch.tensor(values, dtype=dt, device=DEV)[
            torch.randint(0, len(values), (R,), generator=g, device=DEV)]
        s.update(temperature=pick([0.0, 0.6, 0.8, 1.0, 1.0, 1.3], torch.float32),
                 top_k=pick([0, 0, 1, 20, 50, 1000], torch.int32),
                 top_p=pick([1.0, 1.0, 0.95, 0.9, 0.5], torch.float32),
                 min_p=pick([0.0, 0.0, 0.0, 0.05], torch.float32))
    return s


def prepare(case, seed):
    return {"moe": _prepare_moe, "norm": _prepare_norm}.get(case["op"], _prepare_pick)(case, seed)


# ---------------------------------------------------------------------------
# plain forms and calls
# ---------------------------------------------------------------------------
def _moe_plain(s):
    c, x = s["case"], s["x"].float()
    T, F, E, k = c["tokens"], c["ffn"], c["experts"], c["topk"]
    # in 64 bits: the border between two near experts
    logits = s["x"].double() @ s["gate"].double().t()
    ids = logits.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    p = (logits - logits.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    w = p.gather(1, ids)
    if c["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    w = (w * c["scale"]).float()
    dense = torch.zeros(T, E, device=x.device).scatter(1, ids, w)
    h = torch.matmul(s["gu"].float(), x.t())                           # [E, 2F, T]
    a, b = h[:, :F], h[:, F:]
    y = torch.matmul(s["d"].float(), a / (1 + (-a).exp()) * b)         # [E, H, T]
    out = s["residual"].float() + (y * dense.t()[:, None]).sum(0).t()
    if s["sgu"] is not None:
        h = x @ s["sgu"].float().t()
        a, b = h.chunk(2, -1)
        out = out + (a / (1 + (-a).exp()) * b) @ s["sd"].float().t()
    return out.to(s["x"].dtype), ids.to(torch.int32), w


def _moe_own(s):
    from ananta_ocr_b200 import moe
    c = s["case"]
    r = moe.moe_layer(s["x"], s["weights"], c["topk"], renormalize=c["renorm"], scale=c["scale"], residual=s["residual"])
    return r.out, r.ids, r.weights


def _norm_forward(s, dt):
    """stream, normed and what the gradients need, in ``dt``."""
    c = s["case"]
    y, w = s["y"].to(dt), s["weight"].to(dt)
    r1 = yh = None
    z = y
    if c["post"]:
        r1 = ((y * y).mean(-1, keepdim=True) + s["eps"]).rsqrt()
        yh = y * r1
        z = yh * s["post"].to(dt)
    gate = None
    t = z * c["scale"]
    if c["gates"]:
        gate = s["gate"].to(dt).repeat_interleave(c["rows"] // c["gates"], 0)
        t = t * gate
    stream = s["residual"].to(dt) + t
    r2 = ((stream * stream).mean(-1, keepdim=True) + s["eps"]).rsqrt()
    sh = stream * r2
    return stream, sh * w, (w, r1, yh, z, gate, r2, sh)


def _norm_all(s, dt):
    c, T = s["case"], s["y"].dtype
    with torch.no_grad():
        stream, normed, (w, r1, yh, z, gate, r2, sh) = _norm_forward(s, dt)
        if not c["train"]:
            return [stream, normed]
        dh, ds = s["dnormed"].to(dt), s["dstream"].to(dt)
        # column sums over many rows: in 64 bits
        col = lambda t: t.sum(0, dtype=torch.float64)
        dw = col(dh * sh)
        a = dh * w
        ds = ds + r2 * (a - sh * (a * sh).mean(-1, keepdim=True))
        dz = ds * c["scale"]
        dgate = dpost = None
        if c["gates"]:
            dgate = (dz * z).view(c["gates"], -1, c["hidden"]).sum(1, dtype=torch.float64)
            dz = dz * gate
        dy = dz
        if c["post"]:
            dpost = col(dz * yh)
            b = dz * s["post"].to(dt)
            dy = r1 * (b - yh * (b * yh).mean(-1, keepdim=True))
        return [stream, normed, dy, ds, dw] + [t for t in (dgate, dpost) if t is not None]


def _norm_types(s):
    """The outputs' types: the rows', then those of the weights that have gradients."""
    t = s["y"].dtype
    return [t, t, t, t, torch.float32] + [t] * bool(s["case"]["gates"]) + [torch.float32] * s["case"]["post"]


def _norm_plain(s):
    return [v.to(t) for v, t in zip(_norm_all(s, torch.float32), _norm_types(s))]


def _norm_own(s):
    from ananta_ocr_b200 import norms
    c = s["case"]
    out = norms.add_rms_norm(s["y"], s["residual"], s["weight"], s["eps"], gate=s["gate"], post_weight=s["post"],
                             scale=c["scale"])
    if not c["train"]:
        return list(out)
    leaves = [s["y"], s["residual"], s["weight"]] + [t for t in (s["gate"], s["post"]) if t is not None]
    return [*(t.detach() for t in out), *torch.autograd.grad(out, leaves, [s["dstream"], s["dnormed"]])]


def _column(v, rows):
    """A setting as a 64-bit column, one value per row."""
    if not torch.is_tensor(v):
        v = torch.tensor([v], dtype=torch.float32, device=DEV).expand(rows)
    return v.double()[:, None]


def _keep(s):
    """Weights exp((z - max) / temperature) and which tokens are kept, in 64 bits: the
    borders lie between tokens whose shares are small."""
    z = s["logits"].double()
    R, V = z.shape
    temp, k, p, m = (_column(s[n], R) for n in ("temperature", "top_k", "top_p", "min_p"))
    top = z.amax(-1, keepdim=True)
    greedy = temp <= 0
    x = torch.where(z == top, 0.0, (z - top) / torch.where(greedy, 1.0, temp))
    e = torch.where(z == float("-inf"), 0.0, x.exp())
    zs, order = z.sort(dim=-1, descending=True, stable=True)             # equal ones: the lowest index first
    es = e.gather(1, order)
    n = torch.arange(V, device=z.device)[None]
    keep = (es > 0) & ((k <= 0) | (n < k)) & (~greedy | (n == 0))
    cum = (es * keep).cumsum(-1)
    before = cum - es * keep
    keep &= (p >= 1) | (before < p * cum[:, -1:]) | (n == 0)
    keep &= es >= m
    return e, torch.zeros_like(keep).scatter(1, order, keep)


def _sample_plain(s):
    e, keep = _keep(s)
    m = e * keep
    cum = m.cumsum(-1)
    hit = (cum > s["u"].double()[:, None] * cum[:, -1:]) & (m > 0)
    V = m.shape[1]
    n = torch.arange(V, device=m.device)
    first = torch.where(hit, n, V).amin(-1)
    last = torch.where(m > 0, n, -1).amax(-1)
    return torch.where(first < V, first, last)


def _probs_plain(s):
    e, keep = _keep(s)
    m = e * keep
    total = m.sum(-1, keepdim=True)
    return torch.where(total > 0, m / total, 0.0).float()


def _settings(s):
    return {n: s[n] for n in ("temperature", "top_k", "top_p", "min_p")}


def _sample_own(s):
    from ananta_ocr_b200 import sampling
    return sampling.sample(s["logits"], s["u"], **_settings(s))


def _probs_own(s):
    from ananta_ocr_b200 import sampling
    return sampling.probs(s["logits"], **_settings(s))


def run(state):
    return globals()[f"_{state['case']['op']}_{'own' if own else 'plain'}"](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "moe":
        T, H, F, E, k = c["tokens"], c["hidden"], c["ffn"], c["experts"], c["topk"]
        # experts that T tokens of a balanced router pick
        used = E * (1 - (1 - k / E) ** T)
        per = 3 * F * H
        return {"bytes": 2 * (per * (used + c["shared"]) + E * H + 3 * T * H) + 8 * T * k,
                "flops": 2 * T * (per * (k + c["shared"]) + E * H)}
    if c["op"] == "norm":
        e = 4 if c["dtype"] == "fp32" else 2
        n = c["rows"] * c["hidden"]
        small = c["hidden"] * (4 * (1 + c["post"]) + e * c["gates"]) * (2 if c["train"] else 1)
        # y and residual in, stream and normed out; in training the gradients of both in, of both out
        return {"bytes": n * e * (8 if c["train"] else 4) + small, "flops": n * (30 if c["train"] else 8)}
    e = 4 if c["dtype"] == "fp32" else 2
    n = c["rows"] * c["vocab"]
    return {"bytes": n * e + (n * 4 if c["op"] == "probs" else 8 * c["rows"]), "flops": 8 * n}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def _moe_exact(s):
    """Expert by expert, over the tokens that picked it."""
    c = s["case"]
    x = s["x"].double()
    F = c["ffn"]
    score = (x[:, None, :] * s["gate"].double()[None]).sum(-1)
    ids = torch.empty(c["tokens"], c["topk"], dtype=torch.int64, device=x.device)
    left = score.clone()
    for j in range(c["topk"]):
        # the lowest index among the largest
        best = (left == left.amax(-1, keepdim=True)).double().argmax(-1)
        ids[:, j] = best
        left.scatter_(1, best[:, None], float("-inf"))
    share = score.softmax(-1).gather(1, ids)
    w = c["scale"] * (share / share.sum(-1, keepdim=True) if c["renorm"] else share)
    out = s["residual"].double().clone()

    def ffn(rows, gu, d):
        h = rows @ gu.double().t()
        return (torch.nn.functional.silu(h[:, :gu.shape[0] // 2]) * h[:, gu.shape[0] // 2:]) @ d.double().t()

    for e in range(c["experts"]):
        t, j = (ids == e).nonzero(as_tuple=True)
        if len(t):
            out.index_add_(0, t, ffn(x[t], s["gu"][e], s["d"][e]) * w[t, j, None])
    if s["sgu"] is not None:
        out += ffn(x, s["sgu"], s["sd"])
    return out, ids.to(torch.int32), w


def _norm_exact(s):
    """Through torch's own differentiation in 64 bits."""
    c = s["case"]
    leaf = lambda t: None if t is None else t.detach().double().requires_grad_(c["train"])
    y, res, w, gate, post = (leaf(s[n]) for n in ("y", "residual", "weight", "gate", "post"))
    norm = lambda t, v: t / (t.square().sum(-1, keepdim=True) / c["hidden"] + s["eps"]).sqrt() * v
    b = norm(y, post) if c["post"] else y
    if c["gates"]:
        b = (b.view(c["gates"], -1, c["hidden"]) * gate[:, None]).view_as(b)
    stream = res + c["scale"] * b
    normed = norm(stream, w)
    if not c["train"]:
        return [stream, normed]
    leaves = [t for t in (y, res, w, gate, post) if t is not None]
    grads = torch.autograd.grad([stream, normed], leaves, [s["dstream"].double(), s["dnormed"].double()])
    return [stream.detach(), normed.detach(), *grads]


def _rows_exact(s):
    """Row by row: (indices kept in the vocabulary's order, their weights)."""
    z = s["logits"].double().cpu()
    R, V = z.shape
    at = lambda v, i: float(v[i]) if torch.is_tensor(v) else float(torch.tensor(v, dtype=torch.float32))
    host = {n: (s[n].cpu() if torch.is_tensor(s[n]) else s[n]) for n in ("temperature", "top_k", "top_p", "min_p")}
    for i in range(R):
        temp, k, p, m = (at(host[n], i) for n in ("temperature", "top_k", "top_p", "min_p"))
        idx = torch.argsort(z[i], descending=True, stable=True)
        idx = idx[z[i, idx] > float("-inf")]
        if temp <= 0:
            idx = idx[:1]
        if k > 0:
            idx = idx[:int(k)]
        if not len(idx):
            yield idx, z[i, idx]
            continue
        e = ((z[i, idx] - z[i, idx[0]]) / (temp if temp > 0 else 1.0)).exp()
        n = len(idx)
        if p < 1:
            n = 1 + int((e.cumsum(0)[:-1] < p * e.sum()).sum())
        n = min(n, max(1, int((e >= m).sum())))
        kept, back = idx[:n].sort()
        yield kept, e[:n][back]


def _sample_exact(s):
    u = s["u"].double().cpu()
    out = []
    for i, (kept, e) in enumerate(_rows_exact(s)):
        if not len(kept):
            out.append(-1)
            continue
        cum = e.cumsum(0)
        out.append(int(kept[min(len(kept) - 1, int((cum <= u[i] * cum[-1]).sum()))]))
    return torch.tensor(out, device=DEV)


def _probs_exact(s):
    out = torch.zeros(s["logits"].shape, dtype=torch.float64)
    for i, (kept, e) in enumerate(_rows_exact(s)):
        if len(kept):
            out[i, kept] = e / e.sum()
    return out.to(DEV)


def exact(case, seed):
    if case["op"] == "moe" and case["tokens"] * case["experts"] * case["hidden"] > 1 << 28:
        return None                        # the router's products of all pairs, laid out at once
    state = prepare(case, seed)
    return globals()[f"_{case['op']}_exact"](state)
