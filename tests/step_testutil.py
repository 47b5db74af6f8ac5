"""Definitions in 64 bits of the operators around a step's attention (norms, sampling,
mixture of experts), for the tests."""
import numpy as np
import torch

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U = 2.0 ** -24                                # half a step of fp32


def half_step(dt):
    return torch.finfo(dt).eps / 2


# ---------------------------------------------------------------------------
# norms
# ---------------------------------------------------------------------------
def norm_forward(y, residual, weight, gate, post, eps, scale):
    """(stream, normed) in the inputs' (64-bit) type; gate [groups, hidden] or None."""
    rows, hidden = y.shape
    n = lambda t, w: t / (t.square().mean(-1, keepdim=True) + eps).sqrt() * w  # noqa: E731
    z = y if post is None else n(y, post)
    if gate is not None:
        z = (z.reshape(gate.shape[0], -1, hidden) * gate[:, None]).reshape(rows, hidden)
    s = z * scale if residual is None else residual + scale * z
    return s, n(s, weight)


def norm_grads(y, residual, weight, gate, post, eps, scale, ds, dh):
    """By the formulas; with them the sums of the absolute terms that each gradient is made of
    (what its rounding errors are shares of): {name: (gradient, terms)}."""
    rows, hidden = y.shape
    groups = 1 if gate is None else gate.shape[0]
    rep = lambda t: t.repeat_interleave(rows // groups, 0)  # noqa: E731
    f = torch.full_like(y, scale) if gate is None else scale * rep(gate)
    r1 = torch.ones(rows, 1, dtype=y.dtype) if post is None else (y.square().mean(-1, keepdim=True) + eps).rsqrt()
    p = torch.ones_like(y) if post is None else post.expand_as(y)
    q = f * p * y
    s = q * r1 + (0 if residual is None else residual)
    size = (q * r1).abs() + (0 if residual is None else residual.abs())
    r2 = (s.square().mean(-1, keepdim=True) + eps).rsqrt()
    sh, shs = s * r2, size * r2
    a = dh * weight
    mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    d = ds + r2 * (a - sh * mean(a * sh))
    dt = ds.abs() + r2 * (a.abs() + shs * mean(a.abs() * shs)) * (1 + mean(shs * shs))
    out = {"residual": (d, dt), "weight": ((dh * sh).sum(0), (dh.abs() * shs).sum(0))}
    dz, dzt = d * f, dt * f.abs()
    yh = y * r1
    z = yh * p
    gsum = lambda t: t.reshape(groups, -1, hidden).sum(1)  # noqa: E731
    out["gate"] = (gsum(scale * z * d), gsum(abs(scale) * z.abs() * dt))
    if post is None:
        out["y"] = (dz, dzt)
    else:
        b, bt = dz * p, dzt * p.abs()
        out["y"] = (r1 * (b - yh * mean(b * yh)), r1 * (bt + yh.abs() * mean(bt * yh.abs())))
    out["post"] = ((dz * yh).sum(0), (dzt * yh.abs()).sum(0))
    return out


# ---------------------------------------------------------------------------
# sampling
# ---------------------------------------------------------------------------
def kept(z, temperature, top_k, top_p, min_p):
    """One row (64-bit numpy): the kept indices in descending order and their weights."""
    z = z + 0.0
    order = np.argsort(-np.where(np.isnan(z), -np.inf, z), kind="stable")
    order = order[z[order] > -np.inf]
    if not len(order):
        return order, np.zeros(0)
    if temperature <= 0:
        return order[:1], np.ones(1)
    if top_k > 0:
        order = order[:top_k]
    top = z[order[0]]
    with np.errstate(invalid="ignore"):
        e = np.where(z[order] == top, 1.0, np.exp((z[order] - top) / temperature))
    n = len(order)
    if top_p < 1:
        n = 1 + int((np.cumsum(e)[:-1] < top_p * e.sum()).sum())
    n = min(n, max(1, int((e >= min_p).sum())))
    return order[:n], e[:n]


def draw(z, u, *setting):
    order, e = kept(z, *setting)
    if not len(order):
        return -1
    back = np.argsort(order)
    cum = np.cumsum(e[back])
    return int(order[back][min(len(order) - 1, int((cum <= u * cum[-1]).sum()))])


def distribution(z, *setting):
    order, e = kept(z, *setting)
    out = np.zeros(len(z))
    if len(order):
        out[order] = e / e.sum()
    return out


# ---------------------------------------------------------------------------
# mixture of experts
# ---------------------------------------------------------------------------
def moe(x, gate, gu, down, sgu, sd, topk, renorm, scale, residual, dtype, least=2.0 ** -25):
    """64-bit tensors -> (out, ids, weights, tolerance).

    The tolerance counts: the output's rounding; each inner product of n terms in fp32,
    off by n * 2^-24 of the sum of its absolute terms at most; the inner values' two
    numbers of the type (half a step of half a step, and for fp16 its smallest number),
    and 2^-20 of an inner value for exp and the division."""
    T, H = x.shape
    F = down.shape[2]
    score = x @ gate.t()
    score = torch.where(score.isnan(), torch.full_like(score, -torch.inf), score)
    ids = score.sort(dim=-1, descending=True, stable=True).indices[:, :topk]
    p = score.softmax(-1).gather(1, ids)
    w = p / p.sum(-1, keepdim=True) if renorm else p
    w = w * scale
    out = torch.zeros_like(x) if residual is None else residual.clone()
    tol = out.abs() * U * (topk + 3)
    two = half_step(dtype) ** 2 * 2 + 2.0 ** -20            # (`least`: the inner values' smallest error)

    def ffn(v, g, d, weight):
        n = d.shape[1]
        h, ht = g @ v, g.abs() @ v.abs() * H * U
        a, b = h[:n], h[n:]
        act = a * torch.sigmoid(a) * b
        # |d silu| <= 1.1, |silu| <= |a|
        at = 1.1 * ht[:n] * (b.abs() + ht[n:]) + a.abs() * ht[n:] + act.abs() * two + least
        mag = d.abs() @ act.abs()
        return weight * (d @ act), abs(weight) * (d.abs() @ at + mag * (n + topk + 3) * U)

    for t in range(T):
        parts = [ffn(x[t], gu[int(e)], down[int(e)], float(w[t, j])) for j, e in enumerate(ids[t])]
        if sgu is not None:
            parts.append(ffn(x[t], sgu, sd, 1.0))
        for v, e in parts:
            out[t] += v
            tol[t] += e
    return out, ids.to(torch.int32), w, tol + out.abs() * half_step(dtype) + 2.0 ** -25
