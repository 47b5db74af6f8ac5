"""Decode and draft steps with fused norms and MoE layers, and with tokens drawn by
settings: the operators run together as a decoder calls them.

The measure against plain torch forms of the same step is the one of the decoder's own tests,
2% of the largest logit: every row is rounded to bf16 a dozen times per layer on
both sides, in places that are not the same.  The plain forms pick experts by the same
64-bit scores, so that they differ by roundings only."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

from ananta_ocr_b200 import moe, norms, sampling
from ananta_ocr_b200.e2e_decoder import DashDecoder, DecoderConfig
from oracle import draft_oracle as DO
from step_testutil import distribution, draw

pytestmark = pytest.mark.gpu

CFG = DecoderConfig(hidden=256, heads=2, kv_heads=2, layers=3, vocab=1000, dense_ffn=512, moe_ffn=128, experts=8, topk=2, shared=1)


def make(batch=2, fused=True, **kw):
    return DashDecoder(CFG, batch=batch, max_len=420, device=torch.device("cuda"), seed=3, fused_steps=fused, **kw)


def start(dec, S=150, seed=1):
    ids = torch.randint(0, 1000, (dec.B, S), generator=torch.Generator().manual_seed(seed)).cuda()
    dec.prefill(dec.embed[ids])
    dec.tok.fill_(7)
    return dec


def plain_norm(x, w, eps):
    f = x.float()
    return (f * (f.square().mean(-1, keepdim=True) + eps).rsqrt() * w).to(x.dtype)


def plain_add(y, residual, w, eps, **kw):
    f = residual.float() + y.float()
    return f.to(y.dtype), (f * (f.square().mean(-1, keepdim=True) + eps).rsqrt() * w).to(y.dtype)


def plain_moe(x, w, topk, *, residual, **kw):
    gate, gu, d, sgu, sd = (t.double() for t in w.tensors)
    X = x.double()
    score = X @ gate.t()
    ids = score.sort(dim=-1, descending=True, stable=True).indices[:, :topk]
    p = score.softmax(-1).gather(1, ids)
    ffn = lambda v, g, e: (F.silu((v @ g.t()).chunk(2, -1)[0]) * (v @ g.t()).chunk(2, -1)[1]) @ e.t()  # noqa: E731
    out = residual.double() + ffn(X, sgu, sd)
    for t in range(len(x)):
        for j in range(topk):
            out[t] += p[t, j] * ffn(X[t:t + 1], gu[ids[t, j]], d[ids[t, j]])[0]
    return moe.MoeOut(out.to(x.dtype), ids.int(), p.float())


@pytest.mark.parametrize("batch", [1, 2, 5])
def test_steps_are_those_of_the_plain_forms(batch, monkeypatch):
    a, b = start(make(batch)), start(make(batch))
    extra = torch.randint(0, 1000, (batch, 4), generator=torch.Generator().manual_seed(5)).cuda()
    got = [a.decode_step().float(), a.draft_step(extra)[1].float()]
    monkeypatch.setattr(norms, "rms_norm", plain_norm)
    monkeypatch.setattr(norms, "add_rms_norm", plain_add)
    monkeypatch.setattr(moe, "moe_layer", plain_moe)
    first = b.decode_step().float()
    assert torch.isfinite(got[0]).all() and torch.isfinite(got[1]).all()
    assert (got[0] - first).abs().max() <= 0.02 * first.abs().max()
    if torch.equal(got[0].argmax(-1), first.argmax(-1)):               # the same roots of the trees
        w = b.draft_step(extra)[1].float()
        assert (got[1] - w).abs().max() <= 0.02 * w.abs().max()


def test_default_steps_do_not_call_them(monkeypatch):
    def no(*a, **k):
        raise AssertionError("called")
    for m, name in ((norms, "rms_norm"), (norms, "add_rms_norm"), (moe, "moe_layer"), (sampling, "sample"), (sampling, "probs")):
        monkeypatch.setattr(m, name, no)
    dec = start(make(fused=False))
    dec.decode_step()
    dec.draft_step(torch.zeros(2, 3, dtype=torch.int64, device="cuda"))


def test_graphs_equal_eager_steps():
    a, b = start(make(pool_pages=40)), start(make(pool_pages=40))
    u = torch.tensor([0.3, 0.8], device="cuda")
    kw = dict(temperature=0.9, top_k=30, top_p=0.95)
    eager = [a.decode_step(u, **kw).clone() for _ in range(3)]
    b.decode_step(u, **kw)
    start(b)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = b.decode_step(u, **kw)
    for e in eager:
        g.replay()
        assert torch.equal(out, e)
    assert torch.equal(a.tok, b.tok) and torch.equal(a.seq_lens, b.seq_lens)


@pytest.mark.parametrize("fused", [False, True])
def test_drawn_tokens(fused):
    """decode_step draws what the definition draws from its logits."""
    dec = start(make(4, fused))
    for i, kw in enumerate((dict(), dict(temperature=0.7, top_k=5), dict(top_p=0.8, min_p=0.01), dict(temperature=0.0))):
        u = torch.rand(4, generator=torch.Generator().manual_seed(i)).cuda()
        logits = dec.decode_step(u, **kw).double().cpu().numpy()
        f = lambda v: float(np.float32(v))  # noqa: E731
        s = (f(kw.get("temperature", 1.0)), kw.get("top_k", 0), f(kw.get("top_p", 1.0)), f(kw.get("min_p", 0.0)))
        assert dec.tok.tolist() == [draw(logits[r], float(u[r]), *s) for r in range(4)]


def test_settings_per_sequence():
    dec = start(make(3))
    u = torch.tensor([0.9, 0.9, 0.2], device="cuda")
    t = torch.tensor([0.0, 1.0, 2.0], device="cuda")
    k = torch.tensor([0, 1, 10], dtype=torch.int32, device="cuda")
    logits = dec.decode_step(u, temperature=t, top_k=k)
    best = logits.argmax(-1)
    assert dec.tok[0] == best[0] and dec.tok[1] == best[1]
    assert dec.tok[2] in logits[2].float().topk(10).indices


@pytest.mark.parametrize("fused", [False, True])
def test_drafts_against_a_cut_target(fused):
    """Random numbers and settings in, the oracle's tokens on the cut distribution out."""
    n = 5
    dec = start(make(2, fused), S=100)
    extra = torch.randint(0, 1000, (2, n - 1), generator=torch.Generator().manual_seed(6)).cuda()
    g = torch.Generator().manual_seed(7)
    ua, us = torch.rand(2 * n, generator=g).cuda() * 0.2, torch.rand(2, generator=g).cuda()
    tok = dec.tok.clone()
    kept, logits = dec.draft_step(extra, temperature=1.5, u_accept=ua, u_sample=us, top_k=200, top_p=0.9, min_p=0.001)
    rows = logits.reshape(2 * n, -1).double().cpu().numpy()
    f = lambda v: float(np.float32(v))  # noqa: E731
    target = np.stack([distribution(r, 1.5, 200, f(0.9), f(0.001)) for r in rows])
    tokens = torch.cat([tok[:, None], extra], 1).reshape(-1).cpu().numpy()
    want = DO.verify(tokens, None, [0, n, 2 * n], target, None, ua.cpu().numpy(), us.cpu().numpy(), "certain", n)
    for got, w in zip((kept.n_accept, kept.path, kept.next_token, kept.tokens), want):
        np.testing.assert_array_equal(got.cpu().numpy(), w)


def test_more_tokens_than_the_layer_takes(monkeypatch):
    """Steps of more than 256 tokens go through the default MoE."""
    monkeypatch.setattr(moe, "MAX_TOKENS", 8)
    dec = start(make(3))
    assert torch.isfinite(dec.draft_step(torch.zeros(3, 3, dtype=torch.int64, device="cuda"))[1]).all()
