"""Speculative decoding through the end-to-end decoder: the drafted tokens' logits
are those of a prefill of each token's own path, the kept path is what the
verification's definition gives on them, and the caches afterwards are those of
the committed sequence.

Paths that sum in another order differ by what bf16 layers make of it, and by no
fixed share: the router's prior turns small differences of scores into biases.
The measure here is the decode step, whose operators are tested on their own: the
draft step may differ from a prefill by three times the most that decode steps
over the same tokens differ from it (the same kind of roundings, drawn anew),
and by 10% in all (a key too many or too few changes a token by far more).  All
layers have a dense FFN, because an expert gate whose two best experts are near
each other picks another one under such differences."""
import numpy as np
import pytest
import torch

from ananta_ocr_b200 import _lib as L
from ananta_ocr_b200.e2e_decoder import DashDecoder, DecoderConfig
from oracle import draft_oracle as DO

pytestmark = pytest.mark.gpu

SMALL = dict(hidden=256, heads=2, kv_heads=2, layers=3, vocab=1000, dense_ffn=512, moe_ffn=128,
             experts=8, topk=2, shared=1, first_dense=3)
CFGS = {"bs64": DecoderConfig(**SMALL, block_size=64, local_blocks=2, K=4, topm=4, slots=4),
        "bs32": DecoderConfig(**SMALL)}
PARENTS = [-1, 0, 0, 1, 1, 2, 3]


def make(cfg, batch=2, max_len=420, **kw):
    return DashDecoder(cfg, batch=batch, max_len=max_len, device=torch.device("cuda"), seed=3, **kw)


def ids_of(S, seed, batch=2):
    return torch.randint(0, 1000, (batch, S), generator=torch.Generator().manual_seed(seed)).cuda()


def off(a, b):
    """Relative 2-norm of the difference, row by row."""
    return ((a.float() - b.float()).norm(dim=-1) / b.float().norm(dim=-1)).max().item()


def decode_noise(cfg, ids, way, whole):
    """How far decode steps over ``way`` [B, k] are off a prefill's logits."""
    one = make(cfg, batch=ids.shape[0])
    one.prefill(one.embed[ids])
    for i in range(way.shape[1]):
        one.tok.copy_(way[:, i])
        got = one.decode_step()
    return off(got, whole)


def paths(parents):
    out = []
    for i in range(len(parents)):
        p, way = i, []
        while p >= 0:
            way.append(p)
            p = parents[p]
        out.append(way[::-1])
    return out


@pytest.mark.parametrize("pool", [0, 40])
@pytest.mark.parametrize("name", sorted(CFGS))
def test_draft_step_equals_prefills_of_the_paths(name, pool):
    cfg, S, n = CFGS[name], 349, len(PARENTS)         # 349 + 7 crosses a 32-token page
    ids, extra = ids_of(S, 1), ids_of(n, 2)
    dec = make(cfg, pool_pages=pool)
    dec.prefill(dec.embed[ids])
    dec.tok.copy_(extra[:, 0])
    par = torch.tensor(PARENTS, dtype=torch.int32).cuda().expand(2, n)
    # the second sequence drafts what greedy decoding picks, as far as one token tells
    ref = make(cfg)
    first = ref.prefill(ref.embed[torch.cat([ids, extra[:, :1]], 1)]).argmax(-1)
    extra[1, 2] = first[1]
    kept, logits = dec.draft_step(extra[:, 1:], par)
    err, noise = [], []
    for i, way in enumerate(paths(PARENTS)):
        whole = ref.prefill(ref.embed[torch.cat([ids, extra[:, way]], 1)])
        err.append(off(logits[:, i], whole))
        noise.append(decode_noise(cfg, ids, extra[:, way], whole))
    limit = min(0.1, 3 * max(noise))
    assert max(err) <= limit, (err, noise)
    want = DO.verify(torch.cat([extra.reshape(-1).cpu()]).numpy(), np.array(PARENTS * 2), [0, n, 2 * n],
                     logits.reshape(2 * n, -1).double().cpu().numpy(), None, None, None, "greedy", n)
    for got, w in zip((kept.n_accept, kept.path, kept.next_token, kept.tokens), want):
        np.testing.assert_array_equal(got.cpu().numpy(), w)
    assert kept.n_accept[1] >= 1 and kept.path[1, 1] == 2          # a move: token 2 -> 1
    # the committed sequences go on as their prefills do
    assert torch.equal(dec.seq_lens.cpu(), S + 1 + kept.n_accept.cpu())
    step = dec.decode_step()
    for b in range(2):
        k = int(kept.n_accept[b])
        whole = torch.cat([ids[b], extra[b, :1], kept.tokens[b, :k + 1]])
        one = make(cfg, batch=1)
        assert off(step[b:b + 1], one.prefill(one.embed[whole[None]])) <= limit, b
    if pool:
        bs = cfg.block_size
        need = [-(-int(x) // bs) for x in dec.seq_lens]
        assert dec.pool.n_blocks.tolist() == need and dec.pool.n_free.item() == pool - sum(need)


def test_draft_steps_give_the_greedy_text():
    """Ten draft steps whose drafts are the true next tokens (and wrong ones)
    give the text of greedy decoding."""
    cfg, S = CFGS["bs64"], 200
    ids = ids_of(S, 4)
    a, b = make(cfg), make(cfg, pool_pages=30)
    a.tok.copy_(a.prefill(a.embed[ids]).argmax(-1))
    b.tok.copy_(b.prefill(b.embed[ids]).argmax(-1))
    assert torch.equal(a.tok, b.tok)
    text = [a.tok.clone()]
    margins = []
    for _ in range(24):
        top = a.decode_step().float().topk(2, -1).values
        margins.append((top[:, 0] - top[:, 1]) / top[:, 0].abs())
        text.append(a.tok.clone())
    text, margins = torch.stack(text, 1), torch.stack(margins, 1)
    at = torch.zeros(2, dtype=torch.long)
    for step in range(10):
        drafts = torch.stack([torch.stack([text[r, min(24, int(at[r]) + i)] for i in (1, 2, 3)]) for r in range(2)])
        if step % 3 == 2:
            drafts[:, 1] = (drafts[:, 1] + 1) % 1000
        kept, _ = b.draft_step(drafts)
        for r in range(2):
            k, p = int(kept.n_accept[r]), int(at[r])
            if p + k + 1 > 24:
                continue
            same = kept.tokens[r, :k + 1].cpu() == text[r, p + 1:p + k + 2].cpu()
            # a token may differ where two logits are as near as the paths' sums
            assert (same | (margins[r, p:p + k + 1].cpu() < 0.02)).all(), (step, r)
            if not same.all():
                return
            assert k == (1 if step % 3 == 2 else 3) or (margins[r, p:p + 4] < 0.02).any()
            at[r] += k + 1


def test_sampled_draft_step():
    """Random numbers in, the oracle's tokens out."""
    cfg, S, n = CFGS["bs32"], 100, 5
    ids, extra = ids_of(S, 5), ids_of(n, 6)
    dec = make(cfg)
    dec.prefill(dec.embed[ids])
    dec.tok.copy_(extra[:, 0])
    g = torch.Generator().manual_seed(7)
    q = torch.rand(2 * n, 1000, generator=g).softmax(-1).cuda()
    ua, us = torch.rand(2 * n, generator=g).cuda() * 0.5, torch.rand(2, generator=g).cuda()
    kept, logits = dec.draft_step(extra[:, 1:], temperature=2.0, draft_probs=q, u_accept=ua, u_sample=us)
    target = (logits.reshape(2 * n, -1).float() / 2.0).softmax(-1)
    want = DO.verify(extra.reshape(-1).cpu().numpy(), None, [0, n, 2 * n], target.double().cpu().numpy(),
                     q.double().cpu().numpy(), ua.cpu().numpy(), us.cpu().numpy(), "drawn", n)
    for got, w in zip((kept.n_accept, kept.path, kept.next_token, kept.tokens), want):
        np.testing.assert_array_equal(got.cpu().numpy(), w)


def test_pool_decodes_as_the_fixed_table():
    """The same pages' contents under other ids: bit for bit the same logits."""
    cfg, ids = CFGS["bs32"], ids_of(150, 8)
    a, b = make(cfg), make(cfg, pool_pages=60)
    assert torch.equal(a.prefill(a.embed[ids]), b.prefill(b.embed[ids]))
    for d in (a, b):
        d.tok.fill_(7)
    for i in range(12):
        assert torch.equal(a.decode_step(), b.decode_step())
        if i == 5:
            b.compact()
    assert b.pool.n_blocks.tolist() == [6, 6]
    b.prefill(b.embed[ids[:, :40]])                       # pages of the first text go back
    assert b.pool.n_free.item() == 60 - 4


@pytest.mark.parametrize("pool", [0, 80])
def test_fork_continues_as_its_source(pool):
    cfg, ids = CFGS["bs32"], ids_of(150, 9, batch=4)
    dec = make(cfg, batch=4, pool_pages=pool)
    dec.prefill(dec.embed[ids])
    dec.tok.fill_(11)
    dec.fork([0, 0], [2, 3])
    out = dec.decode_step()
    assert off(out[2], out[0]) < 0.02 and off(out[3], out[0]) < 0.02 and off(out[1], out[0]) > 0.3
    dec.tok[2:].fill_(500)                                # the copies go their own way
    before = dec.decode_step()
    ref = make(cfg, batch=1)
    for r, t in ((0, None), (2, 500), (3, 500)):
        # row r: the text, token 11, then row 0's choice or 500
        second = out[0].argmax() if t is None else torch.tensor(t, device="cuda")
        text = torch.cat([ids[0], torch.tensor([11], device="cuda"), second[None]])
        whole = ref.prefill(ref.embed[text[None]])
        noise = decode_noise(cfg, ids[:1], text[None, 150:], whole)
        assert off(before[r:r + 1], whole) <= min(0.1, 3 * max(noise, 0.01)), r
    if pool:
        bt = dec.block_table.cpu()
        assert torch.equal(bt[0, :4], bt[2, :4]) and bt[0, 4] != bt[2, 4] and bt[2, 4] != bt[3, 4]
        held = pool - dec.pool.n_free.item()
        dec.compact()
        assert dec.block_table.max().item() == held - 1
        assert torch.isfinite(dec.decode_step()).all()
    with pytest.raises(ValueError):
        dec.fork([0], [0])
    with pytest.raises(ValueError):
        dec.fork([0], [4])


def test_no_page_left():
    """A pool without a page for a row: recorded, and the other row goes on as
    it would alone (bit for bit: the same rows in the same batch)."""
    cfg, S = CFGS["bs32"], 64                              # two full pages each
    ids = ids_of(S, 12)
    rich, poor = make(cfg, pool_pages=12), make(cfg, pool_pages=5)
    with pytest.raises(ValueError, match="do not fit"):
        poor.prefill(poor.embed[ids_of(81, 1)])
    for d in (rich, poor):
        d.prefill(d.embed[ids])
        d.tok.fill_(5)
        guard = [k.clone() for k in d.kbar]
    for step in range(3):
        if step < 2:
            a, b = (d.decode_step() for d in (rich, poor))
        else:
            x = ids_of(3, 13)
            a, b = (d.draft_step(x)[1] for d in (rich, poor))
        assert torch.equal(a[0], b[0]), step
        assert rich.errors.read()[0] == 0 and poor.errors.read()[0] == L.DASH_DEV_NO_PAGE
    assert poor.block_table[1, 2].item() == -1 and poor.pool.n_free.item() == 0
    held = poor.block_table[1, :2].long()
    for k, g in zip(poor.kbar, guard):
        assert torch.equal(k[held], g[held])


def test_a_root_alone():
    """draft_step without drafts is a decode step."""
    cfg, ids = CFGS["bs64"], ids_of(100, 14)
    a, b = make(cfg), make(cfg, pool_pages=12)
    for d in (a, b):
        d.prefill(d.embed[ids])
        d.tok.fill_(9)
    one = a.decode_step()
    kept, logits = b.draft_step(torch.zeros(2, 0, dtype=torch.int64, device="cuda"))
    assert off(logits[:, 0], one) <= 0.1 and kept.n_accept.tolist() == [0, 0]
    assert torch.equal(b.tok, logits[:, 0].argmax(-1)) and b.seq_lens.tolist() == [101, 101]


def test_draft_step_refusals():
    cfg = CFGS["bs64"]
    dec = make(cfg)
    with pytest.raises(ValueError, match="local window"):
        dec.draft_step(torch.zeros(2, 65, dtype=torch.int64, device="cuda"))
    paged = make(cfg, page_cfg=dict(image_token_id=900, page_token_id=901, per_page_image_tokens=41))
    with pytest.raises(NotImplementedError):
        paged.draft_step(torch.zeros(2, 2, dtype=torch.int64, device="cuda"))
    with pytest.raises(NotImplementedError):
        paged.fork([0], [1])
    with pytest.raises(ValueError, match="pool"):
        dec.compact()


def test_draft_step_in_a_graph():
    """A captured draft step replayed equals the eager steps."""
    cfg, S, n = CFGS["bs32"], 120, 4
    ids = ids_of(S, 10)
    a, b = make(cfg, pool_pages=40), make(cfg, pool_pages=40)
    drafts = [ids_of(n - 1, 20 + i) for i in range(3)]
    for d in (a, b):
        d.prefill(d.embed[ids])
        d.tok.fill_(5)
    buf = drafts[0].clone()
    eager = [a.draft_step(x)[1].clone() for x in drafts]
    b.draft_step(buf)                                      # warm-up, then back to the start
    b.prefill(b.embed[ids])
    b.tok.fill_(5)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kept, logits = b.draft_step(buf)
    for x, e in zip(drafts, eager):
        buf.copy_(x)
        g.replay()
        assert torch.equal(logits, e)
    assert torch.equal(a.seq_lens, b.seq_lens) and torch.equal(a.tok, b.tok)
