"""Draft steps where the pages end: at a row's last token and on an empty pool.
A draft without a page is passed over, a full row stays full, and the other
rows' results are those that they get beside a row with room."""
import numpy as np
import pytest
import torch

from ananta_ocr_b200 import _lib as L
from ananta_ocr_b200.e2e_decoder import DashDecoder, DecoderConfig
from oracle import draft_oracle as DO

pytestmark = pytest.mark.gpu

CFG = DecoderConfig(hidden=256, heads=2, kv_heads=2, layers=3, vocab=1000, dense_ffn=512, moe_ffn=128, experts=8,
                    topk=2, shared=1, first_dense=3)                    # blocks of 32 tokens, a window of 4


def make(max_len=128, pool=0):
    return DashDecoder(CFG, batch=2, max_len=max_len, device=torch.device("cuda"), seed=3, pool_pages=pool)


def ids_of(S, seed):
    return torch.randint(0, 1000, (2, S), generator=torch.Generator().manual_seed(seed)).cuda()


def started(ids, lens, pool):
    """A decoder whose rows hold the first ``lens`` tokens of ``ids``."""
    d = make(pool=pool)
    d.prefill(d.embed[ids])
    d.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
    d.tok.fill_(5)
    return d


def verified(kept, logits, tokens, ok):
    """The verification of the drafts with a slot (``ok`` [2, n]) on these logits."""
    n = tokens.shape[1]
    toks = torch.where(ok, tokens, -1).reshape(-1).cpu().numpy()
    want = DO.verify(toks, None, [0, n, 2 * n], logits.reshape(2 * n, -1).double().cpu().numpy(), None, None, None,
                     "greedy", n)
    for name, got, w in zip(("n_accept", "path", "next_token", "tokens"),
                            (kept.n_accept, kept.path, kept.next_token, kept.tokens), want):
        np.testing.assert_array_equal(got.cpu().numpy(), w, err_msg=name)


@pytest.mark.parametrize("pool", [0, 8])
@pytest.mark.parametrize("length", [124, 126, 127, 128])
def test_drafts_across_the_last_page(length, pool):
    """Row 1 has room for 128 - length tokens, the drafts are what greedy decoding
    picks; then decode steps and another draft step on the full row.  Row 0 beside
    it: bit for bit what it is beside a row with room."""
    ids, n = ids_of(128, 1), 5
    probe, full, ref = (started(ids, [60, length], pool), started(ids, [60, length], pool),
                        started(ids, [60, 60], pool))
    best = []
    for _ in range(n - 1):                                 # (on a full row these mean nothing)
        probe.decode_step()
        best.append(probe.tok.clone())
    drafts = torch.stack(best, 1)
    assert probe.seq_lens.tolist() == [64, min(length + 4, 128)]
    kept, logits = full.draft_step(drafts)
    _, other = ref.draft_step(drafts)
    assert torch.equal(logits[0], other[0])
    ok = torch.tensor([60, length], device="cuda")[:, None] + torch.arange(n, device="cuda") < 128
    tokens = torch.cat([torch.full((2, 1), 5, device="cuda"), drafts], 1)
    verified(kept, logits, tokens, ok)
    assert kept.n_accept[1] <= max(0, 127 - length) and (length > 126 or kept.n_accept[1] >= 1)
    assert full.seq_lens[1].item() == min(length + 1 + kept.n_accept[1].item(), 128)
    # (a pool refuses the root of a full row before the plan finds no page for it)
    assert full.errors.read()[0] == (L.DASH_DEV_BAD_ROW if pool and length == 128 else L.DASH_DEV_BAD_PAGE)
    assert ref.errors.read()[0] == 0
    ref.tok.copy_(full.tok)
    for step in range(6):
        if step == 4:
            x, y = (d.draft_step(drafts)[1] for d in (full, ref))
        else:
            x, y = (d.decode_step() for d in (full, ref))
        assert torch.equal(x[0], y[0]), step
        assert full.seq_lens[0] == ref.seq_lens[0] and full.seq_lens[1].item() <= 128
        assert torch.isfinite(x).all()
        ref.tok.copy_(full.tok)
    assert full.seq_lens[1].item() == 128 and full.errors.read()[0] != 0


def test_a_full_row_in_a_graph():
    """A captured decode step replayed past a row's last page equals eager steps."""
    ids = ids_of(128, 2)
    a, b = started(ids, [60, 125], 0), started(ids, [60, 125], 0)
    b.decode_step()
    b.seq_lens.copy_(torch.tensor([60, 125], dtype=torch.int32))
    b.tok.fill_(5)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = b.decode_step()
    for _ in range(6):
        g.replay()
        assert torch.equal(a.decode_step(), out)
    assert a.seq_lens.tolist() == b.seq_lens.tolist() == [66, 128]


@pytest.mark.parametrize("sampled", [False, True])
def test_a_pool_with_pages_for_the_roots_only(sampled):
    """Two rows of two full pages and two pages left: each root gets one, the
    drafts behind the first page's end get none and are passed over."""
    ids, n = ids_of(64, 4), 40
    drafts = ids_of(n - 1, 5)
    kw = {}
    if sampled:
        # numbers of 0: every draft that is tried is kept
        kw = dict(temperature=1.0, u_accept=torch.zeros(2 * n, device="cuda"), u_sample=torch.full((2,), 0.5, device="cuda"))
    out = []
    for pool in (12, 6):
        d = make(max_len=200, pool=pool)
        d.prefill(d.embed[ids])
        d.tok.fill_(5)
        out.append((d, *d.draft_step(drafts, **kw)))
    (rich, _, a), (poor, kept, b) = out
    assert torch.equal(a[:, :32], b[:, :32])
    assert rich.errors.read()[0] == 0 and poor.errors.read()[0] == L.DASH_DEV_NO_PAGE
    assert poor.pool.n_free.item() == 0 and poor.pool.n_blocks.tolist() == [3, 3]
    if sampled:
        assert kept.n_accept.tolist() == [31, 31] and poor.seq_lens.tolist() == [96, 96]
        assert out[0][1].n_accept.tolist() == [39, 39]
        cum = b[:, 31].float().softmax(-1).double().cumsum(-1)
        for r in range(2):
            t = int(kept.next_token[r])
            assert cum[r, t] > 0.5 * cum[r, -1] and (t == 0 or cum[r, t - 1] <= 0.5 * cum[r, -1])
    else:
        ok = (torch.arange(n, device="cuda") < 32).expand(2, n)
        verified(kept, b, torch.cat([torch.full((2, 1), 5, device="cuda"), drafts], 1), ok)


def test_a_prefill_longer_than_the_tables():
    d = make(max_len=64)
    with pytest.raises(ValueError, match="do not fit"):
        d.prefill(d.embed[ids_of(65, 6)])


def test_refused_calls_change_nothing():
    """What draft_step refuses it refuses before it takes pages or writes."""
    d = started(ids_of(64, 7), [64, 64], 8)
    good = dict(temperature=1.0, u_accept=torch.zeros(8, device="cuda"), u_sample=torch.zeros(2, device="cuda"))
    x = ids_of(3, 8)
    before = [t.clone() for t in (*d.kc, *d.ic, d.pool.block_table, d.pool.n_free, d.seq_lens, d.tok)]
    for args, kw in (((x,), dict(good, u_accept=None)), ((x,), dict(good, u_sample=None)),
                     ((x,), dict(good, u_accept=torch.zeros(7, device="cuda"))),
                     ((x,), dict(good, draft_probs=torch.zeros(8, 999, device="cuda"))),
                     ((x,), dict(good, draft_probs=torch.zeros(8, 1000, device="cuda").half())),
                     ((x[:1],), {}),
                     ((x, torch.zeros(2, 3, dtype=torch.int32, device="cuda")), {})):
        with pytest.raises(ValueError):
            d.draft_step(*args, **kw)
    for a, b in zip(before, (*d.kc, *d.ic, d.pool.block_table, d.pool.n_free, d.seq_lens, d.tok)):
        assert torch.equal(a, b)
    d.draft_step(x, **good)


def test_ids_outside_the_vocabulary_are_no_drafts():
    """Rows may draft fewer tokens than others: ids outside the vocabulary are passed
    over, and the other tokens' logits are what they are without them."""
    ids, n = ids_of(60, 9), 6
    a, b = started(ids, [60, 60], 0), started(ids, [60, 60], 0)
    x = ids_of(n - 1, 10)
    y = x.clone()
    y[0, 3:] = torch.tensor([-1, 1000], device="cuda")
    y[1, 2:] = torch.tensor([-2 ** 40, 2 ** 40, -1001], device="cuda")
    _, la = a.draft_step(x)
    kept, lb = b.draft_step(y)
    assert torch.equal(la[0, :4], lb[0, :4]) and torch.equal(la[1, :3], lb[1, :3])
    root = torch.full((2, 1), 5, device="cuda")
    tokens = torch.cat([root, y], 1)
    verified(kept, lb, tokens, (tokens >= 0) & (tokens < 1000))
