"""Page-aware decoding (image pages) on a page pool: the page state belongs to
the physical pages, so it stays with its sequences when a page is missing, when
a table entry is unused, and when the pool's pages move."""
import numpy as np
import pytest
import torch

from ananta_ocr_b200 import pages as P
from ananta_ocr_b200.e2e_decoder import DashDecoder, DecoderConfig
from ananta_ocr_b200.unlimited_dash_ops import page_state as PS
from oracle import page_oracle as PO

pytestmark = pytest.mark.gpu

IMG, PG, PER, BS = 900, 901, 200, 64
CFG = DecoderConfig(hidden=256, heads=2, kv_heads=2, layers=3, vocab=1000, dense_ffn=512, moe_ffn=128, experts=8,
                    topk=2, shared=1, first_dense=3, block_size=BS, local_blocks=2, K=4, topm=4, slots=4)
PAGE_CFG = dict(image_token_id=IMG, page_token_id=PG, per_page_image_tokens=PER)


def doc_ids(batch, S, n_pages, seed):
    """Documents of n_pages image pages (a marker and image tokens) and text; row r's
    pages are a little shorter the larger r is, so that no two rows have the same
    page bounds."""
    ids = torch.randint(0, 800, (batch, S), generator=torch.Generator().manual_seed(seed))
    for r in range(batch):
        per = PER - 30 * r
        for p in range(n_pages):
            ids[r, p * per] = PG
            ids[r, p * per + 1:(p + 1) * per] = IMG
    return ids.cuda()


def make(batch, max_len=1100, pool=0, mask=False):
    return DashDecoder(CFG, batch=batch, max_len=max_len, device=torch.device("cuda"), seed=3, page_cfg=PAGE_CFG,
                       page_mask=mask, pool_pages=pool)


def slots_of_row(dec, r):
    """Physical slots of row r's tokens, in the tokens' order."""
    t = torch.arange(int(dec.seq_lens[r]), device="cuda")
    return dec.block_table[r, t // BS].long() * BS + t % BS


def state_of_row(dec, r):
    s = slots_of_row(dec, r)
    pages = s[::BS] // BS
    return [x[s] for x in dec.pst._slots] + [dec.pst._blk_lo[pages], dec.pst._blk_hi[pages]]


def test_a_slot_outside_the_state_is_left_out():
    """Tokens without a slot (a block without a page) and a previous token without
    one: nobody's state is written, the other requests' results are theirs."""
    rng = np.random.default_rng(1)
    bs, per, n_pages, R = 16, 24, 12, 3
    pst = PS.PageIsolationState(dict(image_token_id=IMG, page_token_id=PG, per_page_image_tokens=per), bs)
    bt = np.array([[0, 1, 2], [3, -1, -1], [4, 5, 6]], np.int32)
    lens = [40, 30, 33]
    for start in (0, 1):                                  # a prefill, then one more token each
        q_start = np.concatenate([[0], np.cumsum([1] * R if start else lens)])
        T = int(q_start[-1])
        sp = np.array(lens if start else [0] * R)
        ids = rng.choice([IMG, PG, 5], size=T, p=[.6, .1, .3])
        pos = np.concatenate([sp[r] + np.arange(q_start[r + 1] - q_start[r]) for r in range(R)])
        req = np.repeat(np.arange(R), np.diff(q_start))
        page = bt[req, pos // bs]
        slots = np.where(page < 0, page, page * bs + pos % bs)
        slots[(page < 0) & (pos % 2 == 1)] = n_pages * bs + 5      # behind the last slot: none either
        if not start:
            state = PO.new_slot_state(n_pages * bs)
            for t in pst_arrays(pst, n_pages * bs):
                t.zero_()
            pst._slot_img_page.fill_(-1)
        cu = torch.from_numpy(q_start).cuda()
        layout = PS.BatchLayout(num_tokens=T, num_reqs=R, q_start=cu, start_pos=torch.from_numpy(sp).cuda(),
                                block_table=torch.from_numpy(bt).cuda(), req_of_token=PS._req_of_token(cu, T))
        got = pst.step(torch.from_numpy(ids).cuda(), layout, torch.from_numpy(slots).cuda(), n_pages * bs)
        # the oracle on the requests that have their pages, and on the part of
        # the other that has its page
        for r in (0, 2):
            a, b = int(q_start[r]), int(q_start[r + 1])
            want = PO.page_state_step(state, ids[a:b], [0, b - a], sp[r:r + 1], bt[r:r + 1], slots[a:b], n_pages * bs,
                                      bs, per, IMG, PG)
            np.testing.assert_array_equal(got[a:b].cpu().numpy(), want)
        a = int(q_start[1])
        if not start:
            PO.page_state_step(state, ids[a:a + bs], [0, bs], sp[1:2], bt[1:2], slots[a:a + bs], n_pages * bs, bs, per,
                               IMG, PG)
        for name in ("img_page", "marker_cum", "img_run", "prompt_pages"):
            np.testing.assert_array_equal(getattr(pst, f"_slot_{name}").cpu().numpy(), state[name], err_msg=name)


def pst_arrays(pst, n):
    pst._ensure(n, torch.device("cuda"))
    return pst._slots


def test_a_row_without_a_page_leaves_the_others_page_state():
    """A pool that runs out under row 1: row 0 (whose first page is page 0) decodes
    as in a pool with pages enough, and keeps its page state."""
    S = 4 * BS                                            # four full pages each
    ids = doc_ids(2, S, 1, 2)
    rich, poor = make(2, pool=20), make(2, pool=9)
    for d in (rich, poor):
        d.prefill(d.embed[ids], token_ids=ids)
        d.tok.fill_(IMG)
    assert poor.block_table[0, 0].item() == 0
    for step in range(4):
        a, b = rich.decode_step(), poor.decode_step()
        assert torch.equal(a[0], b[0]), step
        for x, y in zip(state_of_row(rich, 0), state_of_row(poor, 0)):
            assert torch.equal(x, y), step
    assert poor.block_table[1, 4].item() == -1


def test_unused_table_entries_are_no_block():
    """The dense mask: an entry below 0 holds no page, whatever page 0 holds."""
    lo = torch.tensor([3, 1, -1], dtype=torch.int32).cuda()
    hi = torch.tensor([3, 2, -1], dtype=torch.int32).cuda()
    bt = torch.tensor([[1, 2, -1, -7], [1, 0, -1, -1]], dtype=torch.int32).cuda()
    q = torch.tensor([3, 3, 2], dtype=torch.int32).cuda()
    seq = torch.tensor([0, 1, 0], dtype=torch.int32).cuda()
    out = P.page_allow(q, lo, hi, width=4, rows=3, row_seq=seq, block_table=bt, desc_width=4, fallback=True)
    # row 0: no block of its sequence holds page 3: open; row 1: its block 1 does
    assert out.bool().tolist() == [[True] * 4, [False, True, False, False], [True, False, False, False]]


@pytest.mark.parametrize("mask", [False, True], ids=["domain", "mask"])
def test_pool_decodes_as_the_fixed_table(mask):
    """The same pages' contents under other ids, with unused table entries behind
    them: the same routes and logits, bit for bit."""
    ids = doc_ids(2, 1000, 4, 3)
    a, b = make(2, mask=mask), make(2, pool=40, mask=mask)
    assert torch.equal(a.prefill(a.embed[ids], token_ids=ids), b.prefill(b.embed[ids], token_ids=ids))
    assert torch.equal(a.last_q_page, b.last_q_page) and torch.equal(a.last_route[0], b.last_route[0])
    for i, t in enumerate((7, PG, 7, 8, IMG, IMG, 9)):
        for d in (a, b):
            d.tok.fill_(t)
        assert torch.equal(a.decode_step(), b.decode_step()), i
        assert torch.equal(a.oi, b.oi), i


@pytest.mark.parametrize("mask", [False, True], ids=["domain", "mask"])
def test_compaction_takes_the_page_state_along(mask):
    """Row 0 gives its pages back and the others' move down: rows 1 and 2 decode
    as without the move, over page boundaries too, and their state is where their
    pages are."""
    ids = doc_ids(3, 1000, 4, 5)
    a, b = make(3, pool=60, mask=mask), make(3, pool=60, mask=mask)
    for d in (a, b):
        d.prefill(d.embed[ids], token_ids=ids)
        d.pool.free(d.rows[:1])
        d.seq_lens[0] = 0
    moved = b.block_table.clone()
    b.compact()
    assert (moved[1:] != b.block_table[1:]).any()
    for r in (1, 2):
        for x, y in zip(state_of_row(a, r), state_of_row(b, r)):
            assert torch.equal(x, y), r
    assert b.pst._blk_lo.numel() >= 60
    lo, hi = b.pst.block_page_bounds(60)
    held = b.block_table[1:].flatten().long()
    held = held[held >= 0]
    assert torch.equal(b.pst._blk_lo[held], lo.int()[held]) and torch.equal(b.pst._blk_hi[held], hi.int()[held])
    for i, t in enumerate((7, PG, 7, IMG, IMG) + (9,) * 30):
        for d in (a, b):
            d.tok.fill_(t)
        x, y = a.decode_step(), b.decode_step()
        assert torch.equal(a.oi[1:], b.oi[1:]), i
        assert torch.equal(x[1:], y[1:]), i


def test_compaction_before_any_page_state():
    """A decoder that has seen no token ids yet has no state to move."""
    d = make(2, pool=40)
    d.prefill(d.embed[doc_ids(2, 200, 1, 6)])
    d.pool.free(d.rows[:1])
    d.compact()
    assert d.block_table[1].max().item() == 3
