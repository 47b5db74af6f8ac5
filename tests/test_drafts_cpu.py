"""Speculative decoding, what needs no GPU: refusals of the C ABI and of the
Python entry points, and the oracle's own properties (the kept tokens follow
the target's distribution, a tree of chains equals its chains)."""
import ctypes as C

import numpy as np
import pytest
import torch

from ananta_ocr_b200 import _lib as L
from oracle import draft_oracle as DO


def status(fn, args):
    return getattr(L.load(), fn)(C.byref(args), None)


def refused(fn, args, code, words):
    assert status(fn, args) == code
    assert words in L.last_error(), L.last_error()


def tree_args(**kw):
    a = L.DashTreeAttnArgs()
    a.seqs.n_seq, a.seqs.q_len_fixed, a.seqs.max_q_len, a.seqs.q_start = 2, 16, 8, 1 << 16
    a.kv.k = a.kv.v = 1 << 20
    a.kv.dtype, a.kv.n_kv_heads, a.kv.head_dim = L.DTYPE_BF16, 2, 128
    a.kv.stride_seq, a.kv.stride_tok, a.kv.stride_head = 64 * 256, 256, 128
    a.kv.block_table, a.kv.bt_stride, a.kv.num_pages = 1 << 18, 8, 32
    a.qo.q = a.qo.out = 1 << 22
    a.qo.n_heads, a.qo.q_stride_tok, a.qo.q_stride_head = 4, 512, 128
    a.qo.o_stride_tok, a.qo.o_stride_head = 512, 128
    a.routes.n_index_heads = 1
    a.ctx_len, a.row_pos, a.mask = 1 << 17, 1 << 17, 1 << 17
    a.mask_words = a.mask_stride = 1
    a.bt_width, a.block_size, a.local_window, a.scale = 8, 64, 256, 0.1
    for k, v in kw.items():
        obj = a
        *path, last = k.split("__")
        for x in path:
            obj = getattr(obj, x)
        setattr(obj, last, v)
    return a


@pytest.mark.parametrize("change,code,words", [
    (dict(seqs__max_q_len=257, mask_words=9, mask_stride=9), L.DASH_ERR_UNSUPPORTED, "drafted tokens"),
    (dict(seqs__max_q_len=0), L.DASH_ERR_INVALID, "max_nodes"),
    (dict(seqs__n_seq=-1), L.DASH_ERR_INVALID, "negative"),
    (dict(seqs__max_q_len=33), L.DASH_ERR_INVALID, "mask"),
    (dict(mask_stride=0), L.DASH_ERR_INVALID, "mask"),
    (dict(kv__dtype=L.DTYPE_F32), L.DASH_ERR_UNSUPPORTED, "dtype"),
    (dict(kv__head_dim=64), L.DASH_ERR_UNSUPPORTED, "head_dim"),
    (dict(kv__n_kv_heads=3), L.DASH_ERR_INVALID, "multiple"),
    (dict(kv__block_table=None), L.DASH_ERR_UNSUPPORTED, "paged"),
    (dict(kv__num_pages=0), L.DASH_ERR_INVALID, "num_pages"),
    (dict(kv__k=(1 << 20) + 8), L.DASH_ERR_INVALID, "aligned"),
    (dict(kv__stride_tok=257), L.DASH_ERR_INVALID, "strides"),
    (dict(qo__n_heads=0), L.DASH_ERR_INVALID, "n_heads"),
    (dict(qo__q=None), L.DASH_ERR_INVALID, "null q"),
    (dict(qo__q_stride_head=127), L.DASH_ERR_INVALID, "strides"),
    (dict(routes__K=4), L.DASH_ERR_INVALID, "route idx"),
    (dict(routes__K=257, routes__idx=16), L.DASH_ERR_UNSUPPORTED, "K 257"),
    (dict(routes__n_index_heads=3), L.DASH_ERR_INVALID, "n_index_heads"),
    (dict(ctx_len=None), L.DASH_ERR_INVALID, "null q_start"),
    (dict(row_pos=None), L.DASH_ERR_INVALID, "null q_start"),
    (dict(mask=None), L.DASH_ERR_INVALID, "null q_start"),
    (dict(bt_width=0), L.DASH_ERR_INVALID, "bt_width"),
    (dict(block_size=0), L.DASH_ERR_INVALID, "block_size"),
    (dict(local_window=-1), L.DASH_ERR_INVALID, "local_window"),
    (dict(num_splits=17), L.DASH_ERR_INVALID, "num_splits"),
])
def test_tree_attn_refuses(change, code, words):
    refused("dash_tree_attn", tree_args(**change), code, words)


def test_empty_calls_launch_nothing():
    n = L.launches()
    assert status("dash_tree_attn", tree_args(seqs__n_seq=0)) == L.DASH_OK
    assert status("dash_tree_attn", tree_args(seqs__q_len_fixed=0)) == L.DASH_OK
    p = L.DashTreePlanArgs()
    p.max_nodes = 4
    assert status("dash_tree_plan", p) == L.DASH_OK
    v = L.DashVerifyArgs()
    v.max_nodes = 4
    assert status("dash_draft_verify", v) == L.DASH_OK
    c = pages_args()
    c.n = 0
    for fn in ("dash_pages_reserve", "dash_pages_free", "dash_pages_fork"):
        assert status(fn, c) == L.DASH_OK
    assert L.launches() == n


def test_plan_refuses():
    a = L.DashTreePlanArgs()
    a.n_seq, a.rows, a.max_nodes = 1, 4, 4
    refused("dash_tree_plan", a, L.DASH_ERR_INVALID, "null q_start")
    a.q_start = a.ctx_len = 16
    a.mask, a.mask_words = 16, 0
    refused("dash_tree_plan", a, L.DASH_ERR_INVALID, "mask_words")
    a.mask_words, a.slots = 1, 16
    refused("dash_tree_plan", a, L.DASH_ERR_INVALID, "slots need")


def verify_args():
    a = L.DashVerifyArgs()
    a.n_seq, a.rows, a.max_nodes, a.vocab = 1, 4, 4, 100
    a.tokens = a.q_start = a.target = a.draft = a.u_accept = a.u_sample = 1 << 16
    a.target_stride = a.draft_stride = 100
    a.n_accept = a.path = a.next_token = a.out_tokens = 1 << 16
    return a


@pytest.mark.parametrize("change,code,words", [
    (dict(mode=3), L.DASH_ERR_INVALID, "mode"),
    (dict(dtype=7), L.DASH_ERR_UNSUPPORTED, "dtype"),
    (dict(vocab=0), L.DASH_ERR_INVALID, "vocab"),
    (dict(q_start=None), L.DASH_ERR_INVALID, "null q_start"),
    (dict(next_token=None), L.DASH_ERR_INVALID, "output"),
    (dict(target=None), L.DASH_ERR_INVALID, "null tokens"),
    (dict(target_stride=99), L.DASH_ERR_INVALID, "shorter"),
    (dict(draft=None), L.DASH_ERR_INVALID, "draft"),
    (dict(draft_stride=99), L.DASH_ERR_INVALID, "draft"),
    (dict(mode=1, u_accept=None), L.DASH_ERR_INVALID, "u_accept"),
    (dict(mode=1, u_sample=None), L.DASH_ERR_INVALID, "u_accept"),
    (dict(max_nodes=300), L.DASH_ERR_UNSUPPORTED, "drafted tokens"),
])
def test_verify_refuses(change, code, words):
    a = verify_args()
    for k, v in change.items():
        setattr(a, k, v)
    refused("dash_draft_verify", a, code, words)


def tensors(**kw):
    t = (L.DashCacheTensor * 1)()
    t[0].base, t[0].page_stride, t[0].tok_stride, t[0].tok_bytes, t[0].page_toks = 1 << 20, 4096, 256, 256, 16
    for k, v in kw.items():
        setattr(t[0], k, v)
    return t


def commit_args(t):
    a = L.DashCommitArgs()
    a.tensors, a.n_tensors, a.n_seq, a.max_nodes, a.block_size = C.addressof(t), 1, 2, 4, 16
    a.bt_width = a.bt_stride = 8
    a.num_pages, a.path_stride = 32, 4
    a.path = a.n_accept = a.ctx_len = a.block_table = 1 << 16
    return a


def test_commit_and_copy_refuse():
    for kw, words in ((dict(base=None), "null base"), (dict(tok_bytes=0), "overlap"), (dict(tok_stride=255), "overlap"),
                      (dict(page_stride=4095), "overlap"), (dict(page_toks=8), "tokens per page")):
        t = tensors(**kw)
        refused("dash_draft_commit", commit_args(t), L.DASH_ERR_INVALID, words)
    t = tensors()
    for k, v, words in (("path_stride", 3, "overlap"), ("bt_stride", 7, "overlap"), ("path", None, "null"),
                        ("num_pages", 0, "num_pages"), ("block_size", 0, "block_size")):
        a = commit_args(t)
        setattr(a, k, v)
        refused("dash_draft_commit", a, L.DASH_ERR_INVALID, words)
    a = L.DashPagesCopyArgs()
    a.tensors, a.n_tensors, a.n, a.num_pages, a.check = C.addressof(t), 1, 3, 32, 1
    refused("dash_pages_copy", a, L.DASH_ERR_INVALID, "null src")
    a.src = a.dst = 1 << 16
    refused("dash_pages_copy", a, L.DASH_ERR_INVALID, "list")
    a.list, a.num_pages = 1 << 16, 1 << 20
    refused("dash_pages_copy", a, L.DASH_ERR_UNSUPPORTED, "2^19")
    a.n = -1
    refused("dash_pages_copy", a, L.DASH_ERR_INVALID, "n < 0")
    a.n, a.num_pages = 1, 0
    refused("dash_pages_copy", a, L.DASH_ERR_INVALID, "num_pages")


def pages_args():
    a = L.DashPagesArgs()
    for p in (a.pool, a.into):
        p.ref = p.free_list = p.n_free = p.block_table = p.n_blocks = 1 << 16
        p.bt_stride = p.bt_width = 8
        p.num_pages, p.max_rows, p.block_size = 32, 4, 16
    a.rows = a.src = a.lens = a.copy_src = a.copy_dst = a.n_moves = a.new_id = 1 << 16
    a.n = 2
    return a


@pytest.mark.parametrize("change,code,words", [
    (dict(pool__ref=None), L.DASH_ERR_INVALID, "null pool"),
    (dict(pool__num_pages=(1 << 19) + 1), L.DASH_ERR_UNSUPPORTED, "2^19"),
    (dict(pool__max_rows=8193), L.DASH_ERR_UNSUPPORTED, "max_rows"),
    (dict(pool__bt_stride=7), L.DASH_ERR_INVALID, "overlap"),
    (dict(n=-1), L.DASH_ERR_INVALID, "n < 0"),
    (dict(rows=None), L.DASH_ERR_INVALID, "null rows"),
])
def test_pool_refuses(change, code, words):
    for fn in ("dash_pages_reserve", "dash_pages_free", "dash_pages_fork"):
        a = pages_args()
        for k, v in change.items():
            obj = a.pool if k.startswith("pool__") else a
            setattr(obj, k.split("__")[-1], v)
        refused(fn, a, code, words)
    a = pages_args()
    a.lens = None
    refused("dash_pages_reserve", a, L.DASH_ERR_INVALID, "lens")
    refused("dash_pages_fork", a, L.DASH_ERR_INVALID, "lens")
    a = pages_args()
    a.copy_dst = None
    refused("dash_pages_fork", a, L.DASH_ERR_INVALID, "copy_dst")
    refused("dash_pages_compact", a, L.DASH_ERR_INVALID, "copy_src")
    a = pages_args()
    a.into.num_pages = 31
    refused("dash_pages_compact", a, L.DASH_ERR_INVALID, "sizes")


def test_python_entry_points_need_cuda():
    from ananta_ocr_b200 import drafts, page_pool
    x = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        drafts.tree_plan(None, x, x, rows=4, max_nodes=4)
    with pytest.raises(RuntimeError, match="CUDA"):
        drafts.verify_drafts(x.long(), None, x, torch.zeros(4, 9), max_nodes=4, greedy=True)
    with pytest.raises(RuntimeError, match="CUDA"):
        page_pool.CacheLayers([torch.zeros(4, 16, 8)])
    with pytest.raises(RuntimeError, match="CUDA"):
        page_pool.PagePool(8, 2, 4, 16, device="cpu")
    with pytest.raises(ValueError, match="at least one"):
        page_pool.CacheLayers([])


# ---------------------------------------------------------------------------
# the oracle itself
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("mode", ["drawn", "certain"])
def test_kept_tokens_follow_the_target(mode):
    """The first new token of a step (a kept child of the root, or the token
    drawn at the root) is distributed as the target says, whatever the drafts:
    20,000 steps, every frequency within 5 standard deviations."""
    rng = np.random.default_rng(0)
    V, N = 5, 20000
    p, q = rng.dirichlet(np.ones(V)), rng.dirichlet(np.ones(V) * 0.7)
    # root, three children of the root
    parents, starts = [-1, 0, 0, 0], [0, 4]
    target = np.stack([p] + [rng.dirichlet(np.ones(V)) for _ in range(3)])
    draft = np.stack([q] * 4)
    count = np.zeros(V)
    for _ in range(N):
        kids = rng.choice(V, 3, p=q) if mode == "drawn" else rng.permutation(V)[:3]
        toks = np.concatenate([[0], kids])
        _, _, _, out = DO.verify(toks, parents, starts, target, draft if mode == "drawn" else None,
                                 rng.random(4), rng.random(1), mode, 4)
        count[out[0, 0]] += 1
    sd = np.sqrt(p * (1 - p) / N)
    assert (np.abs(count / N - p) < 5 * sd).all(), (count / N, p)


def test_one_certain_draft_is_rejection_sampling():
    p = np.array([[0.2, 0.5, 0.3], [0.1, 0.1, 0.8]])
    for u, want in ((0.49, 1), (0.51, 0)):
        acc, path, nxt, toks = DO.verify([9, 1], None, [0, 2], p, None, [0.0, u], [0.0], "certain", 2)
        assert acc[0] == want
        # rejected: token 1 has no mass left, u = 0 picks token 0
        assert nxt[0] == 0
    # a rejected draft: cumulative 0.2, 0.2, 0.5 of 0.5
    assert DO.verify([9, 1], None, [0, 2], p, None, [0.0, 0.9], [0.41], "certain", 2)[2][0] == 2


def test_residual_after_k_rejections():
    """R_k = max(p - c_k q, 0) / W_k with c_(k+1) = c_k + W_k, the form that the
    kernel evaluates, equals the repeated normalised subtraction."""
    rng = np.random.default_rng(1)
    p, q = rng.dirichlet(np.ones(50)), rng.dirichlet(np.ones(50))
    r, c, W = p.copy(), 0.0, 1.0
    for _ in range(4):
        r = np.maximum(r - q, 0)
        r /= r.sum()
        c += W
        W = np.maximum(p - c * q, 0).sum()
        np.testing.assert_allclose(np.maximum(p - c * q, 0) / W, r, atol=1e-13)


def test_pool_oracle_keeps_every_page_once():
    rng = np.random.default_rng(2)
    P = DO.Pool(40, 8, 10, 16)
    for _ in range(200):
        k = rng.integers(0, 4)
        rows = rng.integers(0, 8, rng.integers(1, 4)).tolist()
        if k == 0:
            P.reserve(rows, rng.integers(0, 150, len(rows)).tolist())
        elif k == 1:
            P.release(rows, rng.integers(0, 5, len(rows)).tolist())
        elif k == 2:
            P.fork(rng.integers(0, 8, len(rows)).tolist(), rows, rng.integers(0, 100, len(rows)).tolist())
        else:
            P.compact()
        held = [0] * 40
        for t in P.table:
            for p in t:
                held[p] += 1
        assert held == P.ref
        assert sorted(P.free) == [p for p in range(40) if P.ref[p] == 0]


def test_packer_equals_setting_the_fields():
    """Arguments packed at once hold what setting every field gives."""

    def fill(c, values):
        for name, t in type(c)._fields_:
            if issubclass(t, C.Structure):
                fill(getattr(c, name), values)
            else:
                setattr(c, name, next(values))

    for cls in (L.DashTreeAttnArgs, L.DashVerifyArgs, L.DashCommitArgs, L.DashPagesCopyArgs):
        want, n = cls(), 0
        fill(want, iter(range(1, 100)))
        def count(c):                                      # noqa: E306
            return sum(count(t) if issubclass(t, C.Structure) else 1 for _, t in c._fields_)
        n = count(cls)
        assert bytes(L.packer(cls)(*range(1, n + 1))) == bytes(want), cls.__name__
    want = L.DashPagesArgs()
    fill(want, iter(range(1, 100)))
    rest = L.packer(L.DashPagesArgs, 2)(*range(21, 32))
    assert bytes(want.pool) + bytes(want.into) + rest == bytes(want)
