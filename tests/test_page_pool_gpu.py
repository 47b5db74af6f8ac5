"""Page pool, page copies and commits on the GPU against the oracle (whole
numbers and bytes: equal)."""
import numpy as np
import pytest
import torch

from ananta_ocr_b200 import _lib as L
from ananta_ocr_b200 import drafts, ops
from ananta_ocr_b200.page_pool import CacheLayers, PagePool, copy_pages
from oracle import draft_oracle as DO

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def caches(P, bs, seed=0, layers=2):
    """Entries of several sizes: 16-byte, 8-, 4-, 2- and 1-byte accesses, token
    and page strides, one entry per page."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randint(-2 ** 31, 2 ** 31 - 1, s, generator=g, device="cuda", dtype=torch.int64).to(torch.int32)  # noqa: E731
    out = []
    for _ in range(layers):
        out += [r(P, bs, 2, 64).view(torch.bfloat16), r(P, bs, 32).view(torch.float32), r(P, bs, 2),
                r(P, bs, 3), r(P, bs, 3).to(torch.int16), r(P, bs, 5).to(torch.uint8), r(P, bs),
                r(P, 2, bs, 40)[:, 1], r(P, bs, 2, 8)[:, :, 1], r(P, bs).to(torch.uint8)]
    return out


def bits(t):
    return t.contiguous().view(torch.uint8)


def same_state(pool, want):
    got = (pool.ref, pool.free_list, pool.n_free, pool.block_table, pool.n_blocks)
    for name, a, b in zip(("ref", "free_list", "n_free", "block_table", "n_blocks"), got, want.arrays()):
        np.testing.assert_array_equal(a.cpu().numpy(), np.array(b, np.int32).reshape(a.shape), err_msg=name)


@pytest.mark.parametrize("pages,rows,width,bs", [(40, 8, 10, 16), (1000, 33, 70, 32), (7, 3, 4, 1), (3001, 9, 400, 16)])
def test_pool_against_the_oracle(pages, rows, width, bs):
    """Two hundred random requests, refused ones among them; after each the
    tables equal the oracle's, and a forked or moved page holds its source's
    bytes."""
    rng = np.random.default_rng(pages)
    pool, want = PagePool(pages, rows, width, bs), DO.Pool(pages, rows, width, bs)
    data = torch.arange(pages, device="cuda", dtype=torch.int32)[:, None].repeat(1, 4)
    model = data.cpu().numpy().copy()
    layers = CacheLayers([data])
    same_state(pool, want)
    for step in range(200):
        n = int(rng.integers(1, 6))
        some = rng.integers(-1, rows + 1, n).tolist()
        kind = step % 5
        if kind < 2:
            lens = rng.integers(-1, width * bs + 2, n).tolist() if kind else rng.integers(0, 3 * bs + 1, n).tolist()
            pool.reserve(i32(some), i32(lens))
            want.reserve(some, lens)
        elif kind == 2:
            src = rng.integers(0, rows, n).tolist()
            lens = [int(rng.integers(0, len(want.table[s]) * bs + 1)) for s in src]
            pool.fork(i32(src), i32(some), i32(lens), layers)
            for s, d in want.fork(src, some, lens):
                if d >= 0:
                    model[d] = model[s]
        elif kind == 3:
            keep = rng.integers(-1, 4, n).tolist()
            pool.free(i32(some), i32(keep))
            want.release(some, keep)
        elif step % 10 == 4:
            before = pool.block_table.clone()
            other = PagePool(pages, rows, width, bs)
            moved = pool.compact(layers, into=other)
            pairs = want.compact()
            assert moved.item() == len(pairs)
            assert torch.equal(pool.block_table, before)                 # the old tables are as they were
            for s, d in pairs:
                model[d] = model[s]
            pool = other
        else:
            pool.free(i32(some[:1]))
            want.release(some[:1], [0])
            pool.compact(layers)                                          # in place
            for s, d in want.compact():
                model[d] = model[s]
        same_state(pool, want)
        np.testing.assert_array_equal(data.cpu().numpy(), model)


def test_pool_errors_are_recorded():
    pool = PagePool(4, 3, 8, 16)
    err = ops.DeviceErrorWord("cuda")
    pool.reserve(i32([0, 1, 2]), i32([32, 48, 1]), err)                  # 2 + 3 pages asked for, 4 there
    assert err.read()[0] == L.DASH_DEV_NO_PAGE
    assert pool.n_blocks.tolist() == [2, 0, 0] and pool.n_free.item() == 2
    for call in (lambda: pool.reserve(i32([1, 1]), i32([16, 16]), err),     # the same row twice
                 lambda: pool.reserve(i32([7]), i32([16]), err), lambda: pool.reserve(i32([2]), i32([129]), err),
                 lambda: pool.free(i32([0, 0]), i32([1, 1]), err), lambda: pool.free(i32([-1]), None, err),
                 lambda: pool.fork(i32([0]), i32([0]), i32([3]), [pool.ref.view(4, 1)], err),
                 lambda: pool.fork(i32([0]), i32([2]), i32([100]), [pool.ref.view(4, 1)], err)):
        err.clear()
        call()
        assert err.read()[0] == L.DASH_DEV_BAD_ROW
    assert pool.n_blocks.tolist() == [1, 1, 0] and pool.n_free.item() == 2


def test_pool_largest_sizes():
    """The largest pool: 2^19 pages, 8192 rows."""
    P, R, W = 1 << 19, 8192, 64
    pool = PagePool(P, R, W, 16)
    rows = torch.arange(R, dtype=torch.int32, device="cuda")
    pool.reserve(rows, torch.full_like(rows, W * 16 - 3))
    assert pool.n_free.item() == 0 and (pool.n_blocks == W).all() and (pool.ref == 1).all()
    assert pool.block_table.flatten().sort().values.equal(torch.arange(P, dtype=torch.int32, device="cuda"))
    pool.free(rows[::2].contiguous(), torch.full_like(rows[::2], 10))
    held = R // 2 * (W + 10)
    assert pool.n_free.item() == P - held
    data = torch.arange(P, device="cuda", dtype=torch.int32).view(P, 1)
    table = pool.block_table.clone()
    moved = pool.compact([data])
    live = pool.block_table >= 0
    assert pool.block_table.max().item() == held - 1 and 0 < moved.item() <= P // 2
    assert torch.equal(data.flatten()[pool.block_table[live].long()], table[live])
    assert torch.equal(pool.free_list[:P - held], torch.arange(P - 1, held - 1, -1, dtype=torch.int32, device="cuda"))


def test_requests_whose_sum_passes_32_bits():
    """8192 rows that ask for 2^18 + 64 pages each: 2^31 pages and more in sum,
    none of which fits; a request that fits comes first."""
    W = 2 ** 18 + 64
    pool = PagePool(16, 8192, W, 1)
    err = ops.DeviceErrorWord("cuda")
    pool.reserve(i32([5]), i32([3]))
    rows = torch.arange(8192, dtype=torch.int32, device="cuda")
    pool.reserve(rows, torch.full_like(rows, W), err)
    assert err.read()[0] == L.DASH_DEV_NO_PAGE
    assert pool.n_free.item() == 13 and pool.n_blocks.sum().item() == 3 and pool.ref.sum().item() == 3
    assert pool.free_list.tolist() == list(range(15, 2, -1)) + [-1] * 3


def test_block_counts_outside_the_table():
    """Counts that no call of the pool leaves (below 0, past the table) stay inside it."""
    pool = PagePool(16, 4, 4, 1)
    pool.n_blocks.copy_(i32([-5, 9, 0, 0]))
    pool.reserve(i32([0]), i32([2]))
    assert pool.block_table.tolist()[0] == [0, 1, -1, -1] and pool.n_blocks[0].item() == 2
    t = torch.zeros(16, 1, 4, device="cuda")
    err = ops.DeviceErrorWord("cuda")
    pool.fork(i32([1]), i32([2]), i32([7]), [t], err)
    assert err.read()[0] == L.DASH_DEV_BAD_ROW and pool.n_blocks.tolist() == [2, 9, 0, 0]
    pool.free(i32([1, 0]))
    assert pool.n_free.item() == 16 and pool.n_blocks.tolist() == [0, 0, 0, 0]


def test_fork_copies_the_last_page_in_every_tensor():
    P, bs = 30, 16
    ts = caches(P, bs)
    pool = PagePool(P, 5, 6, bs)
    pool.reserve(i32([0, 1]), i32([40, 32]))
    before = [t.clone() for t in ts]
    pool.fork(i32([0, 1, 0]), i32([2, 3, 4]), i32([40, 32, 35]), ts)
    bt = pool.block_table.cpu().numpy()
    assert (bt[2, :2] == bt[0, :2]).all() and (bt[3, :2] == bt[1, :2]).all() and bt[2, 2] != bt[0, 2]
    assert pool.n_blocks.tolist() == [3, 2, 3, 2, 3] and pool.ref[bt[0, 0]].item() == 3
    new = {int(bt[2, 2]), int(bt[4, 2])}
    assert len(new) == 2
    for t, b in zip(ts, before):
        for p in range(P):
            assert torch.equal(bits(t[p]), bits(b[int(bt[0, 2])] if p in new else b[p]))


@pytest.mark.parametrize("n", [1, 3, 64, 1500])
def test_copy_pages(n):
    P, bs = 4000, 4
    rng = np.random.default_rng(n)
    ts = caches(P, bs, layers=1)
    ids = rng.permutation(P)[:2 * n]
    src, dst = ids[:n].copy(), ids[n:].copy()
    if n > 2:
        src[1] = src[0]                                       # one source, two targets
        src[2] = -1
    before = [t.clone() for t in ts]
    copy_pages(ts, i32(src.tolist()), i32(dst.tolist()))
    for t, b in zip(ts, before):
        for s, d in zip(src, dst):
            if s >= 0:
                b[d] = b[s]
        assert torch.equal(bits(t), bits(b))


def test_copy_pages_conflicts():
    """A destination that is read or written by another pair is left out."""
    ts = [torch.arange(10, device="cuda", dtype=torch.int32).view(10, 1)]
    err = ops.DeviceErrorWord("cuda")
    copy_pages(ts, i32([0, 1, 2, 3, 4, 9]), i32([5, 5, 3, 6, 4, 8]), err)
    # 0->5 and 1->5 share a target; 2->3 writes a source; 3->6 reads 3, a target; 4->4 is nothing
    assert err.read()[0] == L.DASH_DEV_BAD_ROW
    assert ts[0].flatten().tolist() == [0, 1, 2, 3, 4, 5, 6, 7, 9, 9]
    err.clear()
    copy_pages(ts, i32([0, 10, 1]), i32([7, 2, 11]), err)
    assert err.read()[0] == L.DASH_DEV_BAD_ROW and ts[0].flatten().tolist() == [0, 1, 2, 3, 4, 5, 6, 0, 9, 9]


def test_more_tensors_than_one_launch_takes():
    P = 12
    ts = [torch.full((P, 2, 4), float(i), device="cuda") + torch.arange(P, device="cuda")[:, None, None] for i in range(150)]
    copy_pages(ts, i32([1, 2]), i32([8, 9]))
    for i, t in enumerate(ts):
        assert t[8, 0, 0].item() == i + 1 and t[9, 1, 3].item() == i + 2 and t[10, 0, 0].item() == i + 10


def make_commit(seed, R, n, bs, P):
    rng = np.random.default_rng(seed)
    ctx = rng.integers(0, 3 * bs, R)
    W = -(-(3 * bs + n) // bs)
    bt = rng.permutation(P)[:R * W].reshape(R, W).astype(np.int32)
    path, acc = np.full((R, n), -1, np.int32), np.zeros(R, np.int32)
    path[:, 0] = 0
    for r in range(R):
        k = int(rng.integers(0, n))
        path[r, 1:k + 1] = np.sort(rng.permutation(n - 1)[:k]) + 1
        acc[r] = k
    return ctx.astype(np.int32), bt, path, acc


def move(model, ctx, bt, path, acc, bs):
    for m in model:
        old = m.clone()
        for r in range(len(ctx)):
            for i in range(1, acc[r] + 1):
                a, b = ctx[r] + path[r, i], ctx[r] + i
                m[bt[r, b // bs], b % bs] = old[bt[r, a // bs], a % bs]


@pytest.mark.parametrize("R,n,bs", [(1, 2, 16), (5, 17, 32), (3, 64, 16), (2, 256, 7), (4, 9, 1)])
def test_commit(R, n, bs):
    ctx, bt, path, acc = make_commit(R, R, n, bs, 400)
    ts = caches(400, bs)
    want = [t.clone() for t in ts]
    drafts.commit_drafts(ts, i32(path.tolist()), i32(acc.tolist()), i32(ctx.tolist()), i32(bt.tolist()))
    move(want, ctx, bt, path, acc, bs)
    for t, w in zip(ts, want):
        assert torch.equal(bits(t), bits(w))


def test_commit_stops_at_a_bad_path():
    bs, P = 16, 8
    t = torch.arange(P * bs, device="cuda", dtype=torch.int32).view(P, bs)
    err = ops.DeviceErrorWord("cuda")
    bt = i32([[0, 1, 2]])
    drafts.commit_drafts([t], i32([[0, 2, 5, 5, 6]]), i32([4]), i32([3]), bt, err)
    assert err.read()[0] == L.DASH_DEV_BAD_TREE
    assert t[0, 3:9].tolist() == [3, 5, 5, 6, 7, 8]       # 2 -> 1 ran; there is no token 5 of 5
    err.clear()
    t.copy_(torch.arange(P * bs, device="cuda", dtype=torch.int32).view(P, bs))
    drafts.commit_drafts([t], i32([[0, 2, 5, 5, 6, -1, -1]]), i32([4]), i32([3]), bt, err)
    assert err.read()[0] == L.DASH_DEV_BAD_TREE
    assert t[0, 3:9].tolist() == [3, 5, 8, 6, 7, 8]       # 2 -> 1 and 5 -> 2 ran, the second 5 not
    err.clear()
    drafts.commit_drafts([t], i32([[0, 2, -1]]), i32([1]), i32([46]), bt, err)     # token 48 has no page
    assert err.read()[0] == L.DASH_DEV_BAD_PAGE and t[2, 15].item() == 47
    with pytest.raises(ValueError, match="one entry per token"):
        drafts.commit_drafts([t, torch.zeros(P, 1, 4, device="cuda")], i32([[0]]), i32([0]), i32([0]), bt)
    with pytest.raises(ValueError, match="path"):
        drafts.commit_drafts([t], i32([[0]]).long(), i32([0]), i32([0]), bt)


def test_commit_behind_the_last_token_of_32_bits():
    t = torch.arange(64, device="cuda", dtype=torch.float32).view(4, 4, 4)
    want, err = t.clone(), ops.DeviceErrorWord("cuda")
    drafts.commit_drafts([t], i32([[0, 2, 3, -1]]), i32([2]), i32([2 ** 31 - 2]), i32([[0, 1, 2, 3]]), err)
    assert err.read()[0] == L.DASH_DEV_BAD_TREE and torch.equal(t, want)


def test_kbar_of_a_block_without_a_page():
    """A plan entry below 0 writes no row (row -1 lies inside the tensors here)."""
    cache, kbar = torch.ones(5, 16, 128, device="cuda")[1:], torch.zeros(5, 128, device="cuda")
    ops.kbar_pool_paged(cache, torch.tensor([2, -1], device="cuda"), i32([16, 16]), None, kbar[1:])
    assert (kbar[[0, 1, 2, 4]] == 0).all() and (kbar[3] != 0).any()


def test_graph_of_a_pool_step():
    """free + fork + compact captured once and replayed: the tables of three
    eager steps."""
    def build():
        pool = PagePool(64, 6, 8, 16)
        pool.reserve(i32([0, 1, 2, 3]), i32([100, 40, 90, 70]))
        pool.free(i32([1]))
        return pool, [torch.arange(64 * 16, device="cuda", dtype=torch.int32).view(64, 16)]

    def step(pool, data, args):
        pool.free(args[1])
        pool.fork(args[0], args[1], args[2], data)
        pool.compact(data)

    args = (i32([0, 2]), i32([4, 5]), i32([90, 33]))
    (a, da), (b, db) = build(), build()
    for _ in range(4):
        step(a, da, args)
    step(b, db, args)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(b, db, args)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    for x, y in zip((a.ref, a.free_list, a.n_free, a.block_table, a.n_blocks, da[0]),
                    (b.ref, b.free_list, b.n_free, b.block_table, b.n_blocks, db[0])):
        assert torch.equal(x, y)


def test_wrong_tensors_raise():
    pool = PagePool(8, 2, 4, 16)
    with pytest.raises(ValueError, match="contiguous"):
        CacheLayers([torch.zeros(8, 16, 4, 4, device="cuda").transpose(2, 3)])
    with pytest.raises(ValueError, match="pages"):
        pool.compact([torch.zeros(7, 16, device="cuda")])
    with pytest.raises(ValueError, match="lens"):
        pool.reserve(i32([0]), i32([1, 2]))
    with pytest.raises(ValueError, match="block size"):
        pool.compact([torch.zeros(8, 16, device="cuda")], into=PagePool(8, 2, 4, 32))
    with pytest.raises(L.DashError, match="sizes"):
        pool.compact([torch.zeros(8, 16, device="cuda")], into=PagePool(9, 2, 4, 16))
