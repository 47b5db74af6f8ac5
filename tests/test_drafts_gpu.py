"""Draft-tree attention, verification and commit on the GPU against the 64-bit
oracle."""
import numpy as np
import pytest
import torch

from ananta_ocr_b200 import _lib as L
from ananta_ocr_b200 import drafts, ops
from ananta_ocr_b200.unlimited_dash_ops.attend_triton import dash_sparse_attn_decode
from oracle import draft_oracle as DO
from draft_testutil import attention_tolerance, make_tree, tree_parents

pytestmark = pytest.mark.gpu
SCALE = 1.0 / np.sqrt(128)


def attend(t, *, splits=0, out=None, lse=True, err=None, **over):
    d = {k: over[k] if k in over else v.cuda() for k, v in t.items() if isinstance(v, torch.Tensor)}
    rows = d["q"].shape[0]
    HI = d["t_idx"].shape[0]
    ex = (lambda x: x.repeat_interleave(t["Hkv"] // HI, 0)) if HI > 1 else (lambda x: x.expand(t["Hkv"], -1, -1))
    out = torch.full((rows, t["H"], 128), 7.0, dtype=t["dtype"], device="cuda") if out is None else out
    z = torch.full((rows, t["H"]), 7.0, device="cuda") if lse else None
    drafts.dash_sparse_attn_tree(
        d["q"], d["kc"], d["vc"], ex(d["t_idx"]), ex(d["t_bias"]), d["t_bt"], d["t_cu"], d["t_ctx"], d["t_pos"],
        d["t_mask"], max(t["nodes"] + [1]), t["Hkv"], SCALE, out, local_blocks=t["local_blocks"],
        sparse_block_size=t["bs"], num_splits=splits, lse=z, device_error=err)
    return out, z


def check(t, out, z):
    n = t["rows"]
    ref, lse, A = DO.tree_attend(t["q"][:t["rows"]].float().numpy(), t["kc"].float().numpy(), t["vc"].float().numpy(),
                                 t["idx"], t["bias"], t["bt"], t["starts"], t["ctx"], t["pos"], t["vis"], t["bs"],
                                 t["window"], SCALE)
    got = out.float().cpu().numpy()
    off = np.abs(got[:n] - ref) - attention_tolerance(ref, A, t["dtype"])
    assert not np.isnan(got[:n]).any() and off.max() <= 0, f"{off.max()} over the tolerance"
    assert (got[n:] == 7.0).all(), "padding rows were written"
    if z is not None:
        zz = z.cpu().numpy()
        none = np.isneginf(lse)
        assert (np.isneginf(zz[:n]) == none).all()
        # the logits' error (8e-5, see attention_tolerance) and a log of a sum
        assert (np.abs(zz[:n] - lse)[~none] <= 1e-4 + 1e-6 * np.abs(lse[~none])).all()
        assert (zz[n:] == 7.0).all()


CASES = {
    # nodes, ctx, heads, kv heads, block, window blocks, K, type, branch
    "chain": ([5, 1, 8], [300, 64, 1000], 2, 2, 64, 2, 4, "bf16", 1),
    "decoder": ([17, 3, 9], [700, 33, 400], 2, 2, 32, 4, 12, "bf16", 3),
    "short": ([1, 4, 2, 3], [0, 0, 1, 63], 2, 1, 64, 1, 4, "bf16", 2),
    "empty_sequences": ([0, 3, 0, 1, 0], [5, 200, 0, 129, 9], 2, 2, 64, 1, 4, "fp16", 2),
    "gqa": ([33, 7], [900, 257], 8, 2, 128, 1, 5, "bf16", 0),
    "gqa5_blocks16": ([13, 40], [210, 500], 10, 2, 16, 2, 16, "fp16", 4),
    "wide": ([64, 100], [500, 900], 2, 2, 64, 1, 8, "bf16", 4),
    "most_nodes": ([256, 129], [100, 640], 2, 2, 32, 2, 6, "bf16", 3),
    "one_head_for_all": ([20, 11], [333, 90], 16, 1, 64, 2, 4, "fp16", 2),
    "no_routes": ([6, 9], [500, 40], 2, 2, 64, 2, 0, "bf16", 2),
    "no_window": ([6, 9], [500, 40], 2, 2, 64, 0, 4, "bf16", 2),
    "window_over_all": ([6, 9], [500, 777], 2, 2, 32, 40, 3, "bf16", 2),
    "blocks256": ([12, 5], [1500, 255], 2, 1, 256, 1, 3, "fp16", 2),
    "blocks192": ([12, 5], [1500, 191], 2, 1, 192, 1, 3, "bf16", 2),
    "odd_blocks48": ([12, 5], [700, 47], 4, 2, 48, 2, 6, "bf16", 2),
    "odd_blocks7": ([4, 6], [100, 6], 2, 2, 7, 2, 6, "fp16", 2),
    "many_blocks": ([9, 4], [9000, 5000], 1, 1, 16, 1, 200, "bf16", 2),
}


@pytest.mark.parametrize("poison", [False, True], ids=["", "poison"])
@pytest.mark.parametrize("name", sorted(CASES))
def test_tree_attention(name, poison):
    nodes, ctx, H, Hkv, bs, win, K, dt, branch = CASES[name]
    t = make_tree(11 + len(name), nodes, ctx, H=H, Hkv=Hkv, bs=bs, window=win, K=K, dtype=dt, branch=branch,
                  pad_rows=3, poison=poison)
    check(t, *attend(t))


@pytest.mark.parametrize("splits", [*range(1, 9), 11, 16])
@pytest.mark.parametrize("name", ["decoder", "gqa", "short"])
def test_every_split_count(name, splits):
    nodes, ctx, H, Hkv, bs, win, K, dt, branch = CASES[name]
    t = make_tree(5, nodes, ctx, H=H, Hkv=Hkv, bs=bs, window=win, K=K, dtype=dt, branch=branch, pad_rows=1)
    a = attend(t, splits=splits)
    check(t, *a)
    b = attend(t, splits=splits)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("last", [7, 0], ids=["", "nothing_in_the_second"])
def test_more_units_than_the_gpu_holds(last):
    """320 units: 296 of one CTA each, the others in a second launch (whose
    sequences may draft nothing), eager and captured, with work in front of it
    and behind it in the stream."""
    nodes = [3, 1, 0, 5] * 9 + [7] + [last] * 3
    t = make_tree(21, nodes, [1100 + 17 * i for i in range(40)], H=8, Hkv=8, bs=64, window=2, K=16)
    d = {k: v.cuda() for k, v in t.items() if isinstance(v, torch.Tensor)}
    L.launches(reset=True)
    out, z = attend(t, **d)
    assert L.launches() == 2
    check(t, out, z)
    q, o = torch.empty_like(d["q"]), torch.empty_like(out)
    sums = torch.empty_like(out, dtype=torch.float32)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for scale in (0.5, 1.0):                       # the first result must not be what is left
            q.copy_(d["q"] * scale)
            attend(t, out=o, lse=False, **{**d, "q": q})
            sums.copy_(o)
            o.zero_()
    for _ in range(5):
        g.replay()
        torch.cuda.synchronize()
        n = t["rows"]
        assert torch.equal(sums[:n], out[:n].float()) and (o == 0).all()


def test_repeated_ids_and_index_heads():
    """The first of repeated ids counts; two router heads pick their own blocks."""
    t = make_tree(3, [9, 14], [800, 600], H=4, Hkv=2, bs=64, window=2, K=6, index_heads=2, dup=True, pad_rows=2)
    check(t, *attend(t))
    t = make_tree(4, [70], [2000], H=4, Hkv=4, bs=32, window=2, K=40, index_heads=4, dup=True)
    check(t, *attend(t))


def test_repeated_ids_with_biases_near_log4():
    """The first of repeated ids counts whatever its bias is: in units of log2
    these lie around 2.0, bit by bit from 16 units in the last place below to
    above (a table entry that marked slots by such values would be taken twice)."""
    t = make_tree(12, [32], [3000], H=1, Hkv=1, bs=64, window=1, K=12)
    near = np.float32(np.log(4.0)).view(np.int32)
    t["bias"][0] = -5.0
    for r in range(32):
        t["idx"][0, r, 1:] = t["idx"][0, r, 0]
        t["bias"][0, r, 0] = (near - 24 + r).astype(np.int32).view(np.float32)
    t["t_bias"], t["t_idx"] = torch.from_numpy(t["bias"]), torch.from_numpy(t["idx"])
    check(t, *attend(t))


def test_large_logits():
    """Rows whose logits span hundreds: the running maximum has to move."""
    t = make_tree(6, [16, 5], [900, 700], H=4, Hkv=2, bs=64, window=2, K=8, scale_q=30.0)
    out, z = attend(t)
    # logits 30 times larger: their fp32 error (8e-5 at ordinary sizes) grows
    # with them, and so does the weights' relative error
    ref, lse, A = DO.tree_attend(t["q"][:t["rows"]].float().numpy(), t["kc"].float().numpy(), t["vc"].float().numpy(), t["idx"],
                                 t["bias"], t["bt"], t["starts"], t["ctx"], t["pos"], t["vis"], t["bs"], t["window"],
                                 SCALE)
    tol = attention_tolerance(ref, A, t["dtype"]) + 30 * 1e-4 * A
    assert (np.abs(out.float().cpu().numpy() - ref) <= tol).all()
    assert (np.abs(z.cpu().numpy() - lse) <= 30 * 1e-4 + 1e-6 * np.abs(lse)).all()


def test_bias_of_masked_and_lowest_values():
    """Biases of -inf and of the type's lowest value: the block adds nothing
    beside other keys; alone, the lowest value is an ordinary shift."""
    t = make_tree(8, [4, 6], [600, 500], H=2, Hkv=2, bs=64, window=1, K=4)
    t["bias"][0, :5] = -np.inf
    t["bias"][0, 5:] = np.finfo(np.float32).min
    t["t_bias"] = torch.from_numpy(t["bias"])
    check(t, *attend(t))


def test_rows_without_a_key():
    """No committed token, no visible draft: zeros and -inf; also with blocks
    routed whose keys all lie in other rows' reach."""
    t = make_tree(9, [5, 3], [0, 128], H=2, Hkv=2, bs=64, window=0, K=2)
    t["vis"][:] = False
    t["t_mask"].zero_()
    t["idx"][:] = -1
    t["t_idx"].fill_(-1)
    out, z = attend(t)
    assert (out[:8] == 0).all() and torch.isneginf(z[:8]).all()


def test_not_finite_keys_and_values_stay_in_their_rows():
    """A block with NaN and infinite values that one token routed, and a drafted
    token with NaN: the rows that attend them get NaN, all others what they get
    without.  (Such a row may be computed on another path, with the weights in
    fp32 instead of the caches' type: it is held to the exact result with the
    tolerance of any row, not to the bits of the other path.)"""
    t = make_tree(10, [12, 6], [900, 700], H=2, Hkv=2, bs=64, window=1, K=3, branch=2)
    clean, _ = attend(t)
    ref, lse, A = DO.tree_attend(t["q"].float().numpy(), t["kc"].float().numpy(), t["vc"].float().numpy(), t["idx"],
                                 t["bias"], t["bt"], t["starts"], t["ctx"], t["pos"], t["vis"], t["bs"], t["window"],
                                 SCALE)
    tol = attention_tolerance(ref, A, t["dtype"])
    b = 1
    page = int(t["bt"][0, b])
    rows = set(r for r in range(12) if b in t["idx"][0, r].tolist())
    assert 0 < len(rows) < 12
    bad = {k: v for k, v in t.items()}
    bad["kc"], bad["vc"] = t["kc"].clone(), t["vc"].clone()
    bad["vc"][page, 5, :, 3] = float("nan")
    bad["vc"][page, 6, :, 4] = float("inf")
    bad["kc"][page, 7, :, 5] = float("nan")
    slot = int(t["slots"][12 + 4])
    bad["kc"].view(-1, 2, 128)[slot, :, 0] = float("nan")
    rows |= {12 + i for i in range(6) if t["vis"][12 + i, 4]}
    for splits in (0, 1, 3):
        out, z = attend(bad, splits=splits)
        got, zz = out.float().cpu().numpy(), z.cpu().numpy()
        for r in range(18):
            if r in rows:
                assert torch.isnan(out[r]).any() and torch.isnan(z[r]).all()
            else:
                assert (np.abs(got[r] - ref[r]) <= tol[r]).all(), r
                assert (np.abs(zz[r] - lse[r]) <= 1e-4 + 1e-6 * np.abs(lse[r])).all()
    assert not torch.isnan(clean).any()


def test_single_tokens_equal_the_decode_operator():
    """Trees of one token are the decode step: the same keys, so the two
    operators agree within both tolerances."""
    t = make_tree(12, [1] * 5, [1, 64, 300, 999, 2000], H=4, Hkv=2, bs=64, window=2, K=8)
    out, z = attend(t)
    check(t, out, z)
    ref = torch.zeros_like(out)
    d = {k: v.cuda() for k, v in t.items() if isinstance(v, torch.Tensor)}
    dash_sparse_attn_decode(d["q"], d["kc"], d["vc"], d["t_idx"].expand(2, -1, -1), d["t_bias"].expand(2, -1, -1),
                            d["t_bt"], d["t_ctx"] + 1, 2, SCALE, ref, 1, local_blocks=2, sparse_block_size=64)
    # decode's window holds the token itself: the same set when p - window is
    # the same, which it is (both start behind p - window)
    _, _, A = DO.tree_attend(t["q"][:t["rows"]].float().numpy(), t["kc"].float().numpy(), t["vc"].float().numpy(), t["idx"],
                             t["bias"], t["bt"], t["starts"], t["ctx"], t["pos"], t["vis"], 64, t["window"], SCALE)
    r = ref.float().cpu().numpy()
    assert (np.abs(out.float().cpu().numpy() - r) <= 2 * attention_tolerance(r, A, t["dtype"])).all()


def test_strides_and_wide_tables():
    """q and output as parts of wider rows, caches as parts of a joint K/V
    tensor, a table with more columns and another row distance, int64 ids: the
    same bits at the same number of splits (the automatic number goes by the
    table's width)."""
    t = make_tree(13, [9, 4], [500, 260], H=4, Hkv=2, bs=64, window=2, K=5)
    ref, _ = attend(t, splits=2)
    qkv = torch.randn(13, 4 * 128 * 3, dtype=t["dtype"], device="cuda")
    q = qkv[:, 512:1024].view(13, 4, 128)
    q.copy_(t["q"])
    both = torch.randn(t["P"], 2, 64, 2, 128, dtype=t["dtype"], device="cuda")
    both[:, 0].copy_(t["kc"])
    both[:, 1].copy_(t["vc"])
    wide = torch.full((2, 40), -5, dtype=torch.int32, device="cuda")
    wide[:, 8:8 + t["bt"].shape[1]].copy_(t["t_bt"])
    obuf = torch.full((13, 4, 256), 7.0, dtype=t["dtype"], device="cuda")
    out, z = attend(t, splits=2, out=obuf[:, :, 128:], q=q, kc=both[:, 0], vc=both[:, 1], t_bt=wide[:, 8:],
                    t_idx=t["t_idx"].cuda().long())
    assert torch.equal(out, ref) and (obuf[:, :, :128] == 7.0).all()
    check(t, out, z)


def test_bad_ids_are_recorded_and_left_out():
    t = make_tree(14, [4, 3], [400, 300], H=2, Hkv=2, bs=64, window=1, K=4)
    err = ops.DeviceErrorWord("cuda")
    attend(t, err=err)
    assert err.read()[0] == 0
    good = int(t["idx"][0, 2, 0])
    t["t_idx"][0, 2, 0] = t["idx"][0, 2, 0] = 4000
    out, z = attend(t, err=err)
    assert err.read()[0] == L.DASH_DEV_BAD_BLOCK
    check(t, out, z)
    t["t_idx"][0, 2, 0] = t["idx"][0, 2, 0] = good
    err.clear()
    for page in (t["P"], -3, 2 ** 30):
        b = int(t["idx"][0, 0, 1])
        t["bt"][0, b] = page
        t["t_bt"] = torch.from_numpy(t["bt"])
        out, z = attend(t, err=err)
        assert err.read()[0] == L.DASH_DEV_BAD_PAGE
        check(t, out, z)
        err.clear()


def test_table_narrower_than_the_sequence():
    """Keys behind the table's last column do not exist."""
    t = make_tree(15, [6], [256], H=2, Hkv=2, bs=64, window=1, K=2)
    err = ops.DeviceErrorWord("cuda")
    narrow = t["t_bt"][:, :4].contiguous().cuda()          # the drafts' page is missing
    out, z = attend(t, err=err, t_bt=narrow)
    assert err.read()[0] == L.DASH_DEV_BAD_PAGE
    t["bt"] = np.concatenate([t["bt"][:, :4], np.full((1, 2), -1, np.int32)], 1)
    check(t, out, z)


def test_cache_beyond_32_bits():
    """A cache of more than 2^31 elements: pages at its end."""
    P = 2 ** 31 // (64 * 4 * 128) + 70
    t = make_tree(16, [5, 3], [500, 300], H=4, Hkv=4, bs=64, window=2, K=4, shuffle=False)
    kc = torch.zeros(P, 64, 4, 128, dtype=t["dtype"], device="cuda")
    vc = torch.zeros_like(kc)
    n = t["P"]
    kc[P - n:].copy_(t["kc"])
    vc[P - n:].copy_(t["vc"])
    out, z = attend(t, kc=kc, vc=vc, t_bt=t["t_bt"].cuda() + (P - n))
    check(t, out, z)


def test_streams_and_graphs():
    """Two calls on two streams at once, and a captured call replayed on other
    data, give what the plain call gives."""
    a = make_tree(17, [9, 14], [800, 600], H=4, Hkv=2, bs=64, window=2, K=6)
    b = make_tree(18, [9, 14], [800, 600], H=4, Hkv=2, bs=64, window=2, K=6)
    ra, rb = attend(a)[0], attend(b)[0]
    da, db = ({k: v.cuda() for k, v in t.items() if isinstance(v, torch.Tensor)} for t in (a, b))
    outs = [torch.zeros_like(ra) for _ in range(2)]
    st = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, t, d, o in zip(st, (a, b), (da, db), outs):
            with torch.cuda.stream(s):
                attend(t, out=o, lse=False, **d)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], ra) and torch.equal(outs[1], rb)
    g = [torch.cuda.CUDAGraph() for _ in range(2)]
    for k in range(2):
        with torch.cuda.graph(g[k]):
            attend(a, out=outs[k], lse=False, **da)
    for k in da:
        da[k].copy_(db[k])                # the graphs read these tensors
    outs[0].zero_(), outs[1].zero_()
    torch.cuda.synchronize()
    for s, x in zip(st, g):
        with torch.cuda.stream(s):
            x.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], rb) and torch.equal(outs[1], rb)


def test_wrong_tensors_raise():
    t = make_tree(19, [4], [100], H=2, Hkv=2, bs=64, window=1, K=2)
    d = {k: v.cuda() for k, v in t.items() if isinstance(v, torch.Tensor)}
    for over, words in ((dict(q=d["q"].half()), "dtype"), (dict(kc=d["kc"].float(), vc=d["vc"].float()), "dtype"),
                        (dict(vc=d["vc"].transpose(1, 2).contiguous().transpose(1, 2)), "strides"),
                        (dict(t_mask=d["t_mask"].long()), "tree_mask"), (dict(t_pos=d["t_pos"][:2]), "row_pos"),
                        (dict(t_bt=d["t_bt"][:0]), "block_table"), (dict(t_ctx=d["t_ctx"].cpu()), "CUDA|ctx_lens"),
                        (dict(t_bias=d["t_bias"].double()), "blk_bias"), (dict(kc=d["kc"][:, :32], vc=d["vc"][:, :32]), "caches")):
        with pytest.raises((ValueError, RuntimeError, NotImplementedError), match=words):
            attend(t, **over)


# ---------------------------------------------------------------------------
# the plan
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("nodes,branch", [([1], 1), ([5, 0, 9], 2), ([256, 31, 33], 3), ([40, 200], 0), ([256], 1)])
def test_plan(nodes, branch):
    t = make_tree(20, nodes, [37 * (i + 1) for i in range(len(nodes))], H=1, Hkv=1, bs=16, window=1, K=1, branch=branch,
                  pad_rows=2)
    rows = t["rows"] + 2
    par = torch.cat([torch.from_numpy(t["par"]), torch.full((2,), 9, dtype=torch.int32)]).cuda()
    for parents in (par, None) if branch == 1 else (par,):
        p = drafts.tree_plan(parents, t["t_cu"].cuda(), t["t_ctx"].cuda(), rows=rows, max_nodes=max(nodes),
                             block_table=t["t_bt"].cuda(), block_size=16, num_pages=t["P"])
        n = t["rows"]
        np.testing.assert_array_equal(p.depth[:n].cpu().numpy(), t["depth"])
        np.testing.assert_array_equal(p.row_pos[:n].cpu().numpy(), t["pos"])
        np.testing.assert_array_equal(p.slots[:n].cpu().numpy(), t["slots"])
        assert torch.equal(p.mask[:n].cpu(), t["t_mask"][:n])
        np.testing.assert_array_equal(p.row_seq[:n].cpu().numpy(), np.repeat(np.arange(len(nodes)), nodes))
        assert (p.slots[n:] == -1).all() and (p.depth[n:] == 0).all() and (p.mask[n:] == 0).all()


def test_plan_records_bad_parents():
    err = ops.DeviceErrorWord("cuda")
    par = torch.tensor([-1, 0, 2, 7, -1], dtype=torch.int32).cuda()        # 2's parent is itself, 3's lies behind
    cu, ctx = torch.tensor([0, 5], dtype=torch.int32).cuda(), torch.tensor([10], dtype=torch.int32).cuda()
    p = drafts.tree_plan(par, cu, ctx, rows=5, max_nodes=5, device_error=err)
    assert err.read()[0] == L.DASH_DEV_BAD_TREE
    assert p.depth.tolist() == [0, 1, 0, 0, 0] and p.mask.flatten().tolist() == [1, 3, 4, 8, 16]
    err.clear()
    p = drafts.tree_plan(None, cu, ctx, rows=5, max_nodes=3, device_error=err)      # more drafts than allowed
    assert err.read()[0] == L.DASH_DEV_BAD_TREE and p.depth.tolist() == [0, 1, 2, 0, 0]


# ---------------------------------------------------------------------------
# verification
# ---------------------------------------------------------------------------
def make_verify(seed, nodes, V, mode, dtype=torch.float32, branch=2, sharp=2.0):
    rng = np.random.default_rng(seed)
    starts = np.concatenate([[0], np.cumsum(nodes)]).tolist()
    rows = starts[-1]
    par = sum((tree_parents(n, branch) if n else [] for n in nodes), [])
    logit = rng.standard_normal((rows, V)) * sharp
    soft = lambda x: np.exp(x - x.max(-1, keepdims=True)) / np.exp(x - x.max(-1, keepdims=True)).sum(-1, keepdims=True)  # noqa: E731
    target = torch.from_numpy(logit if mode == "greedy" else soft(logit)).to(dtype)
    draft = torch.from_numpy(soft(logit + rng.standard_normal((rows, V)) * 0.5)).to(dtype) if mode == "drawn" else None
    toks = np.zeros(rows, np.int64)
    for s in range(len(nodes)):
        for i in range(1, nodes[s]):
            r = starts[s] + i
            p = starts[s] + par[r]
            if mode == "drawn":
                q = draft[p].double().numpy()
                toks[r] = rng.choice(V, p=q / q.sum())
            else:
                best = np.argsort(-target[p].double().numpy(), kind="stable")
                toks[r] = best[0 if rng.random() < 0.6 else min(V - 1, int(rng.integers(1, 4)))]
    return dict(tokens=toks, par=np.array(par, np.int32), starts=starts, target=target, draft=draft,
                ua=rng.random(rows).astype(np.float32), us=rng.random(len(nodes)).astype(np.float32), mode=mode,
                nodes=nodes)


def run_verify(v, max_nodes=None, parents=True, err=None, target=None, draft=None):
    g = v["mode"] == "greedy"
    cu = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()                        # noqa: E731
    m = max_nodes or max(v["nodes"] + [1])
    r = drafts.verify_drafts(cu(v["tokens"]), cu(v["par"]) if parents else None,
                             torch.tensor(v["starts"], dtype=torch.int32).cuda(),
                             v["target"].cuda() if target is None else target, max_nodes=m,
                             draft=(None if v["draft"] is None else v["draft"].cuda()) if draft is None else draft,
                             u_accept=None if g else cu(v["ua"]), u_sample=None if g else cu(v["us"]), greedy=g,
                             device_error=err)
    return [x.cpu().numpy() for x in (r.n_accept, r.path, r.next_token, r.tokens)]


def check_verify(v, got, max_nodes=None, parents=True):
    want = DO.verify(v["tokens"], v["par"] if parents else None, v["starts"], v["target"].double().numpy(),
                     None if v["draft"] is None else v["draft"].double().numpy(), v["ua"], v["us"], v["mode"],
                     max_nodes or max(v["nodes"] + [1]))
    for name, a, b in zip(("n_accept", "path", "next_token", "tokens"), got, want):
        np.testing.assert_array_equal(a, b, err_msg=name)


@pytest.mark.parametrize("mode", ["drawn", "certain", "greedy"])
@pytest.mark.parametrize("nodes,V,branch", [([4], 129280, 1), ([16] * 6, 1000, 3), ([1, 0, 7, 2], 97, 2), ([9] * 70, 333, 2),
                                            ([12] * 3, 30001, 4), ([256, 40], 64, 0), ([5, 6], 1, 1), ([8] * 4, 8192, 1)])
def test_verify(mode, nodes, V, branch):
    for seed in range(3):
        v = make_verify(seed, nodes, V, mode, branch=branch)
        check_verify(v, run_verify(v))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("mode", ["drawn", "certain", "greedy"])
@pytest.mark.parametrize("V", [4096, 4099])
def test_verify_types(mode, dtype, V):
    """16-bit rows (bf16 logits have equal largest values: the lowest index)."""
    v = make_verify(7, [10] * 5, V, mode, dtype=dtype, branch=2)
    check_verify(v, run_verify(v))


def test_verify_chain_without_parents_and_wider_outputs():
    v = make_verify(8, [6, 3], 500, "drawn", branch=1, sharp=0.5)
    check_verify(v, run_verify(v, parents=False), parents=False)
    check_verify(v, run_verify(v, max_nodes=11), max_nodes=11)


def test_verify_strided_rows():
    v = make_verify(9, [7, 5], 400, "drawn")
    wide = torch.full((12, 1001), float("nan"), device="cuda")
    wide[:, 3:403] = v["target"].cuda()
    wide[:, 503:903] = v["draft"].cuda()
    check_verify(v, run_verify(v, target=wide[:, 3:403], draft=wide[:, 503:903]))


@pytest.mark.parametrize("mode", ["drawn", "certain", "greedy"])
def test_verify_odd_inputs(mode):
    """Tokens outside the vocabulary are passed over; equal siblings; u of 0 and
    just below 1."""
    v = make_verify(10, [9, 9, 9, 9], 50, mode, branch=3)
    v["tokens"][[2, 11, 20]] = [-1, 50, 2 ** 40]
    v["tokens"][[3, 12]] = v["tokens"][[1, 10]]
    v["ua"][9:18], v["us"][:2] = 0.0, 0.0
    v["ua"][18:], v["us"][2:] = np.float32(1 - 2 ** -24), np.float32(1 - 2 ** -24)
    check_verify(v, run_verify(v))


def test_verify_empty_residual():
    """Target and draft equal: a draft is kept whatever the number below 1; where
    it cannot be (probability 0 on both sides) the residual is empty and the
    token is drawn from the row itself; an all-zero row gives -1."""
    V = 40
    p = np.full((6, V), 1.0 / 32)
    p[:, 32:] = 0.0
    p[3:] = 0.0
    v = dict(tokens=np.array([0, 33, 34, 0, 1, 2]), par=np.array([-1, 0, 0, -1, 0, 0], np.int32), starts=[0, 3, 6],
             target=torch.from_numpy(p).float(), draft=torch.from_numpy(p).float(), ua=np.full(6, 0.5, np.float32),
             us=np.array([0.5, 0.5], np.float32), mode="drawn", nodes=[3, 3])
    got = run_verify(v)
    check_verify(v, got)
    assert got[2].tolist() == [16, -1]
    v["mode"], v["draft"] = "certain", None
    check_verify(v, run_verify(v))


def test_verify_greedy_ties_and_nan():
    x = torch.zeros(4, 100)
    x[0, [7, 60]] = 5.0
    x[1] = -0.0
    x[1, 3] = 0.0                                            # equal to -0: index 0 wins
    x[2, [20, 30]] = float("nan")
    x[3] = -float("inf")
    v = dict(tokens=np.array([0, 7, 0, 20]), par=np.array([-1, 0, 1, 2], np.int32), starts=[0, 4], target=x, draft=None,
             ua=None, us=None, mode="greedy", nodes=[4])
    got = run_verify(v)
    assert got[0].tolist() == [3] and got[2].tolist() == [0]
    assert got[3].tolist() == [[7, 0, 20, 0]]


def test_verify_bad_tree_recorded_and_refusals():
    v = make_verify(11, [5], 30, "certain")
    v["par"][3] = 4
    err = ops.DeviceErrorWord("cuda")
    check_verify(v, run_verify(v, err=err))
    assert err.read()[0] == L.DASH_DEV_BAD_TREE
    t = v["target"].cuda()
    tok, cu = torch.zeros(5, dtype=torch.int64).cuda(), torch.tensor([0, 5], dtype=torch.int32).cuda()
    with pytest.raises(ValueError, match="needed unless"):
        drafts.verify_drafts(tok, None, cu, t, max_nodes=5)
    with pytest.raises(ValueError, match="neither"):
        drafts.verify_drafts(tok, None, cu, t, max_nodes=5, greedy=True, u_accept=torch.zeros(5).cuda())
    with pytest.raises(ValueError, match="tokens"):
        drafts.verify_drafts(tok.int(), None, cu, t, max_nodes=5, greedy=True)
    with pytest.raises(ValueError, match="draft"):
        drafts.verify_drafts(tok, None, cu, t, max_nodes=5, draft=t.half(), u_accept=torch.zeros(5).cuda(),
                             u_sample=torch.zeros(1).cuda())
    with pytest.raises(ValueError, match="target"):
        drafts.verify_drafts(tok, None, cu, t.double(), max_nodes=5, greedy=True)


def test_verify_graph_replays_on_new_numbers():
    a, b = make_verify(12, [8] * 4, 5000, "drawn"), make_verify(13, [8] * 4, 5000, "drawn")
    cu = lambda v: [torch.from_numpy(v[k]).cuda() for k in ("tokens", "par", "ua", "us")] + [v["target"].cuda(), v["draft"].cuda()]  # noqa: E731
    x, y = cu(a), cu(b)
    st = torch.tensor(a["starts"], dtype=torch.int32).cuda()
    call = lambda: drafts.verify_drafts(x[0], x[1], st, x[4], max_nodes=8, draft=x[5], u_accept=x[2], u_sample=x[3])  # noqa: E731
    call()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = call()
    for p, q in zip(x, y):
        p.copy_(q)
    g.replay()
    torch.cuda.synchronize()
    check_verify(b, [z.cpu().numpy() for z in (r.n_accept, r.path, r.next_token, r.tokens)])
