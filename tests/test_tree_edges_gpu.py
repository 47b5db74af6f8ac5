"""Draft-tree attention at its edges: router heads shared in part, biases of the
type's lowest value and of -inf, an output that lies on q."""
import numpy as np
import pytest
import torch

from ananta_ocr_b200 import drafts
from oracle import draft_oracle as DO
from draft_testutil import attention_tolerance, make_tree

pytestmark = pytest.mark.gpu
SCALE = 1.0 / np.sqrt(128)
LOW = np.finfo(np.float32).min


def attend(t, idx, bias, *, splits=0, out=None, q=None, scale=SCALE, **over):
    d = {k: over.get(k, v).cuda() for k, v in t.items() if isinstance(v, torch.Tensor)}
    q = d["q"] if q is None else q
    out = torch.full(q.shape, 7.0, dtype=t["dtype"], device="cuda") if out is None else out
    z = torch.full(q.shape[:2], 7.0, device="cuda")
    drafts.dash_sparse_attn_tree(q, d["kc"], d["vc"], idx, bias, d["t_bt"], d["t_cu"], d["t_ctx"], d["t_pos"],
                                 d["t_mask"], max(t["nodes"]), t["Hkv"], scale, out, local_blocks=t["local_blocks"],
                                 sparse_block_size=t["bs"], num_splits=splits, lse=z)
    return out, z


def exact(t, idx, bias, scale=SCALE):
    return DO.tree_attend(t["q"].float().numpy(), t["kc"].float().numpy(), t["vc"].float().numpy(), idx, bias, t["bt"],
                          t["starts"], t["ctx"], t["pos"], t["vis"], t["bs"], t["window"], scale)


def close(t, got, want, rows=slice(None)):
    out, z = (x.float().cpu().numpy()[rows] for x in got)
    ref, lse, A = (x[rows] for x in want)
    assert (np.abs(out - ref) <= attention_tolerance(ref, A, t["dtype"])).all()
    none = np.isneginf(lse)
    assert (np.isneginf(z) == none).all()
    assert (np.abs(z[~none] - lse[~none]) <= 1e-4 + 1e-6 * np.abs(lse[~none])).all()


# ---------------------------------------------------------------------------
# router heads
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("bs", [64, 48])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("shared", ["ids", "biases", "both", "neither", "ids_none"])
def test_ids_and_biases_of_one_head_or_of_each(shared, dtype, bs):
    """Ids and biases are per kv head each for itself: either may be one head
    expanded over the others."""
    t = make_tree(31, [9, 5], [800, 500], H=4, Hkv=2, bs=bs, window=1, K=5, index_heads=2)
    idx, bias = t["idx"].copy(), t["bias"].copy()
    if shared in ("ids", "both", "ids_none"):
        idx[1] = idx[0]
    if shared in ("biases", "both"):
        bias[1] = bias[0]
    gi, gb = torch.from_numpy(idx).cuda().to(dtype), torch.from_numpy(bias).cuda()
    if shared in ("ids", "both", "ids_none"):
        gi = gi[:1].expand(2, -1, -1)
    if shared in ("biases", "both"):
        gb = gb[:1].expand(2, -1, -1)
    if shared == "ids_none":
        gb = bias = None
    close(t, attend(t, gi, gb), exact(t, idx, bias))


# ---------------------------------------------------------------------------
# biases
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("splits", [0, 1, 3])
@pytest.mark.parametrize("bs", [64, 32, 48])
def test_lowest_biases_alone(bs, splits):
    """Rows whose only keys lie in blocks of lowest biases: in the sum of logit and
    bias the logit vanishes (in 32 bits as in 64), so the keys of the largest bias
    share the weight equally; lse is that bias.  Beside another key they add
    nothing.  Biases: the lowest value, values whose product with log2(e) is past
    the type's range, one just inside it, -1e35, and -inf (no key at all)."""
    n = 8
    t = make_tree(32, [n], [6 * bs], H=2, Hkv=2, bs=bs, window=0, K=3)
    t["idx"][0] = np.array([[0, 2, 5]] * n)
    t["vis"][:] = False
    t["t_mask"].zero_()
    b = t["bias"][0]
    b[0] = LOW
    b[1] = [LOW, -3.0e38, LOW]
    b[2] = [-2.5e38, -2.4e38, -2.4e38]
    b[3] = [-2.3e38, LOW, -2.3e38]
    b[4] = [-1e35, -1e35, LOW]
    b[5] = [-np.inf, LOW, -np.inf]
    b[6] = -np.inf
    b[7] = [LOW, 1.0, -np.inf]
    t["idx"][0, 5] = [4, -1, 4]                            # the repeated id: the first, -inf, counts
    b[5] = [-np.inf, 0.0, LOW]
    want = exact(t, t["idx"], t["bias"])
    assert np.isneginf(want[1][5:7]).all()
    gi, gb = torch.from_numpy(t["idx"]).cuda().expand(2, -1, -1), torch.from_numpy(t["bias"]).cuda().expand(2, -1, -1)
    close(t, attend(t, gi, gb, splits=splits), want)


@pytest.mark.parametrize("splits", [0, 1, 3])
@pytest.mark.parametrize("bs", [64, 32, 48])
def test_what_a_bias_of_minus_infinity_masks_may_hold_anything(bs, splits):
    """A bias of -inf masks a block: NaN and infinities in it stay out."""
    n = 6
    t = make_tree(33, [n], [6 * bs], H=2, Hkv=2, bs=bs, window=1, K=3)
    t["idx"][0] = np.array([[0, 2, 3]] * n)
    t["bias"][0, :, 1] = -np.inf
    t["bias"][0, 4] = -np.inf                             # only the drafts are left
    page = int(t["bt"][0, 2])
    want = exact(t, t["idx"], t["bias"])
    t["kc"][page, 3, :, 5] = float("nan")
    t["kc"][page, 4] = float("inf")
    t["vc"][page, 5:9] = float("nan")
    t["vc"][page, 9, :, ::2] = -float("inf")
    gi, gb = torch.from_numpy(t["idx"]).cuda().expand(2, -1, -1), torch.from_numpy(t["bias"]).cuda().expand(2, -1, -1)
    close(t, attend(t, gi, gb, splits=splits), want)


# ---------------------------------------------------------------------------
# an output that lies on q
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("scale", [SCALE, -SCALE])
@pytest.mark.parametrize("splits", [1, 0, 3])
@pytest.mark.parametrize("bs", [64, 48])
def test_output_in_place_of_q(bs, splits, scale):
    """The result may be written over q; also for the rows that are computed again
    because a neighbour attends a NaN (rows of token 0 do, all others must not)."""
    n = 9
    t = make_tree(34, [n], [6 * bs], H=4, Hkv=2, bs=bs, window=1, K=3)
    t["idx"][0] = np.array([[0, -1, 3]] * n)
    t["idx"][0, 0, 1] = 2
    want = exact(t, t["idx"], t["bias"], scale)
    t["vc"][int(t["bt"][0, 2]), 5] = float("nan")
    gi, gb = torch.from_numpy(t["idx"]).cuda().expand(2, -1, -1), torch.from_numpy(t["bias"]).cuda().expand(2, -1, -1)
    got = attend(t, gi, gb, splits=splits, scale=scale)
    close(t, got, want, slice(1, None))
    q = t["q"].cuda()
    here = attend(t, gi, gb, splits=splits, scale=scale, q=q, out=q)
    assert here[0] is q and torch.isnan(q[0]).any()
    close(t, here, want, slice(1, None))
    assert torch.equal(here[0][1:], got[0][1:]) and torch.equal(here[1][1:], got[1][1:])
