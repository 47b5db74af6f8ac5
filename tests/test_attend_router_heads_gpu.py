"""Paged prefill and decode attention: ids and biases are per kv head each for
itself; a call with one of them expanded over the heads equals the call with
both written out."""
import pytest
import torch

from ananta_ocr_b200.unlimited_dash_ops.attend_triton import dash_sparse_attn, dash_sparse_attn_decode
from draft_testutil import make_tree

pytestmark = pytest.mark.gpu


def call(op, t, idx, bias):
    d = {k: v.cuda() for k, v in t.items() if isinstance(v, torch.Tensor)}
    out = torch.zeros_like(d["q"])
    if op == "decode":
        dash_sparse_attn_decode(d["q"], d["kc"], d["vc"], idx, bias, d["t_bt"], d["t_ctx"] + 1, 2, 0.1, out, 1,
                                local_blocks=1, sparse_block_size=64)
    else:
        dash_sparse_attn(d["q"], d["kc"], d["vc"], idx, bias, d["t_bt"], d["t_cu"], d["t_ctx"] + d["t_cu"].diff(),
                         d["t_ctx"], max(t["nodes"]), 2, 0.1, out, local_blocks=1, sparse_block_size=64)
    return out


@pytest.mark.parametrize("shared", ["ids", "biases", "both"])
@pytest.mark.parametrize("op", ["decode", "prefill"])
def test_expanded_ids_or_biases(op, shared):
    nodes = [1, 1, 1] if op == "decode" else [7, 1, 40]
    t = make_tree(35, nodes, [800, 500, 300], H=4, Hkv=2, bs=64, window=1, K=4, index_heads=2, branch=1)
    idx, bias = t["t_idx"].clone(), t["t_bias"].clone()
    if shared != "biases":
        idx[1] = idx[0]
    if shared != "ids":
        bias[1] = bias[0]
    idx, bias = idx.cuda(), bias.cuda()
    want = call(op, t, idx, bias)
    got = call(op, t, idx if shared == "biases" else idx[:1].expand(2, -1, -1),
               bias if shared == "ids" else bias[:1].expand(2, -1, -1))
    assert torch.isfinite(want).all() and torch.equal(got, want)
